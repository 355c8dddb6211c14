"""The scaled 8-bit paged cache against its plain 64-bit implementation (GPU).

append: codes, scales and rotated queries equal the oracle's bit for bit (the
operator defines every fp32 rounding).

attend: |out - exact| <= half a step of the output type * |exact| + d * vmax, the
weights' relative error d bounded by
  logits   2 (D + 8) 2^-24 max_t sum_i |q_i k_ti| scale     (fp32 sums of D products)
  exp      2^-20
  pieces   16-bit types keep a weight as three 8-bit pieces of 4 bits: 2^-11, and
           2^-18 of the largest weight for each token; fp32 keeps six: 2^-23, 2^-28.
lse: the logits' bound + 2^-20 max(1, |lse|).
"""
import numpy as np
import pytest

import scaled_cache_oracle as o

pytestmark = pytest.mark.gpu

TYPES = {"f32": "float32", "bf16": "bfloat16", "f16": "float16"}


@pytest.fixture(scope="module")
def torch():
    return pytest.importorskip("torch")


def f32(t):
    return t.float().cpu().numpy()


class Setup:
    """A pool with random contents, page tables without shared pages, and its oracle twin."""

    def __init__(self, torch, dsd, fmt, lens, D=64, Hk=2, P=16, bt=None, layout="token", seed=0, spare=2, spread=1.0):
        rng = np.random.default_rng(seed)
        self.rng, self.fmt, self.lens, self.D, self.Hk, self.P = rng, fmt, list(lens), D, Hk, P
        bt = P if bt is None else bt
        need = [-(-n // P) for n in lens]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(lens), max(need + [1]) + 1), 10 ** 6, np.int32)   # junk behind the pages
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        shape = (pages, P, Hk, D)
        codes, scales = {}, {}
        for n in "kv":
            x = rng.standard_normal(shape) * (34 if fmt == "int8" else 120)
            codes[n] = o.encode(x, fmt)
            scales[n] = (np.exp(rng.uniform(-spread, spread, (pages, Hk, P // bt))) * 3.7 / o.QMAX[fmt]).astype(np.float32)
        self.pool = o.Pool(fmt, codes, scales)
        kind = torch.float8_e4m3fn if fmt == "fp8" else torch.int8

        def up(c):
            t = torch.from_numpy(c.view(np.int8)).cuda()
            t = t.transpose(1, 2).contiguous().transpose(1, 2) if layout == "head" else t
            return t.view(kind)

        self.cache = dsd.ScaledKVCache.from_tensors(up(codes["k"]), up(codes["v"]), torch.from_numpy(scales["k"]).cuda(),
                                                    torch.from_numpy(scales["v"]).cuda())
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d_lens = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def same(self, torch):
        for n, c, s in (("k", self.cache.k_codes, self.cache.k_scales), ("v", self.cache.v_codes, self.cache.v_scales)):
            assert np.array_equal(s.cpu().numpy(), self.pool.scales[n], equal_nan=True), n
            got = c.view(torch.int8).cpu().numpy().view(np.uint8)
            assert np.array_equal(got, self.pool.codes[n]), (n, np.argwhere(got != self.pool.codes[n])[:5])


def offsets_of(torch, counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)).cuda()


# ------------------------------------------------------------------- append

APPENDS = [
    # fmt, dtype, D, rotary, interleaved, P, bt, layout, lens, new
    ("fp8", "bf16", 128, 128, False, 16, 16, "token", [1, 17, 40, 33, 300], [1, 1, 9, 33, 217]),
    ("int8", "bf16", 64, 64, True, 16, 4, "head", [5, 16, 100], [5, 1, 37]),
    ("int8", "f16", 64, 32, False, 32, 32, "token", [31, 64, 200, 7], [2, 64, 130, 3]),
    ("fp8", "f32", 80, 80, False, 8, 8, "token", [9, 30, 64], [4, 30, 1]),
    ("int8", "f32", 96, 16, True, 64, 16, "head", [70, 128, 3], [6, 100, 3]),
    ("fp8", "f16", 128, 64, True, 128, 128, "token", [129, 500], [3, 372]),
    ("int8", "bf16", 256, 256, False, 256, 256, "head", [300, 513], [300, 250]),
    ("fp8", "bf16", 72, 20, False, 6, 3, "token", [11, 50], [5, 31]),      # nothing a vector could take
    ("int8", "f32", 8, 6, True, 1, 1, "token", [3, 12], [3, 5]),
    ("fp8", "bf16", 128, 0, False, 16, 16, "token", [20, 33], [20, 16]),   # no rotation
]


@pytest.mark.parametrize("fmt,dtype,D,rd,inter,P,bt,layout,lens,new", APPENDS)
@pytest.mark.parametrize("with_q", [True, False])
def test_append_bits(torch, dsd, fmt, dtype, D, rd, inter, P, bt, layout, lens, new, with_q):
    s = Setup(torch, dsd, fmt, lens, D, 3, P, bt, layout, seed=D + P, spread=0.3)
    T, H, dt = sum(new), 6, getattr(torch, TYPES[dtype])
    rows = torch.randn(T, H + 6, D, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(dt)
    rows *= torch.rand(T, 1, 1, device="cuda") * 3      # tails that need a larger scale, and some that do not
    q, k, v = rows[:, :H], rows[:, H:H + 3], rows[:, H + 3:]
    rot = cos = sin = None
    if rd:
        rot = dsd.RotaryTable.from_base(max(lens) + 1, rd, 10000.0, inter)
        cos, sin = rot.cos.cpu().numpy(), rot.sin.cpu().numpy()
    got = s.cache.append(k, v, s.d_table, s.d_lens, offsets_of(torch, new), rotary=rot, q=q if with_q else None)
    at = 0
    for b, n in enumerate(new):
        s.pool.append("k", f32(k[at:at + n]), s.table[b], lens[b], cos, sin, inter)
        s.pool.append("v", f32(v[at:at + n]), s.table[b], lens[b])
        at += n
    s.same(torch)
    s.cache.check()
    if with_q:
        at = 0
        for b, n in enumerate(new):
            for j in range(n):
                p = lens[b] - n + j
                want = o.rotate(f32(q[at + j]), None if cos is None else cos[p], None if sin is None else sin[p], inter)
                assert np.array_equal(f32(got[at + j]), f32(torch.from_numpy(want).to(dt)))
            at += n
    else:
        assert got is None


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_append_one_token_each_many_steps(torch, dsd, fmt):
    """A decode loop: the block's scale grows with its tokens, older codes are rounded again."""
    lens = [1, 15, 16, 31, 40]
    s = Setup(torch, dsd, fmt, [n + 20 for n in lens], 64, 2, 16, 8, seed=3)
    rot = dsd.RotaryTable.from_base(100, 64, 500.0)
    cos, sin = rot.cos.cpu().numpy(), rot.sin.cpu().numpy()
    gen = torch.Generator("cuda").manual_seed(2)
    counts = torch.zeros(s.cache.num_pages, dtype=torch.int32, device="cuda")
    for step in range(20):
        now = [n + step for n in lens]
        k, v = (torch.randn(5, 2, 64, device="cuda", generator=gen).bfloat16() * 1.3 ** step for _ in range(2))
        s.cache.append(k, v, s.d_table, torch.tensor(now, dtype=torch.int32, device="cuda"), rotary=rot, token_counts=counts)
        for b, n in enumerate(now):
            s.pool.append("k", f32(k[b:b + 1]), s.table[b], n, cos, sin)
            s.pool.append("v", f32(v[b:b + 1]), s.table[b], n)
            assert int(counts[s.table[b, (n - 1) // 16]]) == (n - 1) % 16 + 1
    s.same(torch)


def test_append_in_place_query_positions_and_strided_rows(torch, dsd):
    lens, new = [40, 9], [12, 9]
    s = Setup(torch, dsd, "fp8", lens, 64, 2, 16, seed=5)
    rot = dsd.RotaryTable.from_base(5000, 64)
    base = torch.randn(21, 9, 80, device="cuda").half()      # odd strides, rows that start off any boundary
    q, k, v = base[:, 0:4, 3:67], base[:, 4:6, 1:65], base[:, 6:8, 5:69]
    q0 = q.clone()
    pos = torch.randint(0, 5000, (21,), device="cuda", dtype=torch.int32)
    out = s.cache.append(k, v, s.d_table, s.d_lens, offsets_of(torch, new), rotary=rot, positions=pos, q=q, q_out=q)
    assert out.data_ptr() == q.data_ptr()
    cos, sin, P = rot.cos.cpu().numpy(), rot.sin.cpu().numpy(), pos.cpu().numpy()
    at = 0
    for b, n in enumerate(new):
        s.pool.append("k", f32(k[at:at + n]), s.table[b], lens[b], cos, sin, positions=P[at:at + n])
        s.pool.append("v", f32(v[at:at + n]), s.table[b], lens[b])
        at += n
    s.same(torch)
    for t in range(21):
        want = o.rotate(f32(q0[t]), cos[P[t]], sin[P[t]], False)
        assert np.array_equal(f32(q[t]), f32(torch.from_numpy(want).half()))


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_append_zeros_infinities_nan(torch, dsd, fmt):
    """A block of zeros has scale 0; infinities saturate and NaN stays alone: neither reaches the scale."""
    lens = [16, 16, 16, 20]
    s = Setup(torch, dsd, fmt, lens, 64, 2, 16, seed=6)
    k = torch.randn(68, 2, 64, device="cuda")
    v = torch.randn(68, 2, 64, device="cuda")
    k[:16] = 0
    k[16:32] *= 1e-35
    v[20, 0, 5], v[21, 1, 9], v[22, 0, 63] = float("inf"), float("-inf"), float("nan")
    v[40:48] = float("nan")
    k[50] = float("inf")
    offs = offsets_of(torch, lens)
    s.cache.append(k, v, s.d_table, s.d_lens, offs)
    at = 0
    for b, n in enumerate(lens):
        s.pool.append("k", f32(k[at:at + n]), s.table[b], n)
        s.pool.append("v", f32(v[at:at + n]), s.table[b], n)
        at += n
    s.same(torch)


def test_append_leaves_bad_tokens_out(torch, dsd):
    lens = [20, 20, 20, 20]
    s = Setup(torch, dsd, "fp8", lens, 64, 2, 16, seed=7)
    k, v = (torch.randn(80, 2, 64, device="cuda").bfloat16() for _ in range(2))
    table = s.table.copy()
    table[1, 0] = s.pool.pages            # one behind the pool
    table[2, 1] = -1
    bad_len = [20, 20, 20, 3]             # fewer tokens than new ones
    s.cache.append(k, v, torch.from_numpy(table).cuda(), torch.tensor(bad_len, dtype=torch.int32, device="cuda"),
                   offsets_of(torch, lens))
    for name, x in (("k", k), ("v", v)):
        s.pool.append(name, f32(x[0:20]), table[0], 20)
        half = o.Pool("fp8", s.pool.codes, s.pool.scales)
        # request 1: its second page only, request 2: its first page only
        half.append(name, f32(x[20:40]), [s.table[1, 0], table[1, 1]], 20)
        half.append(name, f32(x[40:60]), [table[2, 0], s.table[2, 1]], 20)
        for page in (table[1, 1], table[2, 0]):
            s.pool.codes[name][page], s.pool.scales[name][page] = half.codes[name][page], half.scales[name][page]
    s.same(torch)
    with pytest.raises(dsd.OutOfRange):
        s.cache.check()
    s.cache.check()                       # reported once
    rot = dsd.RotaryTable.from_base(10, 64)
    s.cache.append(k[:4], v[:4], s.d_table, s.d_lens, rotary=rot)   # place 19 of a table with 10
    with pytest.raises(dsd.OutOfRange, match="rotation"):
        s.cache.check()


# ---------------------------------------------------------------- attention

def tolerance(q, pool, ids, length, scale, out, lse, dtype, G, seen=None):
    """Bounds of the docstring for one request: q [n][H][D] as the kernel reads it."""
    n, H, D = q.shape
    tol_o, tol_l = np.zeros(out.shape), np.zeros(lse.shape)
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dtype]
    piece, spot = (2.0 ** -23, 2.0 ** -28) if dtype == "f32" else (2.0 ** -11, 2.0 ** -18)
    for h in range(pool.Hk):
        k, v = (np.nan_to_num(pool.rows(x, ids, np.arange(length), h)) for x in "kv")
        hs = slice(h * G, (h + 1) * G)
        x = np.nan_to_num(q[:, hs].astype(np.float64), posinf=0, neginf=0)
        if not length:
            continue
        big = (np.abs(x) @ np.abs(k).T).max(-1) * abs(scale)
        z = x @ k.T * scale
        total = np.exp(z - z.max(-1, keepdims=True)).sum(-1)
        zerr = 2 * (D + 8) * 2.0 ** -24 * big
        d = zerr + 2.0 ** -20 + piece + length * spot / np.maximum(1.0, total)
        tol_o[:, hs] = half * np.abs(out[:, hs]) + (d * np.abs(v).max())[..., None]
        seen = np.isfinite(lse[:, hs])
        tol_l[:, hs] = np.where(seen, zerr + 2.0 ** -20 * np.maximum(1.0, np.abs(np.where(seen, lse[:, hs], 0))), 0.0)
    return tol_o, tol_l


def close(got, want, tol):
    bad = ~((np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


ATTENDS = [
    # fmt, dtype, D, H, Hk, P, bt, layout, lens, queries, causal, window
    ("fp8", "bf16", 128, 8, 2, 16, 16, "token", [1, 2, 127, 128, 129, 300], None, True, 0),
    ("fp8", "bf16", 128, 8, 1, 16, 16, "head", [700, 3, 256], None, True, 0),
    ("int8", "bf16", 128, 4, 4, 32, 8, "token", [77, 1, 257], None, True, 0),
    ("int8", "f16", 64, 16, 2, 64, 64, "head", [400, 63, 64, 65], None, True, 100),
    ("fp8", "f16", 64, 5, 1, 8, 8, "token", [200, 9], None, True, 0),
    ("int8", "f32", 128, 6, 2, 16, 16, "token", [300, 17], None, True, 0),
    ("fp8", "f32", 128, 4, 2, 128, 16, "head", [300, 129], None, True, 7),
    ("fp8", "f32", 96, 2, 2, 16, 4, "token", [50], None, True, 0),
    ("fp8", "bf16", 80, 28, 4, 16, 16, "token", [100, 33], None, True, 0),
    ("int8", "bf16", 16, 2, 1, 16, 16, "token", [100], None, True, 0),
    ("fp8", "bf16", 128, 4, 2, 256, 128, "token", [255, 256, 300, 700], None, True, 0),
    ("int8", "bf16", 64, 4, 2, 136, 8, "head", [135, 136, 137, 400], None, True, 150),
    ("fp8", "bf16", 256, 4, 2, 16, 16, "token", [150, 20], None, True, 0),      # off the tensor-core path
    ("int8", "f32", 200, 3, 1, 16, 16, "token", [40], None, True, 0),
    ("fp8", "f16", 72, 2, 2, 6, 3, "token", [50, 7], None, True, 9),
    ("int8", "bf16", 64, 2, 2, 1, 1, "token", [130, 5], None, True, 0),
    ("fp8", "bf16", 128, 8, 2, 16, 16, "token", [40, 300, 7, 130], [3, 8, 7, 2], True, 0),
    ("int8", "f16", 64, 4, 4, 16, 16, "token", [200, 50, 10], [60, 50, 1], True, 0),
    ("fp8", "f32", 128, 4, 1, 32, 32, "head", [200, 90], [33, 17], True, 40),
    ("int8", "bf16", 128, 6, 2, 16, 16, "token", [100, 60], [20, 5], False, 0),
    ("fp8", "bf16", 64, 4, 2, 16, 16, "token", [100, 60], [20, 5], False, 30),
    ("fp8", "f16", 96, 40, 1, 16, 16, "token", [140, 33], [4, 2], True, 0),
    # many key heads leave few ranges: several tiles and units to a CTA
    ("fp8", "bf16", 128, 64, 64, 16, 16, "token", [1900, 3, 700, 0, 1300], None, True, 0),
    ("int8", "f32", 64, 128, 64, 32, 8, "head", [900, 1700, 400], None, True, 500),
    ("fp8", "bf16", 128, 512, 64, 16, 16, "token", [1500, 640], None, True, 0),
    ("int8", "f16", 64, 192, 96, 16, 4, "token", [800, 1000], [5, 3], True, 0),
    ("fp8", "bf16", 64, 96, 48, 16, 16, "token", [1200, 500, 90], [70, 130, 90], True, 0),
    ("int8", "bf16", 128, 64, 64, 32, 32, "head", [700, 1000], [150, 40], True, 333),
    ("fp8", "f32", 128, 64, 64, 16, 1, "token", [600, 300], [40, 20], True, 0),
    ("int8", "f16", 80, 144, 72, 16, 16, "token", [1300], [200], False, 0),
    ("fp8", "bf16", 72, 64, 64, 6, 6, "token", [6000, 1000], [3, 20], True, 0),
]


@pytest.mark.parametrize("fmt,dtype,D,H,Hk,P,bt,layout,lens,new,causal,window", ATTENDS)
def test_attend(torch, dsd, fmt, dtype, D, H, Hk, P, bt, layout, lens, new, causal, window):
    s = Setup(torch, dsd, fmt, lens, D, Hk, P, bt, layout, seed=H * P + D)
    counts = new or [1] * len(lens)
    T, dt = sum(counts), getattr(torch, TYPES[dtype])
    q = (torch.randn(T, H, D, device="cuda", generator=torch.Generator("cuda").manual_seed(3)) * 1.5).to(dt)
    offs = offsets_of(torch, counts) if new else None
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, offs, causal=causal, window=window, return_lse=True)
    s.cache.check()
    again, lse2 = s.cache.attend(q, s.d_table, s.d_lens, offs, causal=causal, window=window, return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    only = s.cache.attend(q, s.d_table, s.d_lens, offs, causal=causal, window=window)
    assert torch.equal(only, out)
    at, scale = 0, D ** -0.5
    for b, n in enumerate(counts):
        x = f32(q[at:at + n])
        want, wl = o.attend(s.pool, x, s.table[b], lens[b], scale, causal, window)
        to, tl = tolerance(x, s.pool, s.table[b], lens[b], scale, want, wl, dtype, H // Hk)
        close(f32(lse[at:at + n]).astype(np.float64), wl, tl)
        close(f32(out[at:at + n]).astype(np.float64), want, to)
        at += n


@pytest.mark.parametrize("arrangement", ["kv in one page", "padded rows", "padded pages", "odd base", "rows of tokens"])
@pytest.mark.parametrize("new", [None, [40, 7]])
def test_attend_and_append_other_arrangements(torch, dsd, arrangement, new):
    """Pools whose K and V share pages or whose strides TMA does or does not take give the plain pool's bits."""
    s = Setup(torch, dsd, "fp8", [150, 60], 64, 2, 16, seed=31)
    pages, P, Hk, D = s.pool.codes["k"].shape
    raw = torch.zeros(pages * P * Hk * D * 6 + 4096, dtype=torch.int8, device="cuda")

    def views():
        if arrangement == "kv in one page":
            both = raw[:2 * pages * P * Hk * D].view(pages, 2, P, Hk, D)
            return both[:, 0], both[:, 1]
        if arrangement == "padded rows":          # 72 bytes a row
            both = raw[:2 * pages * P * Hk * 72].view(2, pages, P, Hk, 72)
            return both[0, ..., 4:68], both[1, ..., :64]
        if arrangement == "padded pages":         # a page stride that is no multiple of a token's
            both = raw[:2 * pages * (P * Hk * D + 48)].view(2, pages, -1)
            return tuple(both[i, :, :P * Hk * D].unflatten(1, (P, Hk, D)) for i in range(2))
        if arrangement == "odd base":
            both = raw[8:8 + 2 * pages * P * Hk * D].view(2, pages, P, Hk, D)
            return both[0], both[1]
        both = raw[:2 * pages * P * Hk * D].view(2, P, pages, Hk, D).transpose(1, 2)   # slot-major pool
        return both[0], both[1]

    k, v = views()
    k.copy_(s.cache.k_codes.view(torch.int8))
    v.copy_(s.cache.v_codes.view(torch.int8))
    other = dsd.ScaledKVCache.from_tensors(k.view(torch.float8_e4m3fn),
                                           v.view(torch.float8_e4m3fn), s.cache.k_scales.clone(), s.cache.v_scales.clone())
    counts = new or [1, 1]
    T = sum(counts)
    offs = offsets_of(torch, counts) if new else None
    rot = dsd.RotaryTable.from_base(200, 64)
    x = [torch.randn(T, h, 64, device="cuda").bfloat16() * 2 for h in (2, 2, 8)]
    before = raw.clone()
    outs = []
    for c in (s.cache, other):
        q = c.append(x[0], x[1], s.d_table, s.d_lens, offs, rotary=rot, q=x[2])
        outs.append((q, *c.attend(q, s.d_table, s.d_lens, offs, return_lse=True)))
        c.check()
    assert torch.equal(outs[0][0], outs[1][0])
    for c in "kv":
        assert torch.equal(getattr(s.cache, c + "_codes").view(torch.int8), {"k": k, "v": v}[c])
        assert torch.equal(getattr(s.cache, c + "_scales"), getattr(other, c + "_scales"))
    # nothing outside the views was written
    mine = torch.zeros_like(raw, dtype=torch.bool)
    for y in (k, v):
        mine.as_strided(y.shape, y.stride(), y.storage_offset()).fill_(True)
    assert torch.equal(raw[~mine], before[~mine])
    # the paths differ in rounding only: both within the bound of the exact result
    at = 0
    s.pool.codes = {n: getattr(s.cache, n + "_codes").view(torch.int8).cpu().numpy().view(np.uint8) for n in "kv"}
    s.pool.scales = {n: getattr(s.cache, n + "_scales").cpu().numpy() for n in "kv"}
    for b, n in enumerate(counts):
        y = f32(outs[0][0][at:at + n])
        want, wl = o.attend(s.pool, y, s.table[b], s.lens[b], 0.125)
        to, tl = tolerance(y, s.pool, s.table[b], s.lens[b], 0.125, want, wl, "bf16", 4)
        for _, out, lse in outs:
            close(f32(out[at:at + n]).astype(np.float64), want, to)
            close(f32(lse[at:at + n]).astype(np.float64), wl, tl)
        at += n


def test_empty_tables_and_batches(torch, dsd):
    """A page table without columns, a batch without requests, a call without queries."""
    cache = dsd.ScaledKVCache(4, 16, 2, 64)
    none = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 64, device="cuda").half()
    out, lse = cache.attend(q, none, lens, return_lse=True)
    assert not out.any() and bool((lse == -float("inf")).all())
    out = cache.attend_pages(q, none, lens, torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert not out.any()
    assert cache.attend(q[:0], none[:0], lens[:0]).shape == (0, 4, 64)
    assert cache.append(q[:0, :2], q[:0, :2], none[:0], lens[:0]) is None
    cache.check()
    cache.append(q[:, :2], q[:, :2], none, lens + 1)      # a token but no page
    assert not cache.k_codes.view(torch.int8).any()
    with pytest.raises(dsd.OutOfRange):
        cache.check()


def test_large_batches_take_the_general_plan(torch, dsd):
    """More than 128 requests, and ragged queries with empty requests between."""
    rng = np.random.default_rng(5)
    for B, ragged in ((300, False), (200, True)):
        lens = rng.integers(0, 90, B).tolist()
        s = Setup(torch, dsd, "int8", lens, 64, 2, 16, seed=B)
        new = rng.integers(0, 4, B).tolist() if ragged else [1] * B
        q = torch.randn(sum(new), 4, 64, device="cuda").half()
        out = s.cache.attend(q, s.d_table, s.d_lens, offsets_of(torch, new) if ragged else None)
        s.cache.check()
        at = 0
        for b, n in enumerate(new):
            x = f32(q[at:at + n])
            if n:
                want, wl = o.attend(s.pool, x, s.table[b], lens[b], 0.125)
                to, _ = tolerance(x, s.pool, s.table[b], lens[b], 0.125, want, wl, "f16", 2)
                close(f32(out[at:at + n]).astype(np.float64), want, to)
            at += n


def test_negative_and_zero_logit_scale(torch, dsd):
    s = Setup(torch, dsd, "fp8", [300, 40], 128, 2, 16, seed=41)
    for n in ([1, 1], [30, 20]):
        q = torch.randn(sum(n), 8, 128, device="cuda").bfloat16()
        for scale in (-0.1, 0.0, 0.5):
            out, lse = s.cache.attend(q, s.d_table, s.d_lens, offsets_of(torch, n), scale=scale, return_lse=True)
            at = 0
            for b, m in enumerate(n):
                x = f32(q[at:at + m])
                want, wl = o.attend(s.pool, x, s.table[b], s.lens[b], scale)
                to, tl = tolerance(x, s.pool, s.table[b], s.lens[b], scale, want, wl, "bf16", 4)
                close(f32(out[at:at + m]).astype(np.float64), want, to)
                close(f32(lse[at:at + m]).astype(np.float64), wl, tl)
                at += m


def test_first_call_inside_a_capture(dsd, tmp_path):
    """A process whose first append and attend are captured, then replayed."""
    import subprocess
    import sys
    from conftest import PKG_NAME, ROOT
    code = f"""
import importlib, sys
sys.path.insert(0, {ROOT!r})
import torch
dsd = importlib.import_module({PKG_NAME!r})
cache = dsd.ScaledKVCache(8, 16, 2, 64)
table = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
x = torch.randn(2, 2, 64, device="cuda").bfloat16()
q = torch.randn(2, 8, 64, device="cuda").bfloat16()
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    cache.append(x, x, table, lens)
    out = cache.attend(q, table, lens)
g.replay()
torch.cuda.synchronize()
want = cache.attend(q, table, lens)
assert torch.equal(out, want) and out.isfinite().all()
cache.check()
print("ok")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "ok" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("fmt,dtype,D,H,Hk,P", [("fp8", "bf16", 128, 8, 2, 16), ("int8", "f32", 64, 2, 2, 32),
                                                ("fp8", "f16", 96, 4, 1, 256), ("int8", "bf16", 72, 4, 2, 6)])
def test_attend_pages(torch, dsd, fmt, dtype, D, H, Hk, P):
    s = Setup(torch, dsd, fmt, [P * 9, P * 3, P], D, Hk, P, seed=P)
    rng = np.random.default_rng(1)
    counts = rng.integers(0, P + 1, s.pool.pages).astype(np.int32)
    counts[s.table[1, :3]] = 0                       # a request whose pages hold nothing
    counts[s.table[0, 2]] = P + 5                    # more than a page can hold
    lists = np.full((4, 8), 10 ** 6, np.int32)
    held = [8, 3, 1, 0]
    lists[0] = rng.permutation(s.table[0, :9])[:8]
    lists[1, :3], lists[2, 0] = s.table[1, :3], s.table[2, 0]
    dt = getattr(torch, TYPES[dtype])
    q = torch.randn(4, H, D, device="cuda").to(dt)
    out, lse = s.cache.attend_pages(q, torch.from_numpy(lists).cuda(), torch.tensor(held, dtype=torch.int32, device="cuda"),
                                    torch.from_numpy(counts).cuda(), return_lse=True)
    s.cache.check()
    for b in range(4):
        x = f32(q[b:b + 1])
        want, wl = o.attend_pages(s.pool, x, lists[b, :held[b]], counts, D ** -0.5)
        to, tl = tolerance(x, s.pool, lists[b, :held[b]], held[b] * P, D ** -0.5, want, wl, dtype, H // Hk)
        close(f32(lse[b:b + 1]).astype(np.float64), wl, tl)
        close(f32(out[b:b + 1]).astype(np.float64), want, to)
    assert not out[1].any() and bool((lse[1] == -float("inf")).all())


@pytest.mark.parametrize("D", [128, 72])
def test_rows_that_see_nothing_and_rows_left_alone(torch, dsd, D):
    """Empty requests, more queries than tokens, rows behind the last request."""
    lens, new = [0, 5, 300, 0, 2], [2, 9, 0, 0, 3]
    s = Setup(torch, dsd, "fp8", lens, D, 2, 8, seed=11)
    T = sum(new)
    q = torch.randn(T + 4, 4, D, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    got, lse = s.cache.attend(q, s.d_table, s.d_lens, offsets_of(torch, new), out=out, return_lse=True)
    assert got.data_ptr() == out.data_ptr()
    assert bool((out[T:] == 7).all())
    at = 0
    for b, n in enumerate(new):
        if n:
            x = f32(q[at:at + n])
            want, wl = o.attend(s.pool, x, s.table[b], lens[b], D ** -0.5)
            to, tl = tolerance(x, s.pool, s.table[b], lens[b], D ** -0.5, want, wl, "bf16", 2)
            close(f32(out[at:at + n]).astype(np.float64), want, to)
            close(f32(lse[at:at + n]).astype(np.float64), wl, tl)
        at += n
    s.cache.check()
    none = s.cache.attend(q[:0], s.d_table, s.d_lens, offsets_of(torch, [0] * 5))
    assert none.shape == (0, 4, D)


@pytest.mark.parametrize("D,P", [(128, 16), (72, 6)])
def test_masked_places_may_hold_anything(torch, dsd, D, P):
    """NaN codes and NaN or infinite scales behind a request's tokens, before its window and after a
    query's own place leave its row alone; a NaN that a row does see makes the row NaN."""
    lens, new = [100, 45], [4, 3]
    s = Setup(torch, dsd, "fp8", lens, D, 2, P, bt=1, seed=12)
    clean = o.Pool("fp8", s.pool.codes, s.pool.scales)
    q = torch.randn(7, 4, D, device="cuda").bfloat16()

    def spoil(b, place, codes=True):
        page, slot = int(s.table[b, place // P]), place % P
        for c, sc in ((s.cache.k_codes, s.cache.k_scales), (s.cache.v_codes, s.cache.v_scales)):
            if codes:
                c.view(torch.int8)[page, slot] = 127
            else:
                sc[page, :, slot] = float("inf") if place % 2 else float("nan")

    table = s.table.copy()
    free = next(p for p in range(s.pool.pages) if p not in s.table)
    for slot in range(P):                        # a page behind the request's
        s.cache.v_codes.view(torch.int8)[free, slot] = 127
    for b, n in enumerate(lens):
        table[b, -(-n // P)] = free
        for place in range(n, -(-n // P) * P):
            spoil(b, place, codes=place % 3 > 0)
    spoil(0, 99)                                 # the last token: only the last query sees it
    spoil(1, 2), spoil(1, 3, codes=False)        # before every window of 30
    out, lse = s.cache.attend(q, torch.from_numpy(table).cuda(), s.d_lens, offsets_of(torch, new), window=30, return_lse=True)
    at = 0
    for b, n in enumerate(new):
        x = f32(q[at:at + n])
        want, wl = o.attend(clean, x, s.table[b], lens[b], D ** -0.5, True, 30)
        to, tl = tolerance(x, clean, s.table[b], lens[b], D ** -0.5, want, wl, "bf16", 2)
        rows = n - 1 if b == 0 else n
        close(f32(out[at:at + rows]).astype(np.float64), want[:rows], to[:rows])
        close(f32(lse[at:at + rows]).astype(np.float64), wl[:rows], tl[:rows])
        at += n
    assert bool(out[3].isnan().all()) and bool(lse[3].isnan().all())


def test_scales_of_every_size(torch, dsd):
    """Zero, tiny and huge value scales in one row: each contribution keeps its share, and the sum its value."""
    lens = [64]
    for fmt in ("fp8", "int8"):
        s = Setup(torch, dsd, fmt, lens, 128, 1, 8, seed=13)
        v = s.pool.scales["v"]
        ids = s.table[0, :8]
        v[ids, 0, 0] = np.float32([0, 1e-30, 1e-20, 1e-3, 1, 3e4, 0, 1e4])
        s.cache.v_scales.copy_(torch.from_numpy(v))
        q = torch.randn(1, 2, 128, device="cuda") * 4
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, return_lse=True)
        want, wl = o.attend(s.pool, f32(q), s.table[0], 64, 128 ** -0.5)
        to, tl = tolerance(f32(q), s.pool, s.table[0], 64, 128 ** -0.5, want, wl, "f32", 2)
        close(f32(out).astype(np.float64), want, to)
        close(f32(lse).astype(np.float64), wl, tl)
        v[ids, 0, 0] = 0
        s.cache.v_scales.copy_(torch.from_numpy(v))
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, return_lse=True)
        assert not out.any()
        close(f32(lse).astype(np.float64), wl, tl)


def test_scales_of_every_size_with_many_rows(torch, dsd):
    """The same with 16 query rows a key head: zero scales, and values that grow and shrink by 2^12 between pages,
    so that the reference of the weights moves from tile to tile."""
    for fmt, dtype in (("fp8", "bf16"), ("int8", "f16")):
        s = Setup(torch, dsd, fmt, [700, 130], 64, 2, 16, seed=17)
        v = s.pool.scales["v"]
        for b, n in enumerate(s.lens):
            for i in range(-(-n // 16)):
                v[s.table[b, i]] = np.float32(0.0 if i % 7 == 6 else 2.0 ** (12 * ((i * 5) % 3 - 1)) * 1.3)
        s.cache.v_scales.copy_(torch.from_numpy(v))
        q = (torch.randn(2, 32, 64, device="cuda") * 3).to(getattr(torch, TYPES[dtype]))
        out, lse = s.cache.attend(q, s.d_table, s.d_lens, return_lse=True)
        for b, n in enumerate(s.lens):
            x = f32(q[b:b + 1])
            want, wl = o.attend(s.pool, x, s.table[b], n, 0.125)
            to, tl = tolerance(x, s.pool, s.table[b], n, 0.125, want, wl, dtype, 16)
            got = f32(out[b:b + 1]).astype(np.float64)
            if dtype == "f16":
                # the largest fp16 is 65504 and half a step behind it rounds to infinity: what is
                # beyond 65520 by more than its bound has to be infinite, what may be, may
                assert (np.isinf(got) | (np.abs(want) - to < 65520)).all()
                over = np.isinf(got) & (np.abs(want) + to >= 65520) & (np.sign(got) == np.sign(want))
                got = np.where(over, want, got)
            close(got, want, to)
            close(f32(lse[b:b + 1]).astype(np.float64), wl, tl)
        s.cache.v_scales.zero_()
        out, lse2 = s.cache.attend(q, s.d_table, s.d_lens, return_lse=True)
        assert not out.any()
        for b in range(2):
            x = f32(q[b:b + 1])
            want, wl = o.attend(s.pool, x, s.table[b], s.lens[b], 0.125)
            close(f32(lse2[b:b + 1]).astype(np.float64), wl,
                  tolerance(x, s.pool, s.table[b], s.lens[b], 0.125, want, wl, dtype, 16)[1])


def test_threads_with_their_own_streams(torch, dsd):
    """Calls from several host threads at once, each on its stream, into one cache's reader."""
    import threading
    s = Setup(torch, dsd, "int8", [900, 300, 50], 128, 2, 16, seed=23)
    q = torch.randn(3, 8, 128, device="cuda").bfloat16()
    want = s.cache.attend(q, s.d_table, s.d_lens)
    torch.cuda.synchronize()
    bad = []

    def work():
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(20):
                if not torch.equal(s.cache.attend(q, s.d_table, s.d_lens), want):
                    bad.append(1)
        st.synchronize()

    ts = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not bad


def test_bad_pages_and_lengths_are_masked(torch, dsd):
    for D, P in ((128, 16), (72, 6)):
        s = Setup(torch, dsd, "int8", [100, 60, 30], D, 2, P, seed=14)
        q = torch.randn(3, 4, D, device="cuda").half()
        good = s.cache.attend(q, s.d_table, s.d_lens)
        table = s.table.copy()
        table[1, 1] = s.pool.pages
        table[1, 2] = -7
        out = s.cache.attend(q, torch.from_numpy(table).cuda(), s.d_lens)
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
        x = f32(q[1:2])
        keep = np.array([i // P not in (1, 2) for i in range(60)])
        for h in range(2):
            k, v = (s.pool.rows(n, s.table[1], np.arange(60), h) for n in "kv")
            w, _ = o.attend_rows(x[0, 2 * h:2 * h + 2], k, v, D ** -0.5, keep)
            assert np.abs(f32(out[1, 2 * h:2 * h + 2]) - w).max() < 2.0 ** -11 * np.abs(w).max() + 2.0 ** -9 * np.abs(v).max()
        with pytest.raises(dsd.OutOfRange):
            s.cache.check()
        lens = torch.tensor([-3, 10 ** 9, 30], dtype=torch.int32, device="cuda")
        wide = s.table.copy()
        wide[1] = s.table[1, 0]
        out = s.cache.attend(q, torch.from_numpy(wide).cuda(), lens)
        assert not out[0].any() and torch.equal(out[2], good[2])
        with pytest.raises(dsd.OutOfRange):
            s.cache.check()


def test_cache_beyond_32_bits(torch, dsd):
    """Codes whose byte offsets pass 2^31 and 2^32."""
    pages, P, Hk, D = 300000, 16, 8, 128
    cache = dsd.ScaledKVCache(pages, P, Hk, D)
    lens = [40, 33]
    ids = np.array([[pages - 1, 131073, 2], [140000, 262145, pages - 2]], np.int32)
    table = torch.from_numpy(ids).cuda()
    k, v = (torch.randn(73, Hk, D, device="cuda").bfloat16() for _ in range(2))
    offs, d_lens = offsets_of(torch, lens), torch.tensor(lens, dtype=torch.int32, device="cuda")
    cache.append(k, v, table, d_lens, offs)
    q = torch.randn(2, 8, D, device="cuda").bfloat16()
    out = cache.attend(q, table, d_lens)
    small = dsd.ScaledKVCache(6, P, Hk, D)
    near = torch.arange(6, dtype=torch.int32, device="cuda").reshape(2, 3)
    small.append(k, v, near, d_lens, offs)
    assert torch.equal(out, small.attend(q, near, d_lens))
    assert torch.equal(cache.k_codes.view(torch.int8)[ids[0, 0]], small.k_codes.view(torch.int8)[0])
    cache.check()


def test_a_serving_run_together(torch, dsd):
    """Prompt, chunk, decode steps and page lists over one cache, as a server calls them; the decode step is
    captured once and replayed while the lengths grow, on a stream of its own."""
    fmt, D, Hk, H, P = "fp8", 128, 2, 8, 16
    total = [90, 41, 150]
    s = Setup(torch, dsd, fmt, total, D, Hk, P, seed=20, spare=4)
    rot = dsd.RotaryTable.from_base(256, D)
    cos, sin = rot.cos.cpu().numpy(), rot.sin.cpu().numpy()
    gen = torch.Generator("cuda").manual_seed(4)
    rows = lambda n, h: torch.randn(n, h, D, device="cuda", generator=gen).bfloat16()  # noqa: E731
    start = [60, 1, 100]
    counts = torch.zeros(s.cache.num_pages, dtype=torch.int32, device="cuda")

    def check(q, out, lens, new):
        at = 0
        for b, n in enumerate(new):
            x = f32(q[at:at + n])
            want, wl = o.attend(s.pool, x, s.table[b], lens[b], D ** -0.5)
            to, _ = tolerance(x, s.pool, s.table[b], lens[b], D ** -0.5, want, wl, "bf16", H // Hk)
            close(f32(out[at:at + n]).astype(np.float64), want, to)
            at += n

    def mirror(k, v, lens, new):
        at = 0
        for b, n in enumerate(new):
            s.pool.append("k", f32(k[at:at + n]), s.table[b], lens[b], cos, sin)
            s.pool.append("v", f32(v[at:at + n]), s.table[b], lens[b])
            at += n

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for lens, new in ((start, start), ([80, 31, 130], [20, 30, 30])):      # prompts, then a chunk of each
            k, v, q = rows(sum(new), Hk), rows(sum(new), Hk), rows(sum(new), H)
            d_lens, offs = torch.tensor(lens, dtype=torch.int32, device="cuda"), offsets_of(torch, new)
            q = s.cache.append(k, v, s.d_table, d_lens, offs, rotary=rot, q=q, token_counts=counts)
            out = s.cache.attend(q, s.d_table, d_lens, offs)
            mirror(k, v, lens, new)
            check(q, out, lens, new)
        lens = [80, 31, 130]
        d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        k, v, q = rows(3, Hk), rows(3, Hk), rows(3, H)
        out = torch.zeros_like(q)

        def step():
            d_lens.add_(1)
            turned = s.cache.append(k, v, s.d_table, d_lens, rotary=rot, q=q, token_counts=counts)
            s.cache.attend(turned, s.d_table, d_lens, out=out)
            return turned

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            turned = step()
        for i in range(10):
            for t in (k, v, q):
                t.copy_(rows(3, t.shape[1]))
            graph.replay()
            lens = [n + 1 for n in lens]
            mirror(k, v, lens, [1, 1, 1])
            check(turned, out, lens, [1, 1, 1])
        # the same tokens as a page list, in another order
        need = [-(-n // P) for n in lens]
        lists = np.zeros((3, max(need)), np.int32)
        for b, n in enumerate(need):
            lists[b, :n] = s.table[b, :n][::-1]
        got = s.cache.attend_pages(turned, torch.from_numpy(lists).cuda(), torch.tensor(need, dtype=torch.int32, device="cuda"),
                                   counts)
        check(turned, got, lens, [1, 1, 1])
    stream.synchronize()
    s.same(torch)
    s.cache.check()


def test_two_streams_at_once(torch, dsd):
    """Calls that run at the same time share nothing."""
    s = Setup(torch, dsd, "fp8", [3000, 2500], 128, 2, 16, seed=21)
    q = [torch.randn(2, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [s.cache.attend(x, s.d_table, s.d_lens) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(s.cache.attend(q[i], s.d_table, s.d_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_refusals(torch, dsd):
    s = Setup(torch, dsd, "fp8", [20, 20], 64, 2, 16, seed=22)
    c = s.cache
    k = torch.randn(2, 2, 64, device="cuda").half()
    q = torch.randn(2, 4, 64, device="cuda").half()
    bad = dsd.InvalidArgument
    for call in (
            lambda: c.append(k, k.float(), s.d_table, s.d_lens),
            lambda: c.append(k[:1], k[:1], s.d_table, s.d_lens),
            lambda: c.append(k, k[:, :1], s.d_table, s.d_lens),
            lambda: c.append(k.cpu(), k, s.d_table, s.d_lens),
            lambda: c.append(k, k, s.d_table.long(), s.d_lens),
            lambda: c.append(k, k, s.d_table[:1], s.d_lens),
            lambda: c.append(k, k, s.d_table, s.d_lens.long()),
            lambda: c.append(k, k, s.d_table, s.d_lens, rotary=dsd.RotaryTable.from_base(4, 66)),
            lambda: c.append(k, k, s.d_table, s.d_lens, q_out=q),
            lambda: c.append(k.transpose(1, 2), k, s.d_table, s.d_lens),
            lambda: c.attend(q[:, :3], s.d_table, s.d_lens),
            lambda: c.attend(q[:1], s.d_table, s.d_lens),
            lambda: c.attend(q, s.d_table, s.d_lens, window=-1),
            lambda: c.attend(q, s.d_table, s.d_lens, scale=float("nan")),
            lambda: c.attend(q, s.d_table, s.d_lens, out=q.float()),
            lambda: c.attend(q, s.d_table, s.d_lens, s.d_lens),
            lambda: c.attend_pages(q, s.d_table, s.d_lens, s.d_lens),
            lambda: dsd.ScaledKVCache(4, 16, 2, 60),
            lambda: dsd.ScaledKVCache(4, 16, 2, 64, block_tokens=5),
            lambda: dsd.ScaledKVCache(4, 16, 2, 64, kv_format=dsd.KV_F32),
            lambda: dsd.RotaryTable.from_base(4, 7),
    ):
        with pytest.raises(bad):
            call()
    c.check()
