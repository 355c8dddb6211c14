"""The scaled 8-bit paged cache at its edges (GPU): what a row does not see, or barely sees, leaves it alone.

attend: with p the exact softmax over the tokens that a row SEES and v = code * vs their values,
  |out - exact| <= half a step of the output type * |exact| + (logits + exp + piece) * sum p |v|
                   + spot * max(p vs) * sum |code| + half of the output type's least step
logits, exp and piece as in test_scaled_cache_gpu.py, taken over the tokens seen.  spot: a weight p vs
is kept to an absolute step of the row's largest.  Narrow kernel, largest in [1, 2): int8 2^-20, e4m3
2^-25.  Wide kernel: the largest is at least 2^-3 in fp16, whose least step is 2^-24: 2^-22.  Taken: 2^-19.
"""
import numpy as np
import pytest

import scaled_cache_oracle as o
from test_scaled_cache_gpu import Setup, TYPES, close, f32, offsets_of, torch  # noqa: F401  (torch is a fixture)

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -25}   # the values here stay above 2^-100
SPOT = 2.0 ** -19


def exact_and_bounds(s, b, q, n, causal=True, window=0, dtype="bf16"):
    """q [n][H][D] of request b: exact out and lse, and the bounds above, from the tokens each row sees."""
    pool, L, D = s.pool, s.lens[b], s.D
    H = q.shape[1]
    G, scale = H // pool.Hk, D ** -0.5
    out, lse = np.zeros(q.shape), np.full((n, H), -np.inf)
    tol_o, tol_l = np.zeros(q.shape), np.zeros((n, H))
    t = np.arange(L)
    page, slot = s.table[b][t // s.P].astype(np.int64), t % s.P
    for h in range(pool.Hk):
        code = o.decode(pool.codes["v"][page, slot, h], pool.fmt)
        vs = pool.scales["v"][page, h, slot // pool.bt].astype(np.float64)
        k = pool.rows("k", s.table[b], t, h)
        for j in range(n):
            pos = L - n + j
            seen = (t <= pos if causal else t >= 0) & ((t > pos - window) if window else True)
            if not seen.any():
                continue
            for g in range(h * G, (h + 1) * G):
                x = q[j, g].astype(np.float64)
                z = k[seen] @ x * scale
                p = np.exp(z - z.max())
                total = p.sum()
                p /= total
                v = code[seen] * vs[seen][:, None]
                out[j, g], lse[j, g] = p @ v, z.max() + np.log(total)
                zerr = 2 * (D + 8) * 2.0 ** -24 * (np.abs(k[seen]) @ np.abs(x)).max() * scale
                tol_o[j, g] = (HALF[dtype] * np.abs(out[j, g]) + (zerr + 2.0 ** -20 + 2.0 ** -11) * (p @ np.abs(v))
                               + SPOT * (p * vs[seen]).max() * np.abs(code[seen]).sum(0) + LEAST[dtype])
                tol_l[j, g] = zerr + 2.0 ** -20 * max(1.0, abs(lse[j, g]))
    return out, lse, tol_o, tol_l


def upload(torch, s):
    for n in "kv":
        getattr(s.cache, n + "_scales").copy_(torch.from_numpy(s.pool.scales[n]))
        getattr(s.cache, n + "_codes").view(torch.int8).copy_(torch.from_numpy(s.pool.codes[n].view(np.int8)))


def queries(torch, s, H, counts, dtype):
    gen = torch.Generator("cuda").manual_seed(7)
    q = torch.randn(sum(counts), H, s.D, device="cuda", generator=gen).to(getattr(torch, TYPES[dtype]))
    q[..., 0] = 8.0          # element 0 of a key moves its logits by that element, 8 / sqrt(64)
    return q


def attend(torch, s, H, new, dtype, check=True, causal=True, window=0):
    counts = new or [1] * len(s.lens)
    q = queries(torch, s, H, counts, dtype)
    out, lse = s.cache.attend(q, s.d_table, s.d_lens, offsets_of(torch, counts) if new else None, causal=causal, window=window,
                              return_lse=True)
    s.cache.check()
    at = 0
    for b, n in enumerate(counts if check else []):
        want, wl, to, tl = exact_and_bounds(s, b, f32(q[at:at + n]), n, causal, window, dtype)
        got = f32(out[at:at + n]).astype(np.float64)
        if dtype == "f16":   # behind the largest fp16 there is no value to compare
            got = np.where(np.abs(want) < 65000, got, want)
        close(f32(lse[at:at + n]).astype(np.float64), wl, tl)
        close(got, want, to)
        at += n
    return out, lse


KINDS = [("fp8", "bf16"), ("int8", "bf16"), ("int8", "f16"), ("fp8", "f32")]


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("H,new", [(8, [33, 17]), (2, [150, 40])])
@pytest.mark.parametrize("power", [16, 24, 40])
def test_scales_that_a_row_must_not_see(torch, dsd, fmt, dtype, H, new, power):
    """Later tokens of the same prompt with larger value scales: the rows before them stay as they are, bit for bit."""
    s = Setup(torch, dsd, fmt, [300, 140], 64, 2, 16, bt=1, seed=51, spread=0.3)
    ordinary = attend(torch, s, H, new, dtype, check=False)
    for b, n in enumerate(new):
        for t in range(s.lens[b] - n // 2, s.lens[b]):   # seen by the later half of the queries only
            s.pool.scales["v"][s.table[b, t // 16], :, t % 16] *= np.float32(2.0 ** power)
    upload(torch, s)
    got = attend(torch, s, H, new, dtype)
    at = 0
    for n in new:
        rows = slice(at, at + n - n // 2)
        assert torch.equal(got[0][rows], ordinary[0][rows]) and torch.equal(got[1][rows], ordinary[1][rows])
        at += n


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("H,new", [(8, None), (32, None), (8, [33, 17]), (2, [150, 40])])
@pytest.mark.parametrize("power,drop", [(16, 200), (24, 200), (40, 200), (24, 12), (40, 25), (-40, 0)])
@pytest.mark.parametrize("where", ["first tile", "all over"])
def test_scales_of_tokens_that_weigh_nothing(torch, dsd, fmt, dtype, H, new, power, drop, where):
    """Tokens that a row sees, with a far larger (or smaller) value scale and a logit lower by `drop`."""
    s = Setup(torch, dsd, fmt, [400, 140], 64, 2, 16, bt=1, seed=52, spread=0.3)
    for b, n in enumerate(s.lens):
        for t in range(3, 100 if where == "first tile" else n, 9):
            page, slot = s.table[b, t // 16], t % 16
            s.pool.scales["v"][page, :, slot] *= np.float32(2.0 ** power)
            s.pool.codes["k"][page, slot, :, :] = 0
            s.pool.codes["k"][page, slot, :, 0] = o.encode(np.float32(-o.QMAX[fmt]), fmt)
            s.pool.scales["k"][page, :, slot] = np.float32(drop / o.QMAX[fmt])
    upload(torch, s)
    attend(torch, s, H, new, dtype)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("H,new", [(8, None), (32, None), (2, [150, 40])])
def test_tokens_with_scale_zero_that_weigh_most(torch, dsd, fmt, dtype, H, new):
    """A token whose values are all zero takes most of the weight: the others keep their bits."""
    s = Setup(torch, dsd, fmt, [400, 140], 64, 2, 16, bt=1, seed=53, spread=0.3)
    for b, n in enumerate(s.lens):
        for t in range(0, n, 50):
            page, slot = s.table[b, t // 16], t % 16
            s.pool.scales["v"][page, :, slot] = 0
            s.pool.codes["k"][page, slot, :, :] = 0
            s.pool.codes["k"][page, slot, :, 0] = o.encode(np.float32(o.QMAX[fmt]), fmt)
            s.pool.scales["k"][page, :, slot] = np.float32(25 / o.QMAX[fmt])
    upload(torch, s)
    attend(torch, s, H, new, dtype)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8])
def test_every_group_of_heads_fits_an_SM_as_planned(torch, dsd, fmt, dtype, rows):
    """The first call checks that each kernel fits on an SM as often as the work is cut for; every shape then runs, with
    more requests than one round of CTAs holds."""
    s = Setup(torch, dsd, fmt, [130, 700, 5, 260], 128, 3, 32, bt=8, seed=54, spread=0.3)
    attend(torch, s, 3 * rows, None, dtype)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("H,new", [(18, None), (24, None), (32, None), (34, None), (36, None), (50, None), (8, [4, 4]), (8, [4, 5]),
                                   (8, [1, 7]), (8, [1, 30])])
def test_rows_on_both_sides_of_the_kernels_limit(torch, dsd, fmt, dtype, H, new):
    """9 query rows a key head and more: several narrow units, or one wide one; pages of different scales."""
    s = Setup(torch, dsd, fmt, [400, 140], 64, 2, 16, bt=4, seed=55, spread=1.0)
    attend(torch, s, H, new, dtype)


@pytest.mark.parametrize("fmt,dtype", KINDS)
@pytest.mark.parametrize("power,drop", [(16, 200), (24, 12), (40, 25), (-40, 0)])
def test_scales_of_tokens_that_weigh_nothing_for_large_groups(torch, dsd, fmt, dtype, power, drop):
    """One query each, 32 heads a key head."""
    s = Setup(torch, dsd, fmt, [400, 140], 64, 2, 16, bt=1, seed=56, spread=0.3)
    for b, n in enumerate(s.lens):
        for t in range(3, n, 9):
            page, slot = s.table[b, t // 16], t % 16
            s.pool.scales["v"][page, :, slot] *= np.float32(2.0 ** power)
            s.pool.codes["k"][page, slot, :, :] = 0
            s.pool.codes["k"][page, slot, :, 0] = o.encode(np.float32(-o.QMAX[fmt]), fmt)
            s.pool.scales["k"][page, :, slot] = np.float32(drop / o.QMAX[fmt])
    upload(torch, s)
    attend(torch, s, 64, None, dtype)


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
@pytest.mark.parametrize("D,bt,dtype", [(64, 16, "bf16"), (256, 128, "f16"), (72, 4, "f32"), (128, 16, "f32")])
def test_append_infinities_into_blocks_of_zeros(torch, dsd, fmt, D, bt, dtype):
    """Infinities saturate in a block without any finite value above 2^-100 too, and read as 0 there; NaN stays NaN
    (e4m3) or 0 (int8).  When the block's scale grows they become 0."""
    s = Setup(torch, dsd, fmt, [bt + 1, 1], D, 2, bt, seed=57)
    n = [bt - 1, 1]
    k, v = (torch.zeros(bt, 2, D, device="cuda", dtype=getattr(torch, TYPES[dtype])) for _ in range(2))
    inf, top = float("inf"), 126 if fmt == "fp8" else 127
    k[0, 0, 3], k[0, 1, 4], k[1, 0, 5] = inf, -inf, float("nan")
    v[bt - 1] = inf                       # the one token of the other request: nothing finite
    v[bt - 1, 1, ::2] = -inf
    if dtype != "f16":
        k[2, 0, 1] = -1e-35               # below 2^-100
    lens = torch.tensor(n, dtype=torch.int32, device="cuda")
    s.cache.append(k, v, s.d_table, lens, offsets_of(torch, n))
    minus = 128 + 126 if fmt == "fp8" else 256 - 127
    codes = {x: getattr(s.cache, x + "_codes").view(torch.int8).cpu().numpy().view(np.uint8) for x in "kv"}
    scales = {x: getattr(s.cache, x + "_scales").cpu().numpy() for x in "kv"}
    a, b = s.table[0, 0], s.table[1, 0]
    want = np.zeros((bt - 1, 2, D), np.uint8)
    want[0, 0, 3], want[0, 1, 4] = top, minus
    if fmt == "fp8":
        want[1, 0, 5] = 127
        if dtype != "f16":
            want[2, 0, 1] = 128           # -0
    assert np.array_equal(codes["k"][a, :bt - 1], want) and not scales["k"][a].any()
    want = np.full((2, D), top, np.uint8)
    want[1, ::2] = minus
    assert np.array_equal(codes["v"][b, 0], want) and not scales["v"][b].any()
    # one token more, of ordinary size: the older codes are rounded to its scale
    one = torch.ones(1, 2, D, device="cuda", dtype=k.dtype)
    s.cache.append(one, one, s.d_table[:1], lens[:1] + 1)
    got = s.cache.k_codes.view(torch.int8).cpu().numpy().view(np.uint8)[a]
    assert (got[bt - 1] == top).all() and (got[:bt - 1][want_nan_free(fmt, got[:bt - 1])] & 127 == 0).all()
    assert np.array_equal(s.cache.k_scales.cpu().numpy()[a], np.full((2, 1), np.float32(1 / o.QMAX[fmt]), np.float32))
    s.cache.check()


def want_nan_free(fmt, codes):
    return codes & 127 != 127 if fmt == "fp8" else np.ones(codes.shape, bool)


@pytest.mark.parametrize("lens,offsets,good", [
    ([20, 20, 20], [0, 20, 15, 35], None),                  # the middle request's offsets descend
    ([20, 20, 20], [0, 20, 20, 10], [0]),                   # the last one's
    ([20, -2 ** 31, 20], [0, 20, 40, 60], [0, 2]),          # no length at all
    ([20, -1, 20], [0, 20, 40, 60], [0, 2]),
    ([20, 19, 20], [0, 20, 40, 60], [0, 2]),                # fewer tokens than new ones
    ([20, 20, 20], [0, 20, 40, 2 ** 31 - 1], [0, 1]),       # rows behind the arrays
    ([20, 20, 20], [-2 ** 31, 20, 40, 60], [1, 2]),
])
@pytest.mark.parametrize("bt", [1, 16])
def test_append_reports_lengths_and_offsets_that_fit_nothing(torch, dsd, lens, offsets, good, bt):
    """The request is left out and its status bit set; the others are stored (where no later offset descends)."""
    s = Setup(torch, dsd, "int8", [20, 20, 20], 64, 2, 16, bt=bt, seed=58)
    k, v = (torch.randn(60, 2, 64, device="cuda").bfloat16() for _ in range(2))
    s.cache.append(k, v, s.d_table, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                   torch.tensor(offsets, dtype=torch.int32, device="cuda"))
    for b in good or []:
        for name, x in (("k", k), ("v", v)):
            s.pool.append(name, f32(x[offsets[b]:offsets[b + 1]]), s.table[b], 20)
    if good:
        s.same(torch)
    with pytest.raises(dsd.OutOfRange, match="seq_lens or offsets"):
        s.cache.check()
    s.cache.check()


def test_check_waits_for_every_stream_and_names_all_it_met(torch, dsd):
    """Bits set by a call that still waits on another stream, several at once, each reported once."""
    s = Setup(torch, dsd, "fp8", [20, 20], 64, 2, 16, seed=59)
    k, v = (torch.randn(2, 2, 64, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    rot = dsd.RotaryTable.from_base(10, 64)
    table = s.d_table.clone()
    table[0, 1] = -1
    s.cache.append(k, v, s.d_table, s.d_lens)
    s.cache.attend(q, s.d_table, s.d_lens)
    s.cache.check()
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)                           # a tenth of a second
        s.cache.append(k, v, table, s.d_lens, rotary=rot)        # place 19 of a table with 10; no such page
    with pytest.raises(dsd.OutOfRange, match="(?s)page.*rotation"):
        s.cache.check()
    s.cache.check()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)
        s.cache.attend(q, table, s.d_lens)
    with pytest.raises(dsd.OutOfRange, match="page"):
        s.cache.check()
    s.cache.check()


def test_refusals_of_shapes_and_numbers(torch, dsd):
    """What cannot be an argument is refused as one, not by an error of the binding's inside."""
    s = Setup(torch, dsd, "fp8", [20, 20], 64, 2, 16, seed=60)
    c = s.cache
    k = torch.randn(2, 2, 64, device="cuda").half()
    q = torch.randn(2, 4, 64, device="cuda").half()
    one = torch.tensor(1, dtype=torch.int32, device="cuda")
    codes, scales = torch.zeros(2, 16, 2, 12, dtype=torch.int8, device="cuda"), torch.ones(2, 2, 1, device="cuda")
    for call in (
            lambda: c.attend(q, s.d_table, s.d_lens, scale=1e300),
            lambda: c.attend(q, s.d_table, s.d_lens, window=2.0),
            lambda: c.attend(q, s.d_table, s.d_lens, window=-2 ** 40),
            lambda: c.attend(q, s.d_table, one),
            lambda: c.attend(one, s.d_table, s.d_lens),
            lambda: c.attend(q, one, s.d_lens),
            lambda: c.attend(q, s.d_table, s.d_lens, out=torch.empty_like(q)[:, :1].expand(2, 4, 64)),
            lambda: c.append(k, k, s.d_table, one),
            lambda: c.append(one, k, s.d_table, s.d_lens),
            lambda: c.append(k, k, s.d_table, s.d_lens, q=one),
            lambda: c.append(k, k, s.d_table, s.d_lens, q=q, q_out=q[:1].expand(2, 4, 64)),
            lambda: dsd.ScaledKVCache(1, 512, 2, 64),
            lambda: dsd.ScaledKVCache(1, 8192, 2, 64, block_tokens=16),
            lambda: dsd.ScaledKVCache(1, 16, 129, 64),
            lambda: dsd.ScaledKVCache.from_tensors(codes, codes, scales, scales),
    ):
        with pytest.raises(dsd.InvalidArgument):
            call()
    c.check()


@pytest.mark.parametrize("fmt,dtype", [("fp8", "bf16"), ("int8", "bf16"), ("fp8", "f32"), ("int8", "f32")])
@pytest.mark.parametrize("D,H,new", [(64, 2, None), (64, 8, None), (64, 64, None), (64, 2, [150, 40]), (72, 8, [9, 20])])
@pytest.mark.parametrize("kind", ["least", "both ends", "largest late"])
def test_value_scales_at_the_ends_of_their_range(torch, dsd, fmt, dtype, D, H, new, kind):
    """Scales of 0 and from 2^-64 to 2^36 keep outputs and the softmax sum, alone and together."""
    s = Setup(torch, dsd, fmt, [400, 140], D, 2, 16, bt=1, seed=61, spread=0.3)
    v = s.pool.scales["v"]
    v[:] = np.float32(2.0 ** -64)
    if kind == "both ends":
        v[::2, :, 1::5], v[1::2, :, 2::5], v[:, :, 3::7] = np.float32(2.0 ** 36), 1, 0
    elif kind == "largest late":
        for b, n in enumerate(s.lens):
            t = n - 45 if new else n - 1
            v[s.table[b, t // 16], :, t % 16] = np.float32(2.0 ** 36)
    upload(torch, s)
    attend(torch, s, H, new, dtype)


@pytest.mark.parametrize("fmt,dtype", [("fp8", "bf16"), ("int8", "f16")])
@pytest.mark.parametrize("D", [16, 32, 48, 112])
@pytest.mark.parametrize("P,bt", [(8, 2), (24, 3), (264, 33)])
def test_many_rows_at_other_head_dims_and_pages(torch, dsd, fmt, dtype, D, P, bt):
    s = Setup(torch, dsd, fmt, [310, 77], D, 2, P, bt=bt, seed=62, spread=0.5)
    attend(torch, s, 4, [70, 40], dtype, window=120)


@pytest.mark.parametrize("D,P", [(128, 16), (72, 6)])
def test_a_page_listed_twice_counts_twice(torch, dsd, D, P):
    s = Setup(torch, dsd, "fp8", [3 * P], D, 2, P, seed=63)
    a, b = int(s.table[0, 0]), int(s.table[0, 1])
    counts = np.full(s.pool.pages, P, np.int32)
    q = torch.randn(1, 4, D, device="cuda").bfloat16()

    def pages(ids):
        return s.cache.attend_pages(q, torch.tensor([ids], dtype=torch.int32, device="cuda"),
                                    torch.tensor([len(ids)], dtype=torch.int32, device="cuda"), torch.from_numpy(counts).cuda(),
                                    return_lse=True)

    out, lse = pages([a, b, a])
    want, wl = o.attend_pages(s.pool, f32(q), [a, b, a], counts, D ** -0.5)
    assert np.abs(f32(out) - want).max() <= 2.0 ** -8 * np.abs(want).max() + 2.0 ** -9 * np.abs(want).max()
    assert np.abs(f32(lse) - wl).max() <= 2.0 ** -16 * np.maximum(1, np.abs(wl)).max()
    s.cache.check()
