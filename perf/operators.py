"""Cases and plain forms of the scaled 8-bit paged cache: append (with the position rotation) and attention.

A cache is a pool of pages; a page holds `page` token rows of `kv_heads` x `head_dim` 8-bit codes for keys and for
values, and one fp32 scale for each head and each run of `block` tokens of the page.  A stored value is code * scale.
"""
import importlib
import math
import random

import torch

own = False

QMAX = {"fp8": 448.0, "int8": 127.0}
CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -100
BASE = 500000.0


def _attend(name, **kw):
    c = dict(name=name, op="attend", fmt="fp8", dtype="bf16", heads=32, kv_heads=8, dim=128, page=16, block=16, batch=1, lo=1024,
             hi=1024, q_lo=1, q_hi=1, window=0, layout="token")
    c.update(kw)
    return c


def _append(name, **kw):
    c = dict(name=name, op="append", fmt="fp8", dtype="bf16", heads=32, kv_heads=8, dim=128, page=16, block=16, batch=1, lo=1024,
             hi=1024, q_lo=1, q_hi=1, rotary=128, pairs="half", layout="token")
    c.update(kw)
    return c


def listed():
    return [
        # one user's decode step: nothing but latency
        _attend("attend one short"),
        # one user far into a long document: one request has to fill the machine
        _attend("attend one long", lo=120001, hi=120001, page=64, block=64, layout="head"),
        # batch of 16, 32 heads with a key head each, fp32 queries: the framework's own decode shape with int8 pages
        _attend("attend 16 mha int8 f32", fmt="int8", dtype="f32", kv_heads=32, batch=16, lo=512, hi=2048),
        # continuous serving: ragged batch in its usual range
        _attend("attend 64 ragged", batch=64, lo=1024, hi=4096),
        # the long-context batch: 64 requests of 16k to 32k tokens
        _attend("attend 64 long", batch=64, lo=16384, hi=32768, page=32, block=32),
        # int8, fp16, sliding window, small heads with a finer scale
        _attend("attend window int8 f16", fmt="int8", dtype="f16", heads=16, kv_heads=4, dim=64, page=32, block=8, batch=48, lo=500,
                hi=12000, window=4096),
        # verification of drafted tokens: a few queries for each request
        _attend("attend drafts", batch=24, lo=700, hi=9000, q_lo=2, q_hi=7),
        # prompt chunks that attend over what is there already
        _attend("attend chunks", batch=3, lo=5000, hi=9000, q_lo=300, q_hi=700),
        # sparse decode: 64 selected pages of 16 tokens of each of 64 requests, every head its own keys
        _attend("attend selected pages", op="attend_pages", kv_heads=32, batch=64, lo=16384, hi=32768, pages=64),
        # the decode step's append: one token for each request, queries rotated in the same call
        _append("append decode", batch=64, lo=1024, hi=4096),
        # prompts of ordinary length, some joining what is there
        _append("append prompts int8", fmt="int8", batch=7, lo=600, hi=5000, q_lo=100, q_hi=2000, page=32, block=32, layout="head"),
        # the largest: long prompts, fp16, half of each head rotated in neighbouring pairs, int8
        _append("append long f16", fmt="fp8", dtype="f16", batch=4, lo=15000, hi=33000, q_lo=12000, q_hi=16000, rotary=64, pairs="next",
                page=64, block=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    page = rng.choice([8, 16, 16, 32, 64, 128])
    block = rng.choice([b for b in (1, 4, 8, 16, 32, 64, 128) if page % b == 0 and b >= page // 8])
    heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 2), (8, 8), (64, 8), (24, 8), (28, 4), (12, 1)])
    shape = dict(fmt=rng.choice(["fp8", "int8"]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=heads, kv_heads=kv_heads,
                 dim=rng.choice([128, 128, 64, 96, 80]), page=page, block=block, layout=rng.choice(["token", "head"]))
    kind = rng.choice(["decode", "decode", "chunk", "drafts", "pages", "append one", "append many"])
    if kind in ("decode", "drafts"):
        batch = _log(rng, 1, 96)
        hi = _log(rng, 16, min(60000, 262144 // batch))
        q_hi = 1 if kind == "decode" else rng.randint(2, 8)
        c = _attend("", batch=batch, lo=max(1, _log(rng, 1, hi)), hi=hi, q_lo=1, q_hi=min(q_hi, hi), window=rng.choice([0, 0, 100, 1024]), **shape)
    elif kind == "chunk":
        batch, q_hi = _log(rng, 1, 8), _log(rng, 16, 512)
        hi = q_hi + _log(rng, 1, 8000 // batch)
        c = _attend("", batch=batch, lo=_log(rng, 1, hi), hi=hi, q_lo=_log(rng, 1, q_hi), q_hi=q_hi, window=rng.choice([0, 0, 333]), **shape)
    elif kind == "pages":
        batch = _log(rng, 1, 64)
        c = _attend("", op="attend_pages", batch=batch, lo=page * 2, hi=_log(rng, page * 4, 8000), pages=_log(rng, 1, 64), **shape)
    else:
        batch = _log(rng, 1, 128) if kind == "append one" else _log(rng, 1, 16)
        q_hi = 1 if kind == "append one" else _log(rng, 2, 32768 // batch)
        hi = q_hi + _log(rng, 1, 8000)
        c = _append("", batch=batch, lo=_log(rng, 1, hi), hi=hi, q_lo=_log(rng, 1, q_hi), q_hi=q_hi, pairs=rng.choice(["half", "next"]), **shape)
        c["rotary"] = rng.choice([c["dim"], c["dim"] // 2, 16])
        c["heads"] = rng.choice([0, heads])
    del c["name"]
    c["lo"] = min(c["lo"], c["hi"])
    return c


def _lengths(c):
    """Lengths of the requests and of their new tokens: they belong to the case, so that its work is known."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    lens = [rng.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]
    new = [min(n, rng.randint(c["q_lo"], c["q_hi"])) for n in lens]
    return lens, new


def _codes(c, gen, pages):
    """Codes and scales as a cache holds them: rounded normal values under the scale of their block's largest."""
    P, Hk, D = c["page"], c["kv_heads"], c["dim"]
    shape = (pages, P, Hk, D) if c["layout"] == "token" else (pages, Hk, P, D)
    codes = torch.empty(shape, dtype=CODES[c["fmt"]], device="cuda")
    step = max(1, (1 << 27) // (P * Hk * D))
    for a in range(0, pages, step):
        x = torch.randn(codes[a:a + step].shape, generator=gen, device="cuda", dtype=torch.float32)
        if c["fmt"] == "int8":
            codes[a:a + step] = (x * 34).round_().clamp_(-127, 127).to(torch.int8)
        else:
            codes[a:a + step] = (x * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)
    scales = torch.rand((pages, Hk, P // c["block"]), generator=gen, device="cuda") * 1.5 + 0.5
    return codes if c["layout"] == "token" else codes.transpose(1, 2), scales * (3.7 / QMAX[c["fmt"]])


def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    lens, new = _lengths(c)
    B, P, D, H, Hk = c["batch"], c["page"], c["dim"], c["heads"], c["kv_heads"]
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=host, dtype=torch.int64).to(torch.int32)
    table = torch.zeros((B, max(need)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = {"c": c, "lens": torch.tensor(lens, dtype=torch.int32).cuda(), "new": new, "scale": 1.0 / math.sqrt(D)}
    s["k_codes"], s["k_scales"] = _codes(c, gen, pages)
    s["v_codes"], s["v_scales"] = _codes(c, gen, pages)
    T, dt = sum(new), TYPES[c["dtype"]]
    s["offsets"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    if c["op"] == "append":
        # a layer's fused projection: queries, keys and values of a token in one row
        rows = torch.randn((T, H + 2 * Hk, D), generator=gen, device="cuda").to(dt)
        s["q"], s["k"], s["v"] = rows[:, :H], rows[:, H:H + Hk], rows[:, H + Hk:]
        places = c["hi"] + 1
        rd = c["rotary"]
        angle = torch.arange(places, dtype=torch.float64, device="cuda")[:, None] * BASE ** (-torch.arange(0, rd, 2, dtype=torch.float64, device="cuda") / rd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = torch.randn((T, H, D), generator=gen, device="cuda").to(dt)
    if c["op"] == "attend_pages":
        pick = torch.zeros((B, min(c["pages"], max(need))), dtype=torch.int32)
        counts = torch.zeros(pages, dtype=torch.int32)
        for b, n in enumerate(need):
            k = min(c["pages"], n)
            counts[table[b, :n].long()] = P
            counts[table[b, n - 1].long()] = lens[b] - (n - 1) * P
            pick[b, :k] = table[b, :n][torch.randperm(n, generator=host)[:k]]
        s["counts"], table = counts.cuda(), pick
        s["listed"] = torch.tensor([min(c["pages"], n) for n in need], dtype=torch.int32).cuda()
    s["table"] = table.cuda()
    s["ones"] = max(new) == 1
    if own:
        pkg = importlib.import_module("15-618_dynamic_sparse_decode_b200")
        s["cache"] = pkg.ScaledKVCache.from_tensors(s["k_codes"], s["v_codes"], s["k_scales"], s["v_scales"])
        if c["op"] == "append":
            s["rotary"] = pkg.RotaryTable(s["cos"], s["sin"], interleaved=c["pairs"] == "next")
    return s


def _run_own(s):
    c, cache, offsets = s["c"], s["cache"], None if s["ones"] else s["offsets"]
    if c["op"] == "append":
        q = cache.append(s["k"], s["v"], s["table"], s["lens"], token_offsets=offsets, rotary=s["rotary"], q=s["q"] if c["heads"] else None)
        return {"q": q, "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if c["op"] == "attend_pages":
        out, lse = cache.attend_pages(s["q"], s["table"], s["listed"], s["counts"], scale=s["scale"], return_lse=True)
    else:
        out, lse = cache.attend(s["q"], s["table"], s["lens"], q_offsets=offsets, scale=s["scale"], window=c["window"], return_lse=True)
    return {"out": out, "lse": lse}


def _values(codes, scales, table, block):
    """Values of the listed pages: [batch, kv_heads, listed * page, dim] in fp32."""
    t = table.long()
    x = codes[t].float() * scales[t].repeat_interleave(block, -1).transpose(2, 3)[..., None]
    return x.flatten(1, 2).transpose(1, 2)


def _visible(s, Q):
    """Which listed tokens each query sees: [batch, Q, listed * page]."""
    c, P = s["c"], s["c"]["page"]
    L = s["table"].shape[1] * P
    t = torch.arange(L, device="cuda")
    if c["op"] == "attend_pages":
        held = s["counts"][s["table"].long()] * (torch.arange(s["table"].shape[1], device="cuda") < s["listed"][:, None])
        return ((t % P) < held.repeat_interleave(P, 1))[:, None, :]
    new = s["offsets"].diff()
    last = (s["lens"] - new)[:, None] + torch.arange(Q, device="cuda")  # the place of each query
    seen = t <= last[..., None]
    return seen & (t > last[..., None] - c["window"]) if c["window"] else seen


def _attend_plain(s):
    c = s["c"]
    B, H, Hk, D, Q = c["batch"], c["heads"], c["kv_heads"], c["dim"], max(s["new"])
    G = H // Hk
    rows = s["q"].shape[0]
    req = torch.repeat_interleave(torch.arange(B, device="cuda"), s["offsets"].diff().long(), output_size=rows)
    place = torch.arange(rows, device="cuda") - s["offsets"].long()[req]
    q = torch.zeros((B, Q, H, D), device="cuda")
    q[req, place] = s["q"].float()
    q = q.reshape(B, Q, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, Q * G, D)
    logits = (q @ _values(s["k_codes"], s["k_scales"], s["table"], c["block"]).transpose(2, 3)) * s["scale"]
    seen = _visible(s, Q).repeat_interleave(G, 1)[:, None]
    logits = logits.masked_fill(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min(-3e38)
    p = (logits - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p @ _values(s["v_codes"], s["v_scales"], s["table"], c["block"])) / total.clamp_min(1e-38)
    out = out.reshape(B, Hk, Q, G, D).permute(0, 2, 1, 3, 4).reshape(B, Q, H, D)
    lse = (top + total.log()).reshape(B, Hk, Q, G).permute(0, 2, 1, 3).reshape(B, Q, H)
    return {"out": out[req, place].to(s["q"].dtype), "lse": lse[req, place]}


def _rotate(x, cos, sin, pairs, rd):
    x = x.float()
    y = x.clone()
    a, b = (x[..., :rd // 2], x[..., rd // 2:rd]) if pairs == "half" else (x[..., 0:rd:2], x[..., 1:rd:2])
    c, s = cos[:, None], sin[:, None]
    lo, hi = a * c - b * s, b * c + a * s
    if pairs == "half":
        y[..., :rd // 2], y[..., rd // 2:rd] = lo, hi
    else:
        y[..., 0:rd:2], y[..., 1:rd:2] = lo, hi
    return y


def _round(x, fmt):
    q = QMAX[fmt]
    return (x.round() if fmt == "int8" else x).clamp(-q, q).to(CODES[fmt])


def _store(codes, scales, x, where, tail, c):
    """New rows x [T, kv_heads, dim] go to their places; a block that holds older tokens takes the larger scale."""
    fmt, P, bt = c["fmt"], c["page"], c["block"]
    pages, slots = where
    largest = torch.zeros_like(scales)
    at = pages * (P // bt) + slots // bt
    flat = largest.transpose(1, 2).reshape(-1, c["kv_heads"]).contiguous()
    flat.scatter_reduce_(0, at[:, None].expand(-1, c["kv_heads"]), x.abs().amax(-1), "amax")
    largest = flat.reshape(scales.shape[0], -1, c["kv_heads"]).transpose(1, 2)
    fresh = largest * (1.0 / QMAX[fmt])
    fresh = torch.where(largest < TINY, torch.zeros_like(fresh), fresh)
    # the one block of each request that can hold older tokens
    page, slot, held = tail
    first = slot - held
    old = scales[page, :, first // bt]
    both = torch.where(held[:, None] > 0, torch.maximum(old, fresh[page, :, first // bt]), fresh[page, :, first // bt])
    inverse = torch.where(both > 0, 1.0 / both, torch.zeros_like(both))
    t = torch.arange(bt, device="cuda")
    spot = (first[:, None] + t).clamp_max(P - 1)
    before = codes[page[:, None], spot].float()
    moved = _round(before * (old * inverse)[:, None, :, None], fmt).float()
    keep = (both > old) & (held > 0)[:, None]
    after = torch.where(keep[:, None, :, None] & (t < held[:, None])[..., None, None], moved, before)
    touched = torch.zeros(flat.shape[0], dtype=torch.bool, device="cuda").index_fill_(0, at, True).reshape(scales.shape[0], 1, -1)
    scales.copy_(torch.where(touched, fresh, scales))
    scales[page, :, first // bt] = both
    codes[page[:, None], spot] = after.to(codes.dtype)
    r = scales[pages, :, slots // bt]
    codes[pages, slots] = _round(x * torch.where(r > 0, 1.0 / r, torch.zeros_like(r))[..., None], fmt)


def _append_plain(s):
    c, P, bt = s["c"], s["c"]["page"], s["c"]["block"]
    rows = s["k"].shape[0]
    new = s["offsets"].diff().long()
    req = torch.repeat_interleave(torch.arange(c["batch"], device="cuda"), new, output_size=rows)
    start = s["lens"].long() - new
    place = start[req] + torch.arange(rows, device="cuda") - s["offsets"].long()[req]
    where = s["table"][req, place // P].long(), place % P
    tail = s["table"][torch.arange(c["batch"], device="cuda"), start // P].long(), start % P, start % P % bt
    cos, sin = s["cos"][place], s["sin"][place]
    _store(s["k_codes"], s["k_scales"], _rotate(s["k"], cos, sin, c["pairs"], c["rotary"]), where, tail, c)
    _store(s["v_codes"], s["v_scales"], s["v"].float(), where, tail, c)
    q = _rotate(s["q"], cos, sin, c["pairs"], c["rotary"]).to(s["q"].dtype) if c["heads"] else None
    return {"q": q, "k_codes": s["k_codes"], "v_codes": s["v_codes"], "k_scales": s["k_scales"], "v_scales": s["v_scales"]}


def run(state):
    if own:
        return _run_own(state)
    return _append_plain(state) if state["c"]["op"] == "append" else _attend_plain(state)


def work(case):
    c = dict(case)
    lens, new = _lengths(c)
    Hk, H, D, P = c["kv_heads"], c["heads"], c["dim"], c["page"]
    elem = 4 if c["dtype"] == "f32" else 2
    T = sum(new)
    if c["op"] == "append":
        moved = T * (2 * Hk + H) * D * elem + T * (2 * Hk * D + H * D * elem) + T * c["rotary"] * 4
        scales = sum(-(-n // c["block"]) for n in new) * Hk * 8
        return {"bytes": moved + scales + 8 * c["batch"], "flops": T * ((Hk + H) * 3 * c["rotary"] + 4 * Hk * D)}
    if c["op"] == "attend_pages":
        seen = [min(n, P * min(c["pages"], -(-n // P))) for n in lens]
        pairs = read = sum(seen)
    else:
        span = [min(n, c["window"] + m - 1) if c["window"] else n for n, m in zip(lens, new)]
        read = sum(span)
        pairs = sum(min(n - m + j + 1, c["window"] or n) for n, m in zip(lens, new) for j in range(m))
    moved = read * Hk * 2 * (D + 4.0 / c["block"]) + 4.0 * read / P + T * H * (2 * D * elem + 4)
    return {"bytes": moved, "flops": 4.0 * D * H * pairs}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "append":
        return _append_exact(s)
    lens, new, P, G = s["lens"].tolist(), s["new"], c["page"], c["heads"] // c["kv_heads"]
    out, lse, at = [], [], 0
    for b, m in enumerate(new):
        q = s["q"][at:at + m].double()
        at += m
        if c["op"] == "attend_pages":
            ids = s["table"][b, :int(s["listed"][b])].long()
            live = (torch.arange(P, device="cuda") < s["counts"][ids][:, None]).reshape(-1)
        else:
            ids = s["table"][b, :-(-lens[b] // P)].long()
            live = torch.arange(len(ids) * P, device="cuda") < lens[b]
        o, l = [], []
        for h in range(c["kv_heads"]):
            k = (s["k_codes"][ids, :, h].double() * s["k_scales"][ids, h].double().repeat_interleave(c["block"], 1)[..., None]).flatten(0, 1)[live]
            v = (s["v_codes"][ids, :, h].double() * s["v_scales"][ids, h].double().repeat_interleave(c["block"], 1)[..., None]).flatten(0, 1)[live]
            z = torch.einsum("mgd,td->mgt", q[:, h * G:(h + 1) * G], k) * s["scale"]
            if c["op"] == "attend":
                t, place = torch.arange(lens[b], device="cuda"), lens[b] - m + torch.arange(m, device="cuda")[:, None]
                hidden = t > place
                if c["window"]:
                    hidden = hidden | (t <= place - c["window"])
                z = z.masked_fill(hidden[:, None], -math.inf)
            o.append(torch.softmax(z, -1) @ v)
            l.append(torch.logsumexp(z, -1))
        out.append(torch.cat(o, 1))
        lse.append(torch.cat(l, 1))
    return {"out": torch.cat(out), "lse": torch.cat(lse)}


def _append_exact(s):
    """Rotated queries and the scales in 64 bits, angles from their definition; codes next to a border have no value of their own."""
    c, P, bt, rd = s["c"], s["c"]["page"], s["c"]["block"], s["c"]["rotary"]
    lens, table = s["lens"].tolist(), s["table"].tolist()
    freq = BASE ** (-2.0 * torch.arange(rd // 2, dtype=torch.float64, device="cuda") / rd)

    def turn(x, places):
        unit = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), places.double()[:, None] * freq)[:, None]
        x = x.double()
        head = torch.view_as_complex(torch.stack((x[..., :rd // 2], x[..., rd // 2:rd]), -1)) if c["pairs"] == "half" else torch.view_as_complex(x[..., :rd].unflatten(-1, (-1, 2)).contiguous())
        y = torch.view_as_real(head * unit)
        y = torch.cat((y[..., 0], y[..., 1]), -1) if c["pairs"] == "half" else y.flatten(-2)
        return torch.cat((y, x[..., rd:]), -1)

    scales = {"k": s["k_scales"].double(), "v": s["v_scales"].double()}
    qs, at = [], 0
    for b, m in enumerate(s["new"]):
        start = lens[b] - m
        places = torch.arange(start, lens[b], device="cuda")
        if c["heads"]:
            qs.append(turn(s["q"][at:at + m], places))
        lead = start % bt
        for name, x in (("k", turn(s["k"][at:at + m], places)), ("v", s["v"][at:at + m].double())):
            size = x.abs().amax(-1)
            size = torch.nn.functional.pad(size, (0, 0, lead, -(lead + m) % bt)).unflatten(0, (-1, bt)).amax(1) / QMAX[c["fmt"]]
            run = torch.arange(size.shape[0], device="cuda") + start // bt
            page = torch.tensor(table[b], device="cuda")[run * bt // P]
            if lead:
                size[0] = torch.maximum(size[0], scales[name][page[0], :, run[0] % (P // bt)])
            scales[name][page, :, run % (P // bt)] = size
        at += m
    return {"q": torch.cat(qs) if qs else None, "k_codes": None, "v_codes": None, "k_scales": scales["k"], "v_scales": scales["v"]}
