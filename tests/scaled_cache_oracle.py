"""Plain 64-bit implementation of the scaled 8-bit paged cache, one request, head and token at a time."""
import numpy as np

QMAX = {"fp8": 448.0, "int8": 127.0}


def e4m3_table():
    """Value of every e4m3 code: sign, exponent (bias 7), 3 mantissa bits; S.1111.111 is NaN."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if e == 15 and m == 7:
            v = np.nan
        out[c] = -v if c & 128 else v
    return out


TABLE = e4m3_table()
_POSITIVE = TABLE[:127]   # codes 0..126 ascend to 448


def encode(x, fmt):
    """Codes (uint8) of fp32 values: nearest, ties to even, saturating; NaN -> NaN code (e4m3) or 0 (int8)."""
    x = np.asarray(x, np.float32)
    if fmt == "int8":
        r = np.where(np.isnan(x), 0.0, np.clip(np.rint(x.astype(np.float64)), -127, 127))
        return r.astype(np.int8).view(np.uint8)
    a = np.abs(np.where(np.isnan(x), 0, x).astype(np.float64))
    hi = np.clip(np.searchsorted(_POSITIVE, a, side="left"), 1, 126)
    lo = hi - 1
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = np.where(a >= 448, 126, code)
    code = np.where(np.isnan(x), 127, code) | (np.signbit(x).astype(np.int64) << 7)
    return code.astype(np.uint8)


def decode(codes, fmt):
    codes = np.asarray(codes)
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else TABLE[codes.view(np.uint8)]


def rotate(x, cos, sin, interleaved):
    """fp32 products, each rounded, as the operator defines them."""
    x = np.asarray(x, np.float32)
    y = x.copy()
    if cos is None:
        return y
    h = len(cos)
    ia = 2 * np.arange(h) if interleaved else np.arange(h)
    ib = ia + 1 if interleaved else ia + h
    a, b = x[..., ia], x[..., ib]
    with np.errstate(invalid="ignore"):
        y[..., ia] = a * cos - b * sin
        y[..., ib] = b * cos + a * sin
    return y


class Pool:
    """codes: {"k","v"} uint8 [pages][P][Hk][D]; scales: {"k","v"} float32 [pages][Hk][P/bt]."""

    def __init__(self, fmt, codes, scales):
        self.fmt = fmt
        self.codes = {n: c.copy() for n, c in codes.items()}
        self.scales = {n: s.copy() for n, s in scales.items()}
        self.pages, self.P, self.Hk, self.D = codes["k"].shape
        self.bt = self.P // scales["k"].shape[2]

    def append(self, name, x, page_row, length, cos=None, sin=None, interleaved=False, positions=None):
        """x [n][Hk][D] float32 are the last n of `length` tokens; returns the rotated rows."""
        f32 = np.float32
        n, qmax = len(x), QMAX[self.fmt]
        start = length - n
        y = np.empty(x.shape, f32)
        for j in range(n):
            pos = start + j if positions is None else positions[j]
            y[j] = rotate(x[j], None if cos is None else cos[pos], None if sin is None else sin[pos], interleaved)
        for blk in range(start // self.bt, -(-length // self.bt)):
            a, b = max(start, blk * self.bt), min(length, (blk + 1) * self.bt)
            held, first = a - blk * self.bt, blk * self.bt % self.P
            page = page_row[blk * self.bt // self.P]
            for h in range(self.Hk):
                new = y[a - start:b - start, h]
                fin = np.abs(new[np.isfinite(new)])
                amax = fin.max() if fin.size else f32(0)
                fresh = f32(0) if amax < 2.0 ** -100 else f32(amax * f32(1.0 / qmax))
                old = self.scales[name][page, h, first // self.bt]
                scale = max(old, fresh) if held else fresh
                with np.errstate(all="ignore"):
                    inv = f32(1) / scale if scale > 0 else f32(0)
                    if held and scale > old:
                        c = self.codes[name][page, first:first + held, h]
                        c[:] = encode(decode(c, self.fmt).astype(f32) * f32(old * inv), self.fmt)
                    self.codes[name][page, first + held:first + held + b - a, h] = encode(new * inv, self.fmt)
                self.scales[name][page, h, first // self.bt] = scale
        return y

    def values(self, name, page, slot, h):
        return decode(self.codes[name][page, slot, h], self.fmt) * np.float64(self.scales[name][page, h, slot // self.bt])

    def rows(self, name, page_row, places, h):
        """Values of a request's tokens at `places`, [len][D]."""
        places = np.asarray(places, np.int64)
        page, slot = np.asarray(page_row, np.int64)[places // self.P], places % self.P
        with np.errstate(invalid="ignore"):
            return decode(self.codes[name][page, slot, h], self.fmt) * self.scales[name][page, h, slot // self.bt].astype(np.float64)[:, None]


def attend_rows(q, k, v, scale, seen):
    """q [G][D], k/v [L][D] in 64 bits, seen [L] bool -> out [G][D], lse [G]; nothing seen: zeros, -inf."""
    if not seen.any():
        return np.zeros((len(q), v.shape[1])), np.full(len(q), -np.inf)
    z = np.asarray(q, np.float64) @ k[seen].T * scale
    m = z.max(1, keepdims=True)
    p = np.exp(z - m)
    return p @ v[seen] / p.sum(1, keepdims=True), (m + np.log(p.sum(1, keepdims=True)))[:, 0]


def attend(pool, q, page_row, length, scale, causal=True, window=0):
    """q [n][H][D] are the request's last n tokens' queries."""
    n, H, _ = q.shape
    G = H // pool.Hk
    t = np.arange(length)
    out, lse = np.zeros(q.shape), np.full((n, H), -np.inf)
    for h in range(pool.Hk):
        k, v = pool.rows("k", page_row, t, h), pool.rows("v", page_row, t, h)
        for j in range(n):
            pos = length - n + j
            seen = np.ones(length, bool)
            if causal:
                seen &= t <= pos
            if window:
                seen &= t > pos - window
            hs = slice(h * G, (h + 1) * G)
            out[j, hs], lse[j, hs] = attend_rows(q[j, hs], k, v, scale, seen)
    return out, lse


def attend_pages(pool, q, pages, counts, scale):
    """q [n][H][D]; every query sees the tokens of the listed pages."""
    n, H, _ = q.shape
    G = H // pool.Hk
    spots = [(p, s) for p in pages for s in range(min(counts[p], pool.P))]
    out, lse = np.zeros(q.shape), np.full((n, H), -np.inf)
    for h in range(pool.Hk):
        k = np.array([pool.values("k", p, s, h) for p, s in spots]).reshape(len(spots), pool.D)
        v = np.array([pool.values("v", p, s, h) for p, s in spots]).reshape(len(spots), pool.D)
        for j in range(n):
            hs = slice(h * G, (h + 1) * G)
            out[j, hs], lse[j, hs] = attend_rows(q[j, hs], k, v, scale, np.ones(len(spots), bool))
    return out, lse
