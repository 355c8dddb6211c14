"""Scaled 8-bit paged KV cache: append with the position rotation, attention (torch tensors).

The binding of ``dsd_scaled_append`` / ``dsd_scaled_attention``
(``include/dsd_b200.h``) for programs that keep their tensors in torch.  A
stored key or value is ``code * scale``: an e4m3 or int8 code under one fp32
scale for each page, key head and run of ``block_tokens`` tokens of a page.

For serving: results carry no gradient.  Every call runs on the current torch
stream of the cache's device, allocates only what it returns plus the
attention's workspace (from torch's allocator), never synchronises, and can be
captured into a CUDA graph.  What only the device
can see (page ids, lengths, positions) is checked there: see
:meth:`ScaledKVCache.check`.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch

from . import (DSD_EINVAL, DSD_ERANGE, DSD_ETIMEOUT, KV_FP8_SCALED, KV_I8_SCALED, DsdError, InvalidArgument, OutOfRange,
               ScaledAttentionArgs, ScaledCacheDesc, _check, load_library)

_FORMATS = {torch.float8_e4m3fn: KV_FP8_SCALED, torch.int8: KV_I8_SCALED}
_CODES = {v: k for k, v in _FORMATS.items()}
# dsd_scaled_append_args and dsd_scaled_attention_args: one pack costs a tenth of setting the fields
_APPEND_ARGS = struct.Struct("@4i2P4q3Pq3P4i2P4q2P")
_ATTENTION_ARGS = struct.Struct("@4i3P4q3PqPifiiPqP")
_UNFIT = (struct.error, OverflowError)   # pack: a number of another kind, or beyond its field
_raw_stream = torch._C._cuda_getCurrentRawStream   # the current stream's handle, without a Stream object
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_TIMEOUT = 8
_BAD = ((_TIMEOUT, "a device-side wait exceeded its budget"),
        (1, "a page id is outside the pool or a page is beyond the page-table row"),
        (2, "a position is outside the rotation table"),
        (4, "seq_lens or offsets that fit no token"))


def _invalid(message: str):
    raise InvalidArgument(int(DSD_EINVAL), message)


class RotaryTable:
    """Cosines and sines of the position rotation, fp32 ``[positions, rotary_dim / 2]``.

    ``interleaved`` turns neighbouring elements (2i, 2i+1); otherwise the pairs
    are (i, i + rotary_dim / 2).  Elements from ``rotary_dim`` on stay.
    """

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False):
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1 or cos.shape[1] < 1:
            _invalid("cos and sin must have the same shape [positions, rotary_dim / 2]")
        if cos.dtype != torch.float32 or sin.dtype != torch.float32:
            _invalid("cos and sin must be float32")
        if not (cos.is_contiguous() and sin.is_contiguous()) or cos.device != sin.device:
            _invalid("cos and sin must be contiguous and on one device")
        self.cos, self.sin, self.interleaved = cos, sin, bool(interleaved)

    @classmethod
    def from_base(cls, positions: int, rotary_dim: int, base: float = 10000.0, interleaved: bool = False,
                  device="cuda") -> "RotaryTable":
        """Angles position * base^(-2i / rotary_dim), computed in 64 bits."""
        if rotary_dim < 2 or rotary_dim % 2 or positions < 1:
            _invalid("rotary_dim must be even and positive, positions positive")
        i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
        angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rotary_dim)
        return cls(angle.cos().float(), angle.sin().float(), interleaved)


class ScaledKVCache:
    """A pool of pages of 8-bit keys and values with their scales.

    ``k_codes`` / ``v_codes``: float8_e4m3fn or int8 ``[num_pages, page_size,
    num_kv_heads, head_dim]``, any positive strides with adjacent elements (a
    head-major pool is its transposed view).  ``k_scales`` / ``v_scales``: float32
    ``[num_pages, num_kv_heads, page_size / block_tokens]``, contiguous.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 kv_format: int = KV_FP8_SCALED, block_tokens: int | None = None, head_major: bool = False,
                 device="cuda"):
        if kv_format not in _CODES:
            _invalid("kv_format must be KV_FP8_SCALED or KV_I8_SCALED")
        block = page_size if block_tokens is None else block_tokens
        if min(num_pages, page_size, num_kv_heads, head_dim, block) < 1 or page_size % block:
            _invalid("sizes must be positive and block_tokens must divide page_size")
        if head_dim % 8 or head_dim > 256:
            _invalid("head_dim must be a multiple of 8 in [8, 256]")
        shape = (num_pages, num_kv_heads, page_size, head_dim) if head_major else (
            num_pages, page_size, num_kv_heads, head_dim)
        codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(_CODES[kv_format]) for _ in range(2)]
        if head_major:
            codes = [c.transpose(1, 2) for c in codes]
        scales = [torch.zeros((num_pages, num_kv_heads, page_size // block), device=device) for _ in range(2)]
        self._adopt(*codes, *scales)

    @classmethod
    def from_tensors(cls, k_codes, v_codes, k_scales, v_scales) -> "ScaledKVCache":
        """A cache over the caller's tensors (kept, not copied)."""
        self = cls.__new__(cls)
        self._adopt(k_codes, v_codes, k_scales, v_scales)
        return self

    def _adopt(self, k_codes, v_codes, k_scales, v_scales):
        if k_codes.dim() != 4 or k_codes.shape != v_codes.shape or k_codes.dtype != v_codes.dtype:
            _invalid("k_codes and v_codes must have one shape [num_pages, page_size, num_kv_heads, head_dim] and type")
        if k_codes.dtype not in _FORMATS:
            _invalid("codes must be float8_e4m3fn or int8")
        pages, page_size, heads, dim = k_codes.shape
        for c in (k_codes, v_codes):
            if dim > 1 and c.stride(3) != 1:
                _invalid("the elements of a code row must be adjacent")
            if any(n > 1 and s < 1 for n, s in zip(c.shape, c.stride())):
                _invalid("code strides must be positive")
        if k_scales.dim() != 3 or k_scales.shape != v_scales.shape or tuple(k_scales.shape[:2]) != (pages, heads):
            _invalid("scales must be [num_pages, num_kv_heads, page_size / block_tokens]")
        blocks = k_scales.shape[2]
        if blocks < 1 or page_size % blocks:
            _invalid("the number of scales per page must divide page_size")
        for s in (k_scales, v_scales):
            if s.dtype != torch.float32 or not s.is_contiguous():
                _invalid("scales must be contiguous float32")
        device = k_codes.device
        if device.type != "cuda" or any(t.device != device for t in (v_codes, k_scales, v_scales)):
            _invalid("codes and scales must be on one CUDA device")
        self.lib = load_library()
        self.device = device
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.num_pages, self.page_size, self.num_kv_heads, self.head_dim = pages, page_size, heads, dim
        self.block_tokens = page_size // blocks
        if dim % 8 or not 8 <= dim <= 256 or page_size > 4096 or self.block_tokens > 256 or heads > 128:
            _invalid("head_dim must be a multiple of 8 in [8, 256]; page_size at most 4096, block_tokens 256, num_kv_heads 128")
        self.kv_format = _FORMATS[k_codes.dtype]
        strides = lambda c: [max(1, s) for s in c.stride()[:3]]  # noqa: E731  (a dimension of one may have any)
        self._desc = ScaledCacheDesc(self.kv_format, pages, page_size, heads, dim, self.block_tokens,
                                     k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                     (ctypes.c_int64 * 3)(*strides(k_codes)), (ctypes.c_int64 * 3)(*strides(v_codes)))
        self._desc_at = ctypes.addressof(self._desc)
        self._workspace = {}
        self._index = device.index
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._status_at = self.status.data_ptr()

    # ---- checks
    def _ints(self, name, t, n=None):
        if t.dtype != torch.int32 or t.dim() != 1 or t.device != self.device or (t.numel() > 1 and t.stride(0) != 1):
            _invalid(f"{name} must be a contiguous int32 vector on {self.device}")
        if n is not None and t.shape[0] != n:
            _invalid(f"{name} must have {n} entries")
        return t.data_ptr()

    def _rows(self, name, t, dtype=None, shape=None):
        if t.dim() != 3 or t.device != self.device or t.dtype not in _TYPES or (
                t.shape[2] > 1 and t.stride(2) != 1):
            _invalid(f"{name} must be [rows, heads, head_dim] float32, bfloat16 or float16 on {self.device}, elements adjacent")
        if t.shape[2] != self.head_dim:
            _invalid(f"{name} must have head_dim {self.head_dim}")
        if dtype is not None and t.dtype != dtype:
            _invalid(f"{name} must be {dtype}")
        if shape is not None and tuple(t.shape) != tuple(shape):
            _invalid(f"{name} must be {tuple(shape)}")
        return t.data_ptr()

    def _table(self, table, batch):
        if table.dim() != 2 or table.dtype != torch.int32 or table.device != self.device or table.shape[0] != batch or (
                table.shape[1] > 1 and table.stride(1) != 1):
            _invalid(f"the page table must be int32 [{batch}, pages] on {self.device}, rows contiguous")
        return table.data_ptr(), table.stride(0) if batch > 1 else table.shape[1]

    def check(self) -> None:
        """Waits for the device, all its streams, and raises if a call since the last check met bad device data.

        The message names all that was met.  What a call that is launched meanwhile meets
        is raised here or by the next check.
        """
        torch.cuda.synchronize(self.device)
        taken = self.status.new_empty(1)
        _check(self.lib.dsd_scaled_take_status(self._index, self._status_at, taken.data_ptr(), _raw_stream(self._index)))
        bits = int(taken.item())
        if bits:
            message = "; ".join(text for bit, text in _BAD if bits & bit)
            if bits & _TIMEOUT:
                raise DsdError(DSD_ETIMEOUT, message)
            raise OutOfRange(DSD_ERANGE, message)

    # ---- operators
    def append(self, k, v, page_table, seq_lens, token_offsets=None, rotary: RotaryTable | None = None,
               positions=None, q=None, q_out=None, token_counts=None):
        """Writes the new tokens' keys and values; returns the rotated queries (or None).

        ``k`` / ``v`` ``[tokens, num_kv_heads, head_dim]`` and ``q`` ``[tokens, num_q_heads,
        head_dim]`` hold the requests' new tokens back to back: request b's are rows
        ``token_offsets[b] : token_offsets[b + 1]`` (None: one token for each request).
        ``seq_lens`` counts each request's tokens with the new ones; ``page_table`` ``[batch,
        pages]`` lists its pages.  ``rotary`` turns keys and queries by ``positions`` (None: the
        token's place in its request).  ``q_out`` may be ``q``; the rows of tokens that are left out (a
        bad position or length, behind the last request) keep what it held, and mean nothing in a fresh one.  ``token_counts`` ``[num_pages]``
        receives the tokens that the touched pages hold (what :meth:`attend_pages` reads).
        """
        lens = self._ints("seq_lens", seq_lens)
        batch, heads, dim = seq_lens.shape[0], self.num_kv_heads, self.head_dim
        tokens = k.shape[0] if k.dim() else 0
        kp = self._rows("k", k, None, (tokens, heads, dim))
        vp = self._rows("v", v, k.dtype, (tokens, heads, dim))
        table, stride = self._table(page_table, batch)
        offsets = None if token_offsets is None else self._ints("token_offsets", token_offsets, batch + 1)
        cos = sin = None
        places = turned = pairs = 0
        if rotary is not None:
            if rotary.cos.device != self.device:
                _invalid(f"the rotation table must be on {self.device}")
            cos, sin, pairs = rotary.cos.data_ptr(), rotary.sin.data_ptr(), rotary.interleaved
            places, half = rotary.cos.shape
            turned = 2 * half
        at = None if positions is None else self._ints("positions", positions, tokens)
        qp = op = None
        q_heads = 0
        q_stride = out_stride = (0, 0, 1)
        if q is not None:
            qp = self._rows("q", q, k.dtype)
            if q.shape[0] != tokens:
                _invalid("q must have a row for each token")
            if q_out is None:
                q_out = torch.empty_like(q)
                op = q_out.data_ptr()
            else:
                op = self._rows("q_out", q_out, q.dtype, q.shape)
            q_heads, q_stride, out_stride = q.shape[1], q.stride(), q_out.stride()
        elif q_out is not None:
            _invalid("q_out needs q")
        counts = None if token_counts is None else self._ints("token_counts", token_counts, self.num_pages)
        k_stride, v_stride = k.stride(), v.stride()
        try:
            args = _APPEND_ARGS.pack(
                _TYPES[k.dtype], batch, tokens, page_table.shape[1], kp or 0, vp or 0, k_stride[0], k_stride[1], v_stride[0],
                v_stride[1], offsets or 0, lens or 0, table or 0, stride, cos or 0, sin or 0, at or 0, places, turned, pairs,
                q_heads, qp or 0, op or 0, q_stride[0], q_stride[1], out_stride[0], out_stride[1], counts or 0, self._status_at)
        except _UNFIT as e:
            _invalid(f"a size does not fit: {e}")
        _check(self.lib.dsd_scaled_append(self._index, self._desc_at, args, _raw_stream(self._index)))
        return q_out

    def _attend(self, q, table, lens, q_offsets, counts, scale, causal, window, out, return_lse):
        lens_at = self._ints("lens", lens)
        qp = self._rows("q", q)
        batch, rows, heads = lens.shape[0], q.shape[0], q.shape[1]
        if out is None:
            out = torch.empty_like(q)
            op = out.data_ptr()
        else:
            op = self._rows("out", out, q.dtype, q.shape)
        table_at, stride = self._table(table, batch)
        offsets = None if q_offsets is None else self._ints("q_offsets", q_offsets, batch + 1)
        held = None if counts is None else self._ints("page_counts", counts, self.num_pages)
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)
        lse = self.k_scales.new_empty((rows, heads)) if return_lse else None
        key = (batch, rows, heads, offsets is None, q.dtype)
        need = self._workspace.get(key)   # bytes, a function of the sizes alone
        if need is None:
            need = self._workspace_bytes(key)
        # a new block each call: torch orders its reuse by stream, and a captured graph keeps its own
        work = self.status.new_empty((need + 3) // 4)
        q_stride, out_stride = q.stride(), out.stride()
        try:
            args = _ATTENTION_ARGS.pack(
                _TYPES[q.dtype], batch, rows, heads, qp or 0, op or 0, lse.data_ptr() if return_lse else 0, q_stride[0],
                q_stride[1], out_stride[0], out_stride[1], offsets or 0, lens_at or 0, table_at or 0, stride, held or 0,
                table.shape[1], scale, causal, min(window, 0x7fffffff), work.data_ptr() or 0, need, self._status_at)
        except _UNFIT as e:
            _invalid(f"scale, window or a size does not fit: {e}")
        _check(self.lib.dsd_scaled_attention(self._index, self._desc_at, args, _raw_stream(self._index)))
        return (out, lse) if return_lse else out

    def _workspace_bytes(self, key):
        if len(self._workspace) >= 1024:
            self._workspace.clear()
        batch, rows, heads, single, dtype = key
        a = ScaledAttentionArgs(dtype=_TYPES[dtype], batch=batch, total_queries=rows, num_q_heads=heads,
                                q_offsets=None if single else 4, scale=1.0)
        n = ctypes.c_int64()
        _check(self.lib.dsd_scaled_attention_workspace(self._index, self._desc_at, ctypes.byref(a), ctypes.byref(n)))
        need = self._workspace[key] = n.value
        return need

    def attend(self, q, page_table, seq_lens, q_offsets=None, scale: float | None = None, causal: bool = True,
               window: int = 0, out=None, return_lse: bool = False):
        """Attention of each request's last queries over its first ``seq_lens[b]`` tokens.

        ``q`` ``[queries, num_q_heads, head_dim]``: request b's are rows ``q_offsets[b] :
        q_offsets[b + 1]`` (None: one query for each request), its last tokens.  ``scale`` defaults
        to ``head_dim ** -0.5``.  ``window`` > 0 lets a query see that many tokens, itself
        included.  A query that sees nothing gets zeros and -inf; rows behind the last request's stay as
        they are in ``out`` and mean nothing in a fresh one.  Returns ``out`` or
        ``(out, lse)``, lse float32 ``[queries, num_q_heads]``.
        """
        return self._attend(q, page_table, seq_lens, q_offsets, None, scale, causal, window, out, return_lse)

    def attend_pages(self, q, page_lists, list_lens, page_counts, q_offsets=None, scale: float | None = None,
                     out=None, return_lse: bool = False):
        """Attention over listed pages in any order, such as a top-k selection.

        Request b attends to the tokens of the pages ``page_lists[b, :list_lens[b]]``; page p holds
        ``page_counts[p]`` tokens (:meth:`append` keeps them in ``token_counts``).
        """
        return self._attend(q, page_lists, list_lens, q_offsets, page_counts, scale, False, 0, out, return_lse)
