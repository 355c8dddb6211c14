"""The scaled 8-bit cache without a GPU: the oracle's rounding, and what the C ABI refuses before it looks for one."""
import ctypes

import numpy as np
import pytest

import scaled_cache_oracle as o
from conftest import load_pkg

dsd = load_pkg()


def test_oracle_rounds_like_torch():
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).standard_normal(100000) * 100
    x = np.concatenate([x, o.TABLE[~np.isnan(o.TABLE)], (o._POSITIVE[1:] + o._POSITIVE[:-1]) / 2,
                        [1e9, -1e9, np.inf, -np.inf, np.nan, 1e-9]]).astype(np.float32)
    t = torch.from_numpy(x)
    fp8 = torch.where(t.isnan(), t, t.clamp(-448, 448)).to(torch.float8_e4m3fn)
    assert np.array_equal(fp8.view(torch.uint8).numpy(), o.encode(x, "fp8"))
    assert np.array_equal(fp8.double().numpy(), o.decode(o.encode(x, "fp8"), "fp8"), equal_nan=True)
    i8 = torch.where(t.isnan(), torch.zeros_like(t), t.round().clamp(-127, 127)).to(torch.int8)
    assert np.array_equal(i8.numpy().view(np.uint8), o.encode(x, "int8"))


@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_oracle_append_keeps_values(fmt):
    """Each stored value is within half a step of the input, once for its own rounding and once more for every
    growth of its block's scale."""
    rng = np.random.default_rng(1)
    P, bt, D, n = 16, 8, 16, 40
    zero = np.zeros((4, P, 1, D), np.uint8)
    pool = o.Pool(fmt, {"k": zero, "v": zero}, {x: np.zeros((4, 1, P // bt), np.float32) for x in "kv"})
    x = rng.standard_normal((n, 1, D)).astype(np.float32)
    row, at = [2, 0, 3], 0
    for part in (13, 1, 1, 5, 20):
        at += part
        pool.append("v", x[at - part:at], row, at)
    for t in range(n):
        got = pool.values("v", row[t // P], t % P, 0)
        scale = float(pool.scales["v"][row[t // P], 0, t % P // bt])
        if fmt == "int8":
            step = np.full(D, 0.5 * scale)
        else:
            step = np.maximum(np.abs(x[t, 0]) * 2.0 ** -4 * (1 + 2.0 ** -4), scale * 2.0 ** -10)
        assert (np.abs(got - x[t, 0]) <= 3 * step * (1 + 1e-6)).all()


def cache(**kw):
    c = dsd.ScaledCacheDesc(dsd.KV_FP8_SCALED, 4, 16, 2, 64, 16, 4096, 4096, 4096, 4096,
                            (ctypes.c_int64 * 3)(2048, 128, 64), (ctypes.c_int64 * 3)(2048, 128, 64))
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def append_args(**kw):
    a = dsd.ScaledAppendArgs(dtype=1, batch=2, total_tokens=2, max_pages_per_request=2, k=4096, v=4096, seq_lens=4096,
                             page_table=4096, page_table_stride=2)
    a.k_stride[:] = a.v_stride[:] = (128, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attention_args(**kw):
    a = dsd.ScaledAttentionArgs(dtype=1, batch=2, total_queries=2, num_q_heads=4, q=4096, out=4096, lens=4096, page_table=4096,
                                page_table_stride=2, max_pages_per_request=2, scale=0.1, causal=1)
    a.q_stride[:] = a.out_stride[:] = (256, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(fn, *args):
    lib = dsd.load_library()
    rc = getattr(lib, fn)(0, *args)
    return rc == dsd.DSD_EINVAL and len(lib.dsd_last_error()) > 0


BAD_CACHE = [dict(kv_format=2), dict(kv_format=5), dict(num_pages=0), dict(page_size=0), dict(page_size=4112),
             dict(num_kv_heads=0), dict(head_dim=60), dict(head_dim=264), dict(head_dim=0), dict(block_tokens=5),
             dict(block_tokens=0), dict(block_tokens=512, page_size=512), dict(k_stride=(ctypes.c_int64 * 3)(0, 1, 1)),
             dict(k_codes=None), dict(v_scales=None), dict(k_scales=4097)]
BAD_APPEND = [dict(dtype=3), dict(batch=-1), dict(total_tokens=3), dict(num_q_heads=-1), dict(num_q_heads=2),
              dict(max_pages_per_request=-1), dict(cos=4096), dict(cos=4096, sin=4096, rotary_dim=7, rotary_positions=4),
              dict(cos=4096, sin=4096, rotary_dim=66, rotary_positions=4), dict(cos=4096, sin=4096, rotary_dim=64),
              dict(k=None), dict(seq_lens=None), dict(page_table=None), dict(k=4097), dict(k_stride=(ctypes.c_int64 * 2)(-1, 64))]
BAD_ATTENTION = [dict(dtype=-1), dict(batch=4097, total_queries=4097), dict(total_queries=3), dict(num_q_heads=3),
                 dict(num_q_heads=0), dict(window=-1), dict(page_counts=4096), dict(scale=float("inf")), dict(q=None),
                 dict(lens=None), dict(out=4097), dict(out_stride=(ctypes.c_int64 * 2)(256, -64)),
                 dict(total_queries=2 ** 30, q_offsets=4096)]


@pytest.mark.parametrize("kw", BAD_CACHE, ids=str)
def test_refuses_caches(kw):
    assert refused("dsd_scaled_append", ctypes.byref(cache(**kw)), ctypes.byref(append_args()), None)
    assert refused("dsd_scaled_attention", ctypes.byref(cache(**kw)), ctypes.byref(attention_args()), None)


@pytest.mark.parametrize("kw", BAD_APPEND, ids=str)
def test_refuses_appends(kw):
    assert refused("dsd_scaled_append", ctypes.byref(cache()), ctypes.byref(append_args(**kw)), None)


@pytest.mark.parametrize("kw", BAD_ATTENTION, ids=str)
def test_refuses_attention(kw):
    assert refused("dsd_scaled_attention", ctypes.byref(cache()), ctypes.byref(attention_args(**kw)), None)


def test_refuses_null_and_takes_empty_calls():
    lib = dsd.load_library()
    assert refused("dsd_scaled_append", None, ctypes.byref(append_args()), None)
    assert refused("dsd_scaled_append", ctypes.byref(cache()), None, None)
    assert refused("dsd_scaled_attention", ctypes.byref(cache()), None, None)
    assert refused("dsd_scaled_attention_workspace", ctypes.byref(cache()), ctypes.byref(attention_args()), None)
    assert lib.dsd_scaled_append(0, ctypes.byref(cache()), ctypes.byref(append_args(batch=0, total_tokens=0)), None) == 0
    assert lib.dsd_scaled_attention(0, ctypes.byref(cache()), ctypes.byref(attention_args(batch=0, total_queries=0)), None) == 0


def test_tensors_on_the_cpu_are_refused():
    torch = pytest.importorskip("torch")
    c = torch.zeros(4, 16, 2, 64, dtype=torch.int8)
    s = torch.zeros(4, 2, 1)
    with pytest.raises(dsd.InvalidArgument):
        dsd.ScaledKVCache.from_tensors(c, c, s, s)
    with pytest.raises(dsd.InvalidArgument):
        dsd.RotaryTable(s[0], s[0, :1])


def test_struct_sizes_match_the_header(tmp_path):
    """The ctypes mirrors have the C structs' sizes and last offsets."""
    import os
    import subprocess
    from conftest import ROOT
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "dsd_b200.h"\nint main(void){printf("%zu %zu %zu %zu %zu %zu\\n",'
                   "sizeof(dsd_scaled_cache),sizeof(dsd_scaled_append_args),sizeof(dsd_scaled_attention_args),"
                   "offsetof(dsd_scaled_cache,v_stride),offsetof(dsd_scaled_append_args,status),"
                   "offsetof(dsd_scaled_attention_args,status));return 0;}")
    subprocess.run(["gcc", "-I" + os.path.join(ROOT, "include"), "-o", str(tmp_path / "s"), str(src)], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()))
    mine = [dsd.ScaledCacheDesc, dsd.ScaledAppendArgs, dsd.ScaledAttentionArgs]
    assert got[:3] == [ctypes.sizeof(m) for m in mine]
    from importlib import import_module
    binding = import_module(dsd.__name__ + ".scaled_cache")
    assert [binding._APPEND_ARGS.size, binding._ATTENTION_ARGS.size] == got[1:3]
    assert got[3:] == [dsd.ScaledCacheDesc.v_stride.offset, dsd.ScaledAppendArgs.status.offset,
                       dsd.ScaledAttentionArgs.status.offset]


def test_kernels_that_start_early_use_no_read_only_loads():
    """They are placed before their predecessor ends: what it writes must not be read through the read-only path."""
    import glob
    import os
    from conftest import PKG_NAME, ROOT
    files = glob.glob(os.path.join(ROOT, PKG_NAME, "csrc", "dsd_scaled_*"))
    assert len(files) > 4
    for f in files:
        code = "\n".join(line.split("//")[0] for line in open(f))
        assert "__ldg" not in code and "ld.global.nc" not in code, f


def test_refuses_status_words():
    for status, bits in ((None, 4096), (4096, None), (4098, 4096), (4096, 4097)):
        assert refused("dsd_scaled_take_status", status, bits, None)


@pytest.mark.parametrize("field", ["token_offsets", "seq_lens", "page_table", "positions", "token_counts", "status"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_refuses_misaligned_ints_of_an_append(field, off):
    assert refused("dsd_scaled_append", ctypes.byref(cache()), ctypes.byref(append_args(**{field: 4096 + off})), None)


@pytest.mark.parametrize("field", ["q_offsets", "lens", "page_table", "page_counts", "status"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_refuses_misaligned_ints_of_an_attention(field, off):
    args = attention_args(causal=0, **{field: 4096 + off})
    args.workspace, args.workspace_bytes = 4096, 2 ** 40
    assert refused("dsd_scaled_attention", ctypes.byref(cache()), ctypes.byref(args), None)


def strides(*n):
    return (ctypes.c_int64 * len(n))(*n)


def test_refuses_rows_that_overlap():
    """Rows that a call writes must not share memory; rows that it reads may."""
    lib = dsd.load_library()
    for st in (strides(0, 64), strides(256, 0), strides(63, 256), strides(256, 8), strides(64, 64)):
        args = append_args(num_q_heads=4, q=4096, q_out=4096, q_stride=strides(0, 0), q_out_stride=st)
        assert refused("dsd_scaled_append", ctypes.byref(cache()), ctypes.byref(args), None)
        assert b"q_out overlap" in lib.dsd_last_error()
        args = attention_args(q_stride=strides(0, 0), out_stride=st, workspace=4096, workspace_bytes=2 ** 40)
        assert refused("dsd_scaled_attention", ctypes.byref(cache()), ctypes.byref(args), None)
        assert b"out overlap" in lib.dsd_last_error()
    for name in ("k_stride", "v_stride"):
        for st in (strides(32, 128, 64), strides(2048, 64, 64), strides(2048, 128, 1)):
            assert refused("dsd_scaled_append", ctypes.byref(cache(**{name: st})), ctypes.byref(append_args()), None)
            assert b"the cache overlap" in lib.dsd_last_error()


def test_dimensions_of_one_may_have_any_stride():
    lib = dsd.load_library()
    args = append_args(batch=1, total_tokens=1, num_q_heads=1, q=4096, q_out=4096, q_out_stride=strides(0, 0))
    one = cache(num_pages=1, page_size=1, block_tokens=1, num_kv_heads=1, k_stride=strides(1, 1, 1))
    # the arrays are made up: no device has this index, so the call ends behind its checks
    assert lib.dsd_scaled_append(99, ctypes.byref(one), ctypes.byref(args), None) not in (dsd.DSD_OK, dsd.DSD_EINVAL)
    assert b"overlap" not in lib.dsd_last_error()
