"""The 8-bit KV cache without a GPU: exports, the refusals of the C ABI and of the Python calls, the oracle's own parts."""
import ctypes
import math

import pytest
import torch

import flash_attention_b200 as fa
from flash_attention_b200 import _lib
from oracle import fp8_cache_oracle as orc


class Cache(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, ctypes.c_int32) for n in ("num_pages", "page_size", "block", "Hkv", "D")] + \
               [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, ctypes.c_int64) for n in ("kp", "kt", "kh", "vp", "vt", "vh")] + \
               [("page_table", ctypes.c_void_p), ("pages_per_seq", ctypes.c_int32), ("reserved", ctypes.c_uint32)]


class Append(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, ctypes.c_int32) for n in ("B", "S", "Hq")] + \
               [(n, ctypes.c_void_p) for n in ("k", "v", "q", "q_out")] + \
               [(n, ctypes.c_int64) for n in ("kb", "ks", "kh", "vb", "vs", "vh", "qb", "qs", "qh")] + \
               [(n, ctypes.c_void_p) for n in ("seqlens", "seqused_new", "cos", "sin")] + \
               [(n, ctypes.c_int32) for n in ("rotary_dim", "rotary_rows", "rotary_bf16", "interleaved")] + [("status", ctypes.c_void_p)]


class Fwd(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, ctypes.c_int32) for n in ("B", "Sq", "Hq")] + \
               [(n, ctypes.c_void_p) for n in ("q", "out", "lse")] + [(n, ctypes.c_int64) for n in ("qb", "qs", "qh", "ob", "os", "oh")] + \
               [(n, ctypes.c_void_p) for n in ("seqused_k", "seqused_q", "sink")] + [("softmax_scale", ctypes.c_float), ("softcap", ctypes.c_float)] + \
               [(n, ctypes.c_int32) for n in ("causal", "window_left", "window_right", "num_splits")] + \
               [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_uint64), ("status", ctypes.c_void_p), ("wait_budget_ns", ctypes.c_uint64)]


def cache(**kw):
    c = Cache(struct_size=ctypes.sizeof(Cache), num_pages=8, page_size=64, block=32, Hkv=2, D=128, k=4096, v=8192, k_scale=64, v_scale=64,
              kp=64 * 256, kt=256, kh=128, vp=64 * 256, vt=256, vh=128, page_table=64, pages_per_seq=4)
    for n, v in kw.items():
        setattr(c, n, v)
    return c


def append(**kw):
    a = Append(struct_size=ctypes.sizeof(Append), B=2, S=3, Hq=0, k=4096, v=4096, kb=768, ks=256, kh=128, vb=768, vs=256, vh=128, seqlens=64)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def fwd(**kw):
    f = Fwd(struct_size=ctypes.sizeof(Fwd), B=2, Sq=1, Hq=8, q=4096, out=4096, qb=1024, qs=1024, qh=128, ob=1024, os=1024, oh=128, seqused_k=64,
            softmax_scale=0.1, window_left=-1, window_right=-1)
    for n, v in kw.items():
        setattr(f, n, v)
    return f


NULL, SHAPE, STRIDE, ALIGN, STRUCT, LARGE = -1, -2, -3, -4, -7, -8

BAD_CACHES = [(dict(struct_size=1), STRUCT), (dict(k=None), NULL), (dict(v_scale=None), NULL), (dict(block=8), SHAPE), (dict(block=48), SHAPE),
              (dict(page_size=80), SHAPE), (dict(num_pages=0), SHAPE), (dict(Hkv=0), SHAPE), (dict(D=96), SHAPE), (dict(D=192), SHAPE),
              (dict(pages_per_seq=0), SHAPE), (dict(page_table=None), SHAPE), (dict(kt=0), STRIDE), (dict(kt=-256), STRIDE), (dict(vh=8), STRIDE),
              (dict(k=4104), ALIGN), (dict(pages_per_seq=1 << 26), LARGE)]


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_bad_caches_are_refused(kw, rc):
    L = fa.lib()
    assert L.fa4_fp8_cache_append(ctypes.byref(cache(**kw)), ctypes.byref(append()), None) == rc
    assert L.fa4_fp8_cache_fwd(ctypes.byref(cache(**kw)), ctypes.byref(fwd()), None) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=1), STRUCT), (dict(k=None), NULL), (dict(seqlens=None), NULL), (dict(B=0), SHAPE), (dict(S=-1), SHAPE),
    (dict(cos=64), NULL), (dict(cos=64, sin=64), SHAPE), (dict(cos=64, sin=64, rotary_dim=24, rotary_rows=9), SHAPE),
    (dict(cos=64, sin=64, rotary_dim=144, rotary_rows=9), SHAPE), (dict(cos=64, sin=72, rotary_dim=64, rotary_rows=9), ALIGN),
    (dict(q=4096, q_out=4096, Hq=4), NULL), (dict(q=4096, Hq=4, cos=64, sin=64, rotary_dim=64, rotary_rows=9), NULL),
    (dict(q=4096, q_out=4096, Hq=0, cos=64, sin=64, rotary_dim=64, rotary_rows=9), SHAPE),
    (dict(ks=4), STRIDE), (dict(k=4098), ALIGN), (dict(B=1 << 20, S=1 << 12), LARGE)])
def test_bad_appends_are_refused(kw, rc):
    assert fa.lib().fa4_fp8_cache_append(ctypes.byref(cache()), ctypes.byref(append(**kw)), None) == rc


def test_a_contiguous_cache_has_a_page_for_every_sequence():
    L = fa.lib()
    c = cache(page_table=None, pages_per_seq=1, num_pages=1)
    assert L.fa4_fp8_cache_append(ctypes.byref(c), ctypes.byref(append()), None) == SHAPE
    assert L.fa4_fp8_cache_fwd(ctypes.byref(c), ctypes.byref(fwd()), None) == SHAPE


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=1), STRUCT), (dict(q=None), NULL), (dict(seqused_k=None), NULL), (dict(B=0), SHAPE), (dict(Hq=3), SHAPE),
    (dict(softmax_scale=0.0), SHAPE), (dict(softmax_scale=math.nan), SHAPE), (dict(softcap=-1.0), SHAPE), (dict(num_splits=129), SHAPE),
    (dict(num_splits=-1), SHAPE), (dict(qs=4), STRIDE), (dict(oh=12), STRIDE), (dict(out=4098), ALIGN), (dict(B=65536), LARGE),
    (dict(Sq=1 << 26), LARGE)])
def test_bad_attention_calls_are_refused(kw, rc):
    L = fa.lib()
    assert L.fa4_fp8_cache_fwd(ctypes.byref(cache()), ctypes.byref(fwd(**kw)), None) == rc
    L.fa4_fp8_cache_fwd_workspace_bytes.restype = ctypes.c_int64
    assert L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(cache()), ctypes.byref(fwd(**kw))) == rc


@pytest.mark.parametrize("Sq,splits", [(1, 2), (100, 2), (1, 128), (100, 128)])
def test_a_workspace_that_is_none_is_refused(Sq, splits):
    """(8 pages x 4 a sequence: nothing is launched)"""
    L = fa.lib()
    L.fa4_fp8_cache_fwd_workspace_bytes.restype = ctypes.c_int64
    c, f = cache(), fwd(Sq=Sq, num_splits=splits)
    need = L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(c), ctypes.byref(f))
    # partial results of every split: D values and a sum for each of B x Sq x Hq rows
    assert need == splits * 2 * Sq * 8 * 129 * 4
    for kw, rc in ((dict(), NULL), (dict(workspace=4104, workspace_bytes=need), ALIGN), (dict(workspace=4096, workspace_bytes=need - 1), LARGE)):
        assert L.fa4_fp8_cache_fwd(ctypes.byref(c), ctypes.byref(fwd(Sq=Sq, num_splits=splits, **kw)), None) == rc


def test_sizes_beyond_a_launch_are_refused():
    L = fa.lib()
    L.fa4_fp8_cache_fwd_workspace_bytes.restype = ctypes.c_int64
    assert L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(cache(Hkv=1 << 10)), ctypes.byref(fwd(B=1 << 15, Hq=1 << 10, num_splits=128))) == LARGE
    # tiles of all sequences and heads
    assert L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(cache(Hkv=1 << 10, pages_per_seq=1 << 12)), ctypes.byref(fwd(B=1 << 10, Hq=1 << 10))) == LARGE


def test_exports():
    for name in _lib.EXPORTS_FP8:
        assert hasattr(fa.lib(), name)


def test_tensors_on_the_cpu_are_refused():
    c = fa.FP8KVCache.empty(4, 64, 2, 128, device="cpu")
    assert c.block == 64 and c.k_scale.shape == (4, 1, 2)
    k = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(AssertionError, match="must be on CUDA"):
        fa.append_kv_fp8(c, k, k, n)
    with pytest.raises(AssertionError, match="must be on CUDA"):
        fa.flash_attn_fp8_cache_func(k, c, n)
    with pytest.raises(TypeError, match="seqused_k must be a torch.Tensor"):
        fa.flash_attn_fp8_cache_func(k, c, 3)
    with pytest.raises(AssertionError, match="k of the cache must be uint8"):
        fa.append_kv_fp8(fa.FP8KVCache(c.k.float(), c.v, c.k_scale, c.v_scale), k, k, n)


@pytest.mark.parametrize("size,block", [(24, None), (64, 48), (64, 128), (100, 16), (64, 8)])
def test_pages_that_are_no_whole_blocks_are_refused(size, block):
    with pytest.raises(ValueError, match="block"):
        fa.FP8KVCache.empty(4, size, 2, 128, block, device="cpu")


def test_dequantize():
    c = fa.FP8KVCache.empty(2, 32, 1, 64, 16, device="cpu")
    x = torch.randn(2, 32, 1, 64)
    for t, s in ((c.k, 2.0), (c.v, 0.5)):
        t.copy_((x / s).to(torch.float8_e4m3fn))
    c.k_scale.fill_(2.0)
    c.v_scale.fill_(0.5)
    k, v = c.dequantize()
    assert ((k - x).abs() <= x.abs() * 2.0 ** -4 + 2.0 ** -9).all() and ((v - x).abs() <= x.abs() * 2.0 ** -4 + 2.0 ** -9).all()


def test_oracle_rounding_is_the_types():
    """The oracle's e4m3 rounding against every value of the type, the midpoints and what torch does with them."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 1e-6), mid * (1 - 1e-6)])
    assert torch.equal(orc.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())
    assert torch.equal(orc.round_e4m3(-x), -orc.round_e4m3(x))


def test_oracle_scale():
    for top in (448.0, 448.1, 224.0, 1e-40, 3.5, 3.4999, 1e38):
        s = orc.scale_for(top)
        assert top <= 448 * s and (s == 2.0 ** -120 or top > 448 * s / 2) and math.log2(s).is_integer()


def test_a_cache_of_another_type_is_refused():
    """Two 4-bit values a byte are no e4m3 values, though they come as bytes as well."""
    c = fa.FP8KVCache.empty(4, 64, 2, 128, device="cpu")
    k = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    n = torch.zeros(1, dtype=torch.int32)
    for dtype in (torch.float4_e2m1fn_x2, torch.float8_e5m2, torch.int8):
        other = c.k.view(torch.uint8).view(dtype)
        for bad, name in ((fa.FP8KVCache(other, c.v, c.k_scale, c.v_scale), "k"), (fa.FP8KVCache(c.k, other, c.k_scale, c.v_scale), "v")):
            with pytest.raises(AssertionError, match=f"{name} of the cache must be uint8 / float8_e4m3fn"):
                fa.append_kv_fp8(bad, k, k, n)
            with pytest.raises(AssertionError, match=f"{name} of the cache must be uint8 / float8_e4m3fn"):
                fa.flash_attn_fp8_cache_func(k, bad, n)


@pytest.mark.parametrize("kw", [dict(softcap=math.inf), dict(softcap=3e38), dict(softcap=1e-41), dict(softmax_scale=math.inf), dict(softmax_scale=3e38),
                                dict(softcap=math.nan), dict(softmax_scale=1e-30, softcap=1e20), dict(softmax_scale=1e20, softcap=1e-30)])
def test_scales_and_soft_caps_beyond_fp32_are_refused(kw):
    """(0.1 over a cap of 1e-41 is infinite, 1e-30 over 1e20 is 0: every score would be NaN or 0)"""
    L = fa.lib()
    L.fa4_fp8_cache_fwd_workspace_bytes.restype = ctypes.c_int64
    f = fwd(**kw)
    assert L.fa4_fp8_cache_fwd(ctypes.byref(cache()), ctypes.byref(f), None) == SHAPE
    assert L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(cache()), ctypes.byref(f)) == SHAPE
    for ok in (dict(softcap=1e30), dict(softcap=1e-30), dict(softmax_scale=1e-30), dict(softmax_scale=1e30)):
        assert L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(cache()), ctypes.byref(fwd(**ok))) >= 0
