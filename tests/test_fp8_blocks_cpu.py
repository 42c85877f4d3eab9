"""Chosen blocks of the 8-bit KV cache, and its pages, without a GPU: exports, the refusals of the C ABI and of the Python calls,
the oracle's own parts."""
import ctypes
import math

import pytest
import torch

import flash_attention_b200 as fa
from flash_attention_b200 import _lib
from oracle import fp8_blocks_oracle as orc
from tests.test_fp8_cache_cpu import ALIGN, BAD_CACHES, LARGE, NULL, SHAPE, STRIDE, STRUCT, cache, fwd

P, I32, I64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64


class Index(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32), ("reserved", ctypes.c_uint32), ("bounds", P), ("scale", P)]


class IndexCall(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32), ("B", I32), ("S", I32), ("reserved", ctypes.c_uint32), ("seqlens", P), ("seqused_new", P), ("status", P)]


class Select(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, I32) for n in ("B", "Sq", "Hq")] + [("q", P)] + [(n, I64) for n in ("qb", "qs", "qh")] + \
               [("seqused_k", P), ("seqused_q", P)] + [(n, I32) for n in ("num_blocks", "query_block", "front_blocks", "recent_blocks")] + [("blocks", P), ("status", P)]


class Blocks(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32), ("num_blocks", I32), ("query_block", I32), ("reserved", ctypes.c_uint32), ("blocks", P)]


class Pages(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, I32) for n in ("B", "pages_per_seq", "num_pages", "page_size")] + \
               [("reserved", ctypes.c_uint32), ("table", P), ("refs", P), ("status", P)]


class Paged(ctypes.Structure):
    _fields_ = [("base", P)] + [(n, I64) for n in ("page", "inner", "outer", "row_bytes", "rows_inner", "rows_outer")]


class Copy(ctypes.Structure):
    _fields_ = [("struct_size", ctypes.c_uint32)] + [(n, I32) for n in ("num_pairs", "num_pages", "num_tensors")] + [("pairs", P), ("status", P), ("t", Paged * 8)]


def made(cls, defaults, kw):
    x = cls(struct_size=ctypes.sizeof(cls), **defaults)
    for n, v in kw.items():
        setattr(x, n, v)
    return x


index = lambda **kw: made(Index, dict(bounds=4096, scale=64), kw)
index_call = lambda **kw: made(IndexCall, dict(B=2, S=3, seqlens=64), kw)
select = lambda **kw: made(Select, dict(B=2, Sq=1, Hq=8, q=4096, qb=1024, qs=1024, qh=128, seqused_k=64, num_blocks=4, query_block=1, front_blocks=1,
                                        recent_blocks=1, blocks=64), kw)
blocks = lambda **kw: made(Blocks, dict(num_blocks=4, query_block=1, blocks=64), kw)
pages = lambda **kw: made(Pages, dict(B=3, pages_per_seq=4, num_pages=10, page_size=16, table=64, refs=64), kw)


def copy(paged=None, **kw):
    c = made(Copy, dict(num_pairs=2, num_pages=10, num_tensors=1, pairs=64), kw)
    for i in range(8):
        c.t[i] = Paged(**{**dict(base=4096, page=1024, inner=0, outer=0, row_bytes=1024, rows_inner=1, rows_outer=1), **(paged or {})})
    return c


def test_exports():
    for name in _lib.EXPORTS_FP8 + _lib.EXPORTS_PAGES:
        assert hasattr(fa.lib(), name)


@pytest.mark.parametrize("kw,rc", BAD_CACHES)
def test_bad_caches_are_refused(kw, rc):
    L, c = fa.lib(), cache(**kw)
    assert L.fa4_fp8_cache_index(ctypes.byref(c), ctypes.byref(index()), ctypes.byref(index_call()), None) == rc
    assert L.fa4_fp8_cache_select(ctypes.byref(c), ctypes.byref(index()), ctypes.byref(select()), None) == rc
    assert L.fa4_fp8_cache_fwd_blocks(ctypes.byref(c), ctypes.byref(fwd(causal=1)), ctypes.byref(blocks()), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(struct_size=1), STRUCT), (dict(bounds=None), NULL), (dict(scale=None), NULL), (dict(bounds=4104), ALIGN)])
def test_bad_indexes_are_refused(kw, rc):
    L = fa.lib()
    assert L.fa4_fp8_cache_index(ctypes.byref(cache()), ctypes.byref(index(**kw)), ctypes.byref(index_call()), None) == rc
    assert L.fa4_fp8_cache_select(ctypes.byref(cache()), ctypes.byref(index(**kw)), ctypes.byref(select()), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(struct_size=1), STRUCT), (dict(seqlens=None), NULL), (dict(B=0), SHAPE), (dict(S=0), SHAPE), (dict(S=-1), SHAPE),
                                   (dict(B=1 << 30, S=1 << 20), LARGE)])
def test_bad_index_calls_are_refused(kw, rc):
    L = fa.lib()
    assert L.fa4_fp8_cache_index(ctypes.byref(cache()), ctypes.byref(index()), ctypes.byref(index_call(**kw)), None) == rc
    assert L.fa4_fp8_cache_index(ctypes.byref(cache()), None, ctypes.byref(index_call()), None) == NULL
    assert L.fa4_fp8_cache_index(ctypes.byref(cache()), ctypes.byref(index()), None, None) == NULL


@pytest.mark.parametrize("kw,rc", [
    (dict(struct_size=1), STRUCT), (dict(q=None), NULL), (dict(seqused_k=None), NULL), (dict(blocks=None), NULL), (dict(B=0), SHAPE), (dict(Sq=0), SHAPE),
    (dict(Hq=3), SHAPE), (dict(num_blocks=0), SHAPE), (dict(num_blocks=1), SHAPE), (dict(query_block=0), SHAPE), (dict(front_blocks=-1), SHAPE),
    (dict(recent_blocks=0), SHAPE), (dict(front_blocks=4), SHAPE), (dict(front_blocks=2 ** 31 - 1, recent_blocks=2 ** 31 - 1), SHAPE),
    (dict(Sq=100, query_block=98), SHAPE), (dict(qs=4), STRIDE), (dict(q=4098), ALIGN), (dict(B=1 << 20, Sq=1 << 12), LARGE),
    (dict(Sq=1 << 14, query_block=1 << 14, num_blocks=1 << 12), LARGE)])
def test_bad_choices_are_refused(kw, rc):
    L = fa.lib()
    assert L.fa4_fp8_cache_select(ctypes.byref(cache()), ctypes.byref(index()), ctypes.byref(select(**kw)), None) == rc


def test_what_is_always_chosen_has_to_fit():
    """(blocks of 32 tokens: 33 rows may touch two, 34 three)"""
    L = fa.lib()
    for rows, need in ((1, 2), (2, 3), (33, 3), (34, 4)):
        for chosen in (need - 1, need):
            s = select(Sq=64, query_block=rows, num_blocks=chosen, q=4098)
            assert L.fa4_fp8_cache_select(ctypes.byref(cache()), ctypes.byref(index()), ctypes.byref(s), None) == (SHAPE if chosen < need else ALIGN)


def test_more_blocks_than_fit_into_shared_memory_are_refused():
    L = fa.lib()
    c = cache(pages_per_seq=26625)                                   # (two blocks a page)
    assert L.fa4_fp8_cache_select(ctypes.byref(c), ctypes.byref(index()), ctypes.byref(select()), None) == LARGE


@pytest.mark.parametrize("kw,more,rc", [
    (dict(), dict(struct_size=1), STRUCT), (dict(), dict(blocks=None), NULL), (dict(), dict(num_blocks=0), SHAPE), (dict(), dict(query_block=0), SHAPE),
    (dict(causal=0), dict(), SHAPE), (dict(window_left=5), dict(), SHAPE), (dict(window_right=1), dict(), SHAPE), (dict(num_splits=1), dict(), SHAPE),
    (dict(), dict(num_blocks=1 << 26), LARGE), (dict(Sq=1 << 20, B=1 << 4, Hq=2), dict(num_blocks=1 << 20), LARGE), (dict(struct_size=1), dict(), STRUCT), (dict(q=None), dict(), NULL)])
def test_bad_attention_over_blocks_is_refused(kw, more, rc):
    L = fa.lib()
    L.fa4_fp8_cache_fwd_blocks_workspace_bytes.restype = ctypes.c_int64
    c = cache(pages_per_seq=1 << 12)
    f, x = fwd(**{"causal": 1, **kw}), blocks(**more)
    assert L.fa4_fp8_cache_fwd_blocks(ctypes.byref(c), ctypes.byref(f), ctypes.byref(x), None) == rc
    assert L.fa4_fp8_cache_fwd_blocks_workspace_bytes(ctypes.byref(c), ctypes.byref(f), ctypes.byref(x)) == rc
    assert L.fa4_fp8_cache_fwd_blocks(ctypes.byref(c), ctypes.byref(fwd(causal=1)), None, None) == NULL


def test_a_workspace_that_is_none_is_refused():
    """80 units of 25 tiles are dealt out to the CTAs, whose pieces need one; 2 of them are split among the CTAs of a cluster and need none."""
    L = fa.lib()
    L.fa4_fp8_cache_fwd_blocks_workspace_bytes.restype = ctypes.c_int64
    c, x = cache(pages_per_seq=100), blocks(num_blocks=100)
    assert L.fa4_fp8_cache_fwd_blocks_workspace_bytes(ctypes.byref(c), ctypes.byref(fwd(causal=1, B=1)), ctypes.byref(x)) == 0
    need = L.fa4_fp8_cache_fwd_blocks_workspace_bytes(ctypes.byref(c), ctypes.byref(fwd(causal=1, B=40)), ctypes.byref(x))
    assert need > 0
    for kw, rc in ((dict(), NULL), (dict(workspace=4104, workspace_bytes=need), ALIGN), (dict(workspace=4096, workspace_bytes=need - 1), LARGE)):
        assert L.fa4_fp8_cache_fwd_blocks(ctypes.byref(c), ctypes.byref(fwd(causal=1, B=40, **kw)), ctypes.byref(x), None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(struct_size=1), STRUCT), (dict(table=None), NULL), (dict(refs=None), NULL), (dict(B=0), SHAPE), (dict(pages_per_seq=0), SHAPE),
                                   (dict(num_pages=0), SHAPE), (dict(page_size=0), SHAPE), (dict(pages_per_seq=1 << 20, page_size=1 << 12), LARGE), (dict(num_pages=1 << 30), LARGE)])
def test_bad_pages_are_refused(kw, rc):
    L, k = fa.lib(), pages(**kw)
    for fn in (L.fa4_kv_pages_resize_workspace_bytes, L.fa4_kv_pages_compact_workspace_bytes):
        fn.restype = ctypes.c_int64
        assert fn(ctypes.byref(k)) == rc
    assert L.fa4_kv_pages_resize(ctypes.byref(k), P(64), P(64), P(64), P(64), ctypes.c_uint64(1 << 20), None) == rc
    assert L.fa4_kv_pages_fork(ctypes.byref(k), P(64), P(64), 3, P(64), P(64), None) == rc
    assert L.fa4_kv_pages_compact(ctypes.byref(k), P(64), P(64), P(64), ctypes.c_uint64(1 << 20), None) == rc


def test_bad_calls_on_pages_are_refused():
    L, k = fa.lib(), pages()
    for fn in (L.fa4_kv_pages_resize_workspace_bytes, L.fa4_kv_pages_compact_workspace_bytes):
        fn.restype = ctypes.c_int64
    n, m = L.fa4_kv_pages_resize_workspace_bytes(ctypes.byref(k)), L.fa4_kv_pages_compact_workspace_bytes(ctypes.byref(k))
    assert L.fa4_kv_pages_resize_workspace_bytes(ctypes.byref(pages(B=4097))) == LARGE
    size = lambda x: ctypes.c_uint64(x)
    for args, rc in (((None, 64, 64, 64, n), NULL), ((64, None, 64, 64, n), NULL), ((64, 64, None, 64, n), NULL), ((64, 64, 64, None, n), NULL), ((64, 64, 64, 72, n), ALIGN),
                     ((64, 64, 64, 64, n - 1), LARGE)):
        assert L.fa4_kv_pages_resize(ctypes.byref(k), *(P(a) for a in args[:4]), size(args[4]), None) == rc
    for args, rc in (((None, 64, 64, m), NULL), ((64, None, 64, m), NULL), ((64, 64, None, m), NULL), ((64, 64, 72, m), ALIGN), ((64, 64, 64, m - 1), LARGE)):
        assert L.fa4_kv_pages_compact(ctypes.byref(k), *(P(a) for a in args[:3]), size(args[3]), None) == rc
    for args, rc in (((None, 64, 3, 64, 64), NULL), ((64, None, 3, 64, 64), NULL), ((64, 64, 3, None, 64), NULL), ((64, 64, 3, 64, None), NULL), ((64, 64, 0, 64, 64), SHAPE),
                     ((64, 64, 2 ** 31 - 1, 64, 64), LARGE)):
        assert L.fa4_kv_pages_fork(ctypes.byref(k), P(args[0]), P(args[1]), args[2], P(args[3]), P(args[4]), None) == rc


@pytest.mark.parametrize("kw,paged,rc", [
    (dict(struct_size=1), {}, STRUCT), (dict(pairs=None), {}, NULL), (dict(num_pairs=0), {}, SHAPE), (dict(num_pages=0), {}, SHAPE), (dict(num_tensors=0), {}, SHAPE),
    (dict(num_tensors=9), {}, SHAPE), ({}, dict(base=None), NULL), ({}, dict(row_bytes=0), SHAPE), ({}, dict(rows_inner=0), SHAPE), ({}, dict(page=-1), STRIDE),
    ({}, dict(rows_inner=2, inner=-16), STRIDE), ({}, dict(rows_outer=2, outer=-16), STRIDE), ({}, dict(rows_outer=1 << 16, rows_inner=1 << 16), LARGE),
    ({}, dict(row_bytes=1 << 32), LARGE), ({}, dict(base=4097, row_bytes=(1 << 30) + 1), LARGE), (dict(num_pairs=1 << 30), {}, LARGE)])
def test_bad_copies_are_refused(kw, paged, rc):
    assert fa.lib().fa4_kv_pages_copy(ctypes.byref(copy(paged, **kw)), None) == rc


def test_tensors_on_the_cpu_are_refused():
    c = fa.FP8KVCache.empty(4, 64, 2, 128, device="cpu", indexed=True, by_head=True)
    assert c.block == 64 and c.key_bounds.shape == (4, 1, 2, 2, 128) and c.bound_scale.shape == (4, 1, 2) and c.k.shape == (4, 64, 2, 128) and c.k.stride(1) == 128
    q, n = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: fa.index_kv_fp8(c, n, 1), lambda: fa.select_kv_blocks(q, c, n, 4), lambda: fa.flash_attn_fp8_blocks_func(q, c, n.view(1, 1, 1, 1), n),
                 lambda: fa.append_kv_fp8(c, q, q, n)):
        with pytest.raises(AssertionError, match="must be on CUDA"):
            call()
    with pytest.raises(TypeError, match="cache_seqlens must be a torch.Tensor"):
        fa.index_kv_fp8(c, 3, 1)
    with pytest.raises(TypeError, match="blocks must be a torch.Tensor"):
        fa.flash_attn_fp8_blocks_func(q, c, [[0]], n)
    p = fa.KVPages.empty(2, 3, 4, 16, device="cpu")
    assert (p.table == -1).all() and not p.refs.any()
    for call in (lambda: fa.resize_kv_pages(p, n, n), lambda: fa.fork_kv_pages(p, n, n), lambda: fa.compact_kv_pages(p), lambda: fa.copy_kv_pages(c, n.view(1, 1))):
        with pytest.raises(AssertionError, match="must be on CUDA"):
            call()


def test_oracle_bounds_are_bounds_of_seven_bits():
    g = torch.Generator().manual_seed(1)
    for scale in (1.0, 100.0, 0.01):
        x = (torch.randn(32, 3, 64, generator=g) * scale).to(torch.float8_e4m3fn).double()
        k_scale = torch.rand(3, generator=g)
        bounds, step = orc.index(x, k_scale)
        k = x * k_scale.double()[None, :, None]
        assert (bounds[:, 0].double() * step.double()[:, None] * (1 + 1e-6) + 1e-9 >= k.amax(0)).all() and (bounds[:, 1].double() * step.double()[:, None] * (1 + 1e-6) - 1e-9 <= k.amin(0)).all()
        top = torch.maximum(bounds[:, 0].abs(), bounds[:, 1].abs()).amax(-1)
        assert (top >= 64).all() and (top <= 120).all()


def test_oracle_scores_are_upper_bounds_up_to_their_rounding():
    """The score of a block against the largest q . k in it: at least that much, but for what p and n lose (half a step in 64 a channel, of bounds of 120 steps)."""
    g = torch.Generator().manual_seed(2)
    for _ in range(20):
        x = torch.randn(16, 1, 64, generator=g).mul(60).to(torch.float8_e4m3fn).double()
        q = torch.randn(1, 1, 64, generator=g).bfloat16()
        bounds, step = orc.index(x, torch.ones(1))
        p, n = orc.seven_bits(q)
        most = max(int(p.max()), int(n.max()))
        assert 64 <= most <= 127
        unit = float(q.abs().max()) / most                          # (of a step of p and n, to one in 128)
        score = float(orc.scores(q, bounds, step)[0]) * unit
        assert score >= float((x[:, 0] @ q[0, 0].double()).max()) - 64 * 120 * float(step[0]) * unit
        assert score >= 0


def test_oracle_lists():
    assert orc.keys_of([0, 2, 1, 3], 2) == [0, 1, 4, 5] and orc.keys_of([-1, 0], 2) == [] and orc.keys_of([1, 1], 2) == [2, 3]
    q = torch.ones(1, 1, 4).bfloat16()
    bounds = torch.zeros(6, 2, 4, dtype=torch.int8)
    bounds[:, 0] = torch.tensor([1, 5, 2, 5, 9, 1], dtype=torch.int8)[:, None]
    scale = torch.tensor([1.0, 1.0, math.nan, 1.0, 0.1, 1.0])
    assert orc.select(q, bounds, scale, 90, 91, 16, 4, 1, 1) == [0, 1, 2, 5]
    assert orc.select(q, bounds, scale, 90, 91, 16, 3, 0, 2) == [2, 4, 5]
    assert orc.select(q, bounds, scale, 40, 41, 16, 4, 1, 1) == [0, 1, 2, -1] and orc.select(q, bounds, scale, -1, 0, 16, 2, 1, 1) == [-1, -1]
