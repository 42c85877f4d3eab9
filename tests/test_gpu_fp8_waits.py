"""Bounded waits of the attention over the 8-bit KV cache that run out: a call with next to no time for them returns, says so in the status word or is
right, and leaves the device as it was for the next call."""
import ctypes
import math

import pytest
import torch

import flash_attention_b200 as fa
from tests.test_fp8_cache_cpu import Cache, Fwd

pytestmark = pytest.mark.gpu

SITES = range(130, 151)          # of the waits of these kernels


def call(device, cache, table, lens, q, out, status, splits, budget):
    """The C entry with a limit for each wait; returns what has to live until the launches have run."""
    L = fa.lib()
    L.fa4_fp8_cache_fwd_workspace_bytes.restype = ctypes.c_int64
    pages, size, H, D = cache.k.shape
    B, Sq, Hq, _ = q.shape
    at = lambda t: dict(zip(("p", "t", "h"), t.stride()[:3]))
    k, v = at(cache.k), at(cache.v)
    c = Cache(struct_size=ctypes.sizeof(Cache), num_pages=pages, page_size=size, block=cache.block, Hkv=H, D=D, k=cache.k.data_ptr(), v=cache.v.data_ptr(),
              k_scale=cache.k_scale.data_ptr(), v_scale=cache.v_scale.data_ptr(), kp=k["p"], kt=k["t"], kh=k["h"], vp=v["p"], vt=v["t"], vh=v["h"],
              page_table=table.data_ptr(), pages_per_seq=table.shape[1])
    f = Fwd(struct_size=ctypes.sizeof(Fwd), B=B, Sq=Sq, Hq=Hq, q=q.data_ptr(), out=out.data_ptr(), qb=q.stride(0), qs=q.stride(1), qh=q.stride(2),
            ob=out.stride(0), os=out.stride(1), oh=out.stride(2), seqused_k=lens.data_ptr(), softmax_scale=1 / math.sqrt(D), causal=1, window_left=-1,
            window_right=-1, num_splits=splits, status=status.data_ptr(), wait_budget_ns=budget)
    need = L.fa4_fp8_cache_fwd_workspace_bytes(ctypes.byref(c), ctypes.byref(f))
    assert need >= 0
    room = torch.empty(max(16, need), dtype=torch.uint8, device=device)
    f.workspace, f.workspace_bytes = room.data_ptr(), need
    assert L.fa4_fp8_cache_fwd(ctypes.byref(c), ctypes.byref(f), ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)) == 0
    return room


def batch(device, D, Sq, G=32):
    B, n, size, H = 3, 3000, 64, 2
    per = -(-n // size)
    g = torch.Generator(device=device).manual_seed(1)
    cache = fa.FP8KVCache.empty(B * per, size, H, D, device=device)
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x.copy_((torch.randn(x.shape, generator=g, device=device) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn))
        s.fill_(0.01)
    table = torch.randperm(B * per, generator=g, device=device).view(B, per).int()
    lens = torch.tensor([n, 1111, 77], dtype=torch.int32, device=device)
    return cache, table, lens, torch.randn(B, Sq, G, D, generator=g, device=device).bfloat16()


def run(device, D, Sq, splits, G, host):
    """Calls with little time for their waits; how many of them gave up."""
    cache, table, lens, q = batch(device, D, Sq, G)
    want, _ = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, num_splits=splits)
    torch.cuda.synchronize()
    status = torch.zeros(1, dtype=torch.int32, device=device)
    slow = q.cpu().pin_memory() if host else q
    expired = 0
    for budget in (1, 1, 1, 1000, 0):
        out = torch.zeros_like(want)
        room = call(device, cache, table, lens, slow, out, status, splits, budget)
        torch.cuda.synchronize()
        word = int(status.item()) & 0xFFFFFFFF
        status.zero_()
        if word == 0:
            assert torch.equal(out, want)
        else:
            assert budget > 0 and word >> 24 == 1 and (word >> 16) & 0xFF in SITES
            expired += 1
        del room
    again, _ = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, num_splits=splits)
    fa.check_status(device)
    assert torch.equal(again, want)
    return expired


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,splits,G", [(1, 0, 8), (1, 1, 8), (1, 3, 8), (6, 0, 8), (70, 1, 8), (70, 3, 8), (200, 0, 8)])
def test_a_call_with_little_time_is_right_or_reported(cuda_device, D, Sq, splits, G):
    run(cuda_device, D, Sq, splits, G, host=False)


@pytest.mark.parametrize("splits", [0, 1, 3])
def test_waits_for_queries_that_come_late_run_out(cuda_device, splits):
    """Queries in pinned host memory: 27 MB, half a millisecond on their way, with keys and values long there.  The products' wait for the
    first of them ends after its limit (and the time of its polls, a tenth of a millisecond)."""
    assert run(cuda_device, 128, 1100, splits, 32, host=True) > 0
