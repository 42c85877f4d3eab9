"""The choice of blocks where a unit is a cluster's: every number of CTAs, sequences that some of them have nothing of, ties and bad pages across
them; and that a call gives the same bits every time.  Lists are compared with the oracle's for equality."""
import math

import pytest
import torch

import flash_attention_b200 as fa
from oracle import fp8_blocks_oracle as orc
from tests.test_gpu_fp8_blocks import i32, lists_of

pytestmark = pytest.mark.gpu


def with_bounds(device, pages, size, H, D, block, seed, same=False):
    """A cache of which only the index is anything: bounds of any kind, or the same for every block."""
    g = torch.Generator(device=device).manual_seed(seed)
    values = torch.zeros(pages, size, H, D, dtype=torch.uint8, device=device)
    ones = torch.ones(pages, size // block, H, device=device)
    bounds = torch.randint(-120, 121, (pages, size // block, H, 2, D), generator=g, device=device).to(torch.int8)
    scale = torch.rand(pages, size // block, H, generator=g, device=device) + 0.5
    if same:
        bounds, scale = bounds[:1, :1].expand_as(bounds).contiguous(), ones.clone()
    return fa.FP8KVCache(values, values, ones, ones, bounds, scale)


def parts_of(units, blocks):
    """How many CTAs the rule gives a unit."""
    parts = 1
    while parts < 8 and units * parts * 2 <= 148 and blocks // (parts * 2) >= 256:
        parts *= 2
    return parts


@pytest.mark.parametrize("same", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("per,parts", [(140, 2), (260, 4), (520, 8)])
@pytest.mark.parametrize("H,Sq,rows,fresh", [(3, 1, 1, None), (1, 5, 3, [5, 2, 4, 0]), (2, 70, 64, [70, 1, 66, 3])])
def test_choice_by_clusters(cuda_device, same, D, per, parts, H, Sq, rows, fresh):
    dev, B, size, block = cuda_device, 4, 64, 16
    chosen = 9 if rows < 64 else 13
    units = B * H * -(-Sq // rows)
    if parts_of(units, per * 4) != parts:
        pytest.skip("more units than clusters of that size have room for")
    pages = B * per
    g = torch.Generator(device=dev).manual_seed(per + D)
    cache = with_bounds(dev, pages, size, H, D, block, per, same)
    table = torch.randperm(pages, generator=g, device=dev).view(B, per).to(torch.int32)
    q = torch.randn(B, Sq, 4 * H, D, generator=g, device=dev).bfloat16()
    # (whole; one block more than is chosen; a few tokens; in the middle of a CTA's part)
    for lens in ([per * size, (chosen + 1) * block, 5, per * size // 2 + 33], [per * size - 1, 0, per * size // parts, chosen * block], [0, 1, 7, 2]):
        got = fa.select_kv_blocks(q, cache, i32(lens, dev), chosen, page_table=table, seqused_q=None if fresh is None else i32(fresh, dev), query_block=rows)
        want = lists_of(cache, table.tolist(), q.cpu(), lens, fresh, chosen, rows, 1, 1)
        assert torch.equal(got.cpu(), want)
    fa.check_status(dev)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("per", [140, 260, 520])
def test_bad_pages_of_any_cta_of_a_cluster(cuda_device, D, per):
    """Their blocks come last, whichever part they lie in, and are reported."""
    dev, B, H, size, block = cuda_device, 2, 2, 64, 16
    n = per * 4
    cache = with_bounds(dev, B * per, size, H, D, block, 3)
    table = torch.arange(B * per, device=dev).view(B, per).to(torch.int32)
    q = torch.randn(B, 1, 4, D, generator=torch.Generator(device=dev).manual_seed(1), device=dev).bfloat16()
    for bad in ([per - 2], [per // 3, 1], list(range(2, per - 1))):
        t = table.clone()
        t[1, bad] = torch.tensor([-1, 10 ** 9, B * per], device=dev, dtype=torch.int32).repeat(per)[:len(bad)]
        for chosen in (7, 60):
            got = fa.select_kv_blocks(q, cache, i32([per * size] * B, dev), chosen, page_table=t)
            with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
                fa.check_status(dev)
            for b in range(B):
                for h in range(H):
                    bounds, scale = (x[table[b].long()].flatten(0, 1)[:, h].cpu() for x in (cache.key_bounds, cache.bound_scale))
                    s = orc.scores(q[b, :, 2 * h:2 * h + 2].cpu(), bounds, scale)
                    if b == 1:
                        s[(torch.tensor(bad)[:, None] * 4 + torch.arange(4)).flatten()] = -math.inf
                    s = s.tolist()
                    want = sorted([0, n - 1] + sorted(range(1, n - 1), key=lambda j: (-s[j], j))[:chosen - 2])
                    assert got[b, 0, h].tolist() == want


def test_the_same_bits_every_time(cuda_device):
    """Lists, results and LSE of one call repeat, in each way that the attention is dealt."""
    dev = cuda_device
    for B, Sq, H, G, rows, per, chosen in ((1, 1, 8, 4, 1, 40, 16), (32, 1, 8, 4, 1, 20, 9), (40, 1, 8, 4, 1, 20, 40), (8, 5, 8, 4, 1, 24, 20), (1, 300, 2, 4, 64, 30, 24)):
        size, block, D = 64, 64, 128
        g = torch.Generator(device=dev).manual_seed(B)
        cache = fa.FP8KVCache.empty(B * per, size, H, D, block, device=dev, indexed=True, by_head=True)
        table = torch.randperm(B * per, generator=g, device=dev).view(B, per).to(torch.int32)
        lens = i32([per * size - 7 * b for b in range(B)], dev)
        k, v = (torch.randn(B, per * size, H, D, generator=g, device=dev).bfloat16() for _ in range(2))
        fa.append_kv_fp8(cache, k, v, torch.zeros_like(lens), page_table=table, seqused_new=lens)
        q = torch.randn(B, Sq, H * G, D, generator=g, device=dev).bfloat16()
        first = None
        for _ in range(6):
            lists = fa.select_kv_blocks(q, cache, lens, chosen, page_table=table, query_block=rows)
            got = (lists, *fa.flash_attn_fp8_blocks_func(q, cache, lists, lens, page_table=table, query_block=rows, return_lse=True))
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))
    fa.check_status(dev)
