"""Page numbers outside the pool in attention over a paged NVFP4 cache: their keys and values read as zeros, which is reported; entries that no
row needs are not looked at.  Results are compared for equality with those of a page of zeros (under the scale factors of another page, which stand in)."""
import pytest
import torch

import flash_attention_b200 as fa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["linear", "tiled"])
@pytest.mark.parametrize("Sq,Hq,Hkv,D,Dv,causal,kw", [
    (1, 8, 2, 128, 128, True, dict(variant=fa.VARIANT_DECODE, num_splits=1)), (4, 8, 2, 128, 128, True, dict(variant=fa.VARIANT_DECODE, num_splits=3)),
    (1, 16, 1, 128, 128, False, dict(variant=fa.VARIANT_DECODE, num_splits=0)), (8, 8, 2, 128, 128, True, dict(variant=fa.VARIANT_DECODE, num_splits=9)),
    (70, 4, 2, 128, 128, True, dict(variant=fa.VARIANT_WS64)), (200, 4, 4, 128, 128, False, dict(variant=fa.VARIANT_WS64)),
    (70, 4, 2, 64, 64, True, dict(variant=fa.VARIANT_WS64)), (33, 2, 1, 192, 128, True, dict(variant=fa.VARIANT_WS64)),
    (70, 4, 2, 128, 128, True, dict(variant=fa.VARIANT_WS64, window_size=(700, 0), softcap=20.0)),
    (70, 4, 2, 128, 128, True, dict(variant=fa.VARIANT_WS64, window_size=(100, 0))), (70, 4, 2, 64, 64, True, dict(variant=fa.VARIANT_WS64, window_size=(100, 0), softcap=20.0)),
    (70, 4, 2, 128, 128, True, dict(variant=fa.VARIANT_WS)), (150, 4, 2, 128, 128, True, dict(variant=fa.VARIANT_WS, num_splits=2)),
    (40, 4, 2, 64, 64, False, dict(variant=fa.VARIANT_WS, num_splits=3))])
def test_pages_outside_the_pool(cuda_device, layout, Sq, Hq, Hkv, D, Dv, causal, kw):
    dev, B, page, per = cuda_device, 3, 256, 5
    n = B * per + 1
    g = torch.Generator(device=dev).manual_seed(Sq + D)
    q, k, v = (torch.randn(b, s, h, d, generator=g, device=dev, dtype=torch.bfloat16)
               for b, s, h, d in ((B, Sq, Hq, D), (n, page, Hkv, D), (n, page, Hkv, Dv)))
    Q, K, V = fa.quantize_qkv_fused(q, k, v)
    for t in (K, V):
        t.data[-1] = 0
    lens = torch.tensor([5 * page - 3, 300, 3 * page], dtype=torch.int32, device=dev)
    table = torch.randperm(n - 1, generator=g, device=dev).to(torch.int32).view(B, per)
    zeros, bad = table.clone(), table.clone()
    for (b, j), number in zip(((0, 1), (0, 4), (2, 0), (2, 2)), (-1, n, 10 ** 9, -2 ** 31 + 3)):
        zeros[b, j], bad[b, j] = n - 1, number
    for t in (zeros, bad):
        t[1, 2:] = 10 ** 9                     # (behind what the entry has)
        t[2, 3:] = -1

    def call(t):
        sf = [x.tiled_sf() if layout == "tiled" else x.sf for x in (Q, K, V)]
        return fa.flash_attn_fp4_func(Q.data, K.data, V.data, *sf, Q.scale, K.scale, V.scale, causal=causal, return_lse=True, sf_layout=layout,
                                      seqused_k=lens, page_table=t, **kw)
    want = [x.clone() for x in call(zeros)]
    torch.cuda.synchronize()
    fa.check_status(dev)
    got = call(bad)
    with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
        fa.check_status(dev)
    assert torch.isfinite(want[0].float()).all()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_attention_by_a_table_that_found_no_page(cuda_device):
    """A table that a pool could not fill, with lengths that were not cut to what was granted: reported, not read; with those that were, right."""
    dev, page, Hq, Hkv, D = cuda_device, 128, 8, 2, 128
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = (torch.randn(b, s, h, D, generator=g, device=dev, dtype=torch.bfloat16) for b, s, h in ((3, 1, Hq), (4, page, Hkv), (4, page, Hkv)))
    Q, K, V = fa.quantize_qkv_fused(q, k, v)
    pages = fa.KVPages.empty(3, 3, 4, page, device=dev)
    held, granted = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 0, 0], [0, 0, 0]))
    wanted = torch.tensor([250, 200, 300], dtype=torch.int32, device=dev)
    fa.resize_kv_pages(pages, held, wanted, granted=granted)
    with pytest.raises(RuntimeError, match="code 2 .*site 125,"):
        fa.check_status(dev)
    assert granted.tolist() == [250, 200, 0] and pages.table.tolist() == [[0, 1, -1], [2, 3, -1], [-1, -1, -1]]

    def call(used, rows, **kw):
        return fa.flash_attn_fp4_func(Q.data[:rows], K.data, V.data, Q.sf[:rows], K.sf, V.sf, Q.scale, K.scale, V.scale, causal=True, return_lse=True,
                                      seqused_k=used[:rows], page_table=pages.table[:rows], **kw)
    for kw in (dict(), dict(variant=fa.VARIANT_WS64), dict(variant=fa.VARIANT_WS)):
        out, lse = (x.clone() for x in call(granted, 3, **kw))
        torch.cuda.synchronize()
        fa.check_status(dev)
        assert not out[2].any() and (lse[2] == -float("inf")).all()
        want = call(wanted, 2, **kw)
        fa.check_status(dev)
        assert torch.equal(out[:2], want[0]) and torch.equal(lse[:2], want[1])
        got = call(wanted, 3, **kw)
        with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
            fa.check_status(dev)
        assert torch.equal(got[0][:2], want[0]) and not got[0][2].any()
