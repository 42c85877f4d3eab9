"""The index of pages that sequences of one call share, against the oracle's whole numbers."""
import pytest

import flash_attention_b200 as fa
from tests.test_gpu_fp8_blocks import i32, index_of, indexed, same_index
from tests.test_gpu_fp8_cache import fill, make_cache

pytestmark = pytest.mark.gpu


def test_index_of_pages_that_sequences_share(cuda_device):
    """Sequences that share pages and hold the same of them write the same bounds; each alone gives these too."""
    dev = cuda_device
    H, D, size, block = 3, 128, 64, 32
    cache = indexed(make_cache(8, size, H, D, block, 1, dev))
    tables, held = [[5, 2, 7], [5, 2, 0], [5, 2, 7], [5, 1, 3]], [150, 140, 150, 190]
    fill(cache, [[5, 2, 7], [5, 2, 0], [5, 1, 3]], [192, 192, 192], 4, spread=8.0)
    want = index_of(cache, tables, [(0, n) for n in held])
    for _ in range(3):
        fa.index_kv_fp8(cache, i32([0] * 4, dev), 190, page_table=i32(tables, dev), seqused_new=i32(held, dev))
        same_index(cache, want)
    cache.key_bounds.fill_(77)
    cache.bound_scale.fill_(77.0)
    for b in range(4):
        fa.index_kv_fp8(cache, i32([0], dev), 190, page_table=i32([tables[b]], dev), seqused_new=i32([held[b]], dev))
    same_index(cache, want)
    fa.check_status(dev)
