"""Pages of a KV cache where the pool runs out: what a row holds it goes on holding, and a later call finds it as it was.  Tables, counts, pairs and
granted lengths against plain loops, contents through the tables; everything is whole numbers or bytes and is compared for equality."""
import random
from collections import Counter

import pytest
import torch

import flash_attention_b200 as fa

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def reported(device, site):
    """Whether calls so far have recorded a bad index, which has to be one of `site`."""
    try:
        fa.check_status(device)
    except RuntimeError as e:
        assert "code 2 " in str(e) and f"site {site}," in str(e), e
        return True
    return False


def test_lengths_outside_the_table_are_reported(cuda_device):
    """Cut, and never without a word: held too."""
    dev = cuda_device
    for held, wanted, table, refs in ((99, 32, [0, 1], [1, 1, 0]), (33, 33, [0, 1], [1, 1, 0]), (2 ** 31 - 1, 3, [0, -1], [1, 0, 0]), (32, 33, [0, 1], [1, 1, 0]),
                                      (-1, 0, [-1, -1], [0, 0, 0]), (32, -1, [-1, -1], [0, 0, 0])):
        pages = fa.KVPages(i32([[0, 1]], dev), i32([1, 1, 0], dev), 16)
        fa.resize_kv_pages(pages, i32([held], dev), i32([wanted], dev))
        assert reported(dev, 124)
        assert pages.table.tolist() == [table] and pages.refs.tolist() == refs
    fa.resize_kv_pages(fa.KVPages(i32([[0, 1]], dev), i32([1, 1, 0], dev), 16), i32([32], dev), i32([32], dev))
    assert not reported(dev, 124)


# ---- entries that are missing among what a row holds ------------------------------------------------------------

def test_a_gap_is_not_filled_without_a_word(cuda_device):
    """Entry 1 of the first row has no page although it holds tokens there: nothing that could be put there is what it holds."""
    dev = cuda_device
    for wanted, row0, refs, first in ((50, [0, -1, 2, -1], [1, 1, 1, 1, 0, 0], 3),       # (grows: gets nothing)
                                      (40, [0, -1, 2, -1], [1, 1, 1, 1, 0, 0], 3),       # (stays)
                                      (20, [0, -1, -1, -1], [1, 1, 1, 0, 0, 0], 2)):     # (loses what is behind)
        pages = fa.KVPages(i32([[0, -1, 2, -1], [1, -1, -1, -1]], dev), i32([1, 1, 1, 0, 0, 0], dev), 16)
        pairs = fa.resize_kv_pages(pages, i32([40, 5], dev), i32([wanted, 20], dev))
        assert reported(dev, 125)
        assert pages.table.tolist() == [row0, [1, first, -1, -1]] and pages.refs.tolist() == refs and pairs.tolist() == [[-1, -1]] * 2
    # cut in front of the gap, or ended, it is a row like others
    for wanted, row0 in ((16, [0, -1, -1, -1]), (3, [0, -1, -1, -1]), (0, [-1] * 4)):
        pages = fa.KVPages(i32([[0, -1, 2, -1]], dev), i32([1, 0, 1], dev), 16)
        fa.resize_kv_pages(pages, i32([40], dev), i32([wanted], dev))
        assert pages.table.tolist() == [row0] and pages.refs.tolist() == [int(row0[0] == 0), 0, 0]
    pages = fa.KVPages(i32([[0, -1, 2, -1]], dev), i32([1, 0, 1], dev), 16)
    fa.resize_kv_pages(pages, i32([16], dev), i32([40], dev))
    assert pages.table.tolist() == [[0, 1, 2, -1]] and not reported(dev, 125)


def test_a_gap_where_a_warp_looks_for_it(cuda_device):
    """The first of several gaps, in each group of entries that a row is read in; a page that others share is not copied for such a row."""
    dev = cuda_device
    width, size = 300, 16
    for gap in (0, 1, 31, 32, 63, 127, 128, 200, 298):
        row = list(range(299)) + [-1]
        row[gap] = -1
        if gap < 297:
            row[gap + 2] = -1
        table = [row, [298] + [-1] * 299]
        refs = [int(p in row) + int(p == 298) for p in range(310)]
        pages = fa.KVPages(i32(table, dev), i32(refs, dev), size)
        pairs = fa.resize_kv_pages(pages, i32([298 * 16 + 4, 4], dev), i32([300 * 16, 4], dev))
        assert reported(dev, 125)
        assert pages.table.tolist() == table and pages.refs.tolist() == refs and pairs.tolist() == [[-1, -1]] * 2
