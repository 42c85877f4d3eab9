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


WAITS = -2 ** 31                 # on the page of an entry that must not be written to


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
    told = i32([0, 0], dev)
    for wanted, row0, refs, first, granted in ((50, [0, -1, 2, -1], [1, 1, 1, 1, 0, 0], 3, told),       # (grows: gets nothing)
                                               (50, [0, -1, WAITS + 2, -1], [1, 1, 1, 1, 0, 0], 3, None),
                                               (48, [0, -1, WAITS + 2, -1], [1, 1, 1, 1, 0, 0], 3, None),
                                               (40, [0, -1, 2, -1], [1, 1, 1, 1, 0, 0], 3, None),       # (stays)
                                               (20, [0, -1, -1, -1], [1, 1, 1, 0, 0, 0], 2, None)):     # (loses what is behind)
        pages = fa.KVPages(i32([[0, -1, 2, -1], [1, -1, -1, -1]], dev), i32([1, 1, 1, 0, 0, 0], dev), 16)
        pairs = fa.resize_kv_pages(pages, i32([40, 5], dev), i32([wanted, 20], dev), granted=granted)
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
        for granted in (None, i32([0, 0], dev)):
            pairs = fa.resize_kv_pages(pages, i32([298 * 16 + 4, 4], dev), i32([300 * 16, 4], dev), granted=granted)
            assert reported(dev, 125)
            if granted is None and gap != 298:
                assert pages.table[0, 298] == WAITS + row[298]
        assert granted.tolist() == [gap * 16, 4]
        assert pages.table.tolist() == table and pages.refs.tolist() == refs and pairs.tolist() == [[-1, -1]] * 2


def test_a_row_with_a_gap_is_not_appended_to(cuda_device):
    """It shares the page its next token would go to; whoever is not told appends all the same."""
    dev = cuda_device
    H, D, size = 2, 64, 16
    g = torch.Generator(device=dev).manual_seed(4)
    cache = fa.FP8KVCache.empty(4, size, H, D, device=dev)
    for t in cache.tensors():
        t.view(torch.uint8).copy_(torch.randint(0, 0x70, t.view(torch.uint8).shape, generator=g, device=dev, dtype=torch.uint8))
    cache.k_scale.fill_(0.5)
    cache.v_scale.fill_(0.5)
    before = [t.view(torch.uint8).clone() for t in cache.tensors()]
    pages = fa.KVPages(i32([[0, -1, 2], [1, 3, 2]], dev), i32([1, 1, 2, 1], dev), size)
    held = i32([40, 44], dev)
    pairs = fa.resize_kv_pages(pages, held, held + i32([1, 0], dev))
    assert reported(dev, 125)
    fa.copy_kv_pages(cache, pairs)
    k, v = (torch.randn(2, 1, H, D, generator=g, device=dev).bfloat16() * 100 for _ in range(2))
    fa.append_kv_fp8(cache, k, v, held, page_table=pages.table, seqused_new=i32([1, 0], dev))
    assert reported(dev, 121)
    assert all(torch.equal(t.view(torch.uint8), x) for t, x in zip(cache.tensors(), before))


# ---- copies that find no page ------------------------------------------------------------------------------------

class Model:
    """The book-keeping as lists."""

    def __init__(self, table, refs, size):
        self.table, self.refs, self.size = [list(r) for r in table], list(refs), size

    def count(self, tokens):
        return -(-tokens // self.size)

    def resize(self, held, wanted):
        """(pairs, granted lengths, whether something was missing)"""
        rows = range(len(self.table))
        for row, h, w in zip(self.table, held, wanted):
            for j in range(self.count(min(h, w)), len(row)):
                if row[j] >= 0:
                    self.refs[row[j]] -= 1
                    row[j] = -1
        gaps = [next((j for j in range(self.count(min(h, w))) if row[j] < 0), None) for row, h, w in zip(self.table, held, wanted)]
        writes = [self.table[b][held[b] // self.size] if gaps[b] is None and wanted[b] > held[b] and held[b] % self.size else -1 for b in rows]
        copied = [p >= 0 and writes[:b].count(p) < self.refs[p] - 1 for b, p in enumerate(writes)]
        free = [p for p, r in enumerate(self.refs) if r == 0]
        pairs, granted, failed, missing, self.refused = [], [], [], False, []
        for b in rows:
            row, at = self.table[b], held[b] // self.size
            pair, room = [-1, -1], wanted[b]
            if gaps[b] is not None:
                room, missing = gaps[b] * self.size, True
            elif (copied[b] and not free) or writes[b] in failed:
                failed.append(writes[b])
                self.refused.append(b)
                room, missing = held[b], True
            else:
                for j in range(self.count(wanted[b])):
                    if row[j] < 0 or (copied[b] and j == at):
                        if not free:
                            room, missing = min(room, j * self.size), True
                            continue
                        page = free.pop(0)
                        self.refs[page] = 1
                        if copied[b] and j == at:
                            pair = [row[j], page]
                            self.refs[row[j]] -= 1
                        row[j] = page
            pairs.append(pair)
            granted.append(room)
        return pairs, granted, missing

    def fork(self, held, parents):
        children = Counter(parents)
        for a, (row, h) in enumerate(zip(self.table, held)):
            for j, p in enumerate(row):
                if p >= 0:
                    self.refs[p] += children[a] - 1 if j < self.count(h) else -1
        width = len(self.table[0])
        self.table = [[-1] * width if a < 0 else [p if j < self.count(held[a]) else -1 for j, p in enumerate(self.table[a])] for a in parents]
        return [0 if a < 0 else held[a] for a in parents]

    def check(self):
        named = Counter(p for row in self.table for p in row if p >= 0)
        assert self.refs == [named[p] for p in range(len(self.refs))]


def test_entries_that_wait_for_a_copy(cuda_device):
    """Rows that were not told go through every call: what they name is counted, moved and given back like other entries."""
    dev = cuda_device

    def made():
        pages = fa.KVPages(i32([[2, 1, -1], [2, 1, -1], [0, -1, -1]], dev), i32([1, 2, 2], dev), 16)
        fa.resize_kv_pages(pages, i32([25, 20, 16], dev), i32([26, 21, 16], dev))
        assert reported(dev, 125)
        assert pages.table.tolist() == [[2, WAITS + 1, -1], [2, WAITS + 1, -1], [0, -1, -1]] and pages.refs.tolist() == [1, 2, 2]
        return pages
    # no growth: entries like others again, with nothing to copy
    pages = made()
    assert fa.resize_kv_pages(pages, i32([25, 20, 16], dev), i32([25, 18, 16], dev)).tolist() == [[-1, -1]] * 3
    assert pages.table.tolist() == [[2, 1, -1], [2, 1, -1], [0, -1, -1]] and pages.refs.tolist() == [1, 2, 2]
    # cut in front of it, ended
    pages = made()
    fa.resize_kv_pages(pages, i32([25, 20, 16], dev), i32([3, 0, 16], dev))
    assert pages.table.tolist() == [[2, -1, -1], [-1, -1, -1], [0, -1, -1]] and pages.refs.tolist() == [1, 0, 1]
    # alone with it: written to as it is
    pages = made()
    assert fa.resize_kv_pages(pages, i32([25, 20, 16], dev), i32([26, 0, 16], dev)).tolist() == [[-1, -1]] * 3
    assert pages.table.tolist() == [[2, 1, -1], [-1, -1, -1], [0, -1, -1]] and pages.refs.tolist() == [1, 1, 1]
    # forked: shared by one more, or one less
    pages = made()
    pages, held = fa.fork_kv_pages(pages, i32([25, 20, 16], dev), i32([0, 0, 1, 0], dev))
    assert pages.table.tolist() == [[2, 1, -1]] * 4 and held.tolist() == [25, 25, 20, 25] and pages.refs.tolist() == [0, 4, 4]
    pages, held = fa.fork_kv_pages(made(), i32([25, 20, 16], dev), i32([2], dev))
    assert pages.table.tolist() == [[0, -1, -1]] and pages.refs.tolist() == [1, 0, 0]
    # moved: pages 3 to 5 of six, the first waited for
    pages = fa.KVPages(i32([[4, WAITS + 3], [4, WAITS + 3], [5, -1]], dev), i32([0, 0, 0, 2, 2, 1], dev), 16)
    pairs, used = fa.compact_kv_pages(pages)
    assert pairs.tolist() == [[3, 0], [4, 1], [5, 2]] and used.tolist() == [3]
    assert pages.table.tolist() == [[1, WAITS], [1, WAITS], [2, -1]] and pages.refs.tolist() == [2, 2, 1, 0, 0, 0]
    fa.check_status(dev)
    # numbers that no pool has
    pages = fa.KVPages(i32([[WAITS + 9, 0]], dev), i32([1, 0, 0], dev), 16)
    fa.resize_kv_pages(pages, i32([0], dev), i32([0], dev))
    assert reported(dev, 123) and pages.table.tolist() == [[-1, -1]] and pages.refs.tolist() == [0, 0, 0]
    pages = fa.KVPages(i32([[WAITS + 9, 0]], dev), i32([1, 0, 0], dev), 16)
    new, _ = fa.fork_kv_pages(pages, i32([32], dev), i32([0], dev))
    assert reported(dev, 123) and new.table.tolist() == [[-1, 0]] and new.refs.tolist() == [1, 0, 0]


def both(pages, model, held, wanted, device, told=True):
    """The call and the model's, compared; the pairs and what was granted."""
    granted = torch.full((len(held),), -7, dtype=torch.int32, device=device) if told else None
    pairs = fa.resize_kv_pages(pages, i32(held, device), i32(wanted, device), granted=granted)
    want, room, missing = model.resize(held, wanted)
    assert pairs.tolist() == want and (not told or granted.tolist() == room)
    table = [list(row) for row in model.table]
    if not told:
        for b in model.refused:
            table[b][held[b] // model.size] += WAITS               # (no row has a gap)
    assert pages.table.tolist() == table and pages.refs.tolist() == model.refs
    assert reported(device, 125) == missing
    model.check()
    return pairs, room


def test_a_copy_that_finds_no_page_can_be_asked_for_again(cuda_device):
    """Two rows share a page that both are to write to, and there is none for the copy.  Both go on holding it and do not grow; once a third row has ended
    the same call makes the copy."""
    dev = cuda_device
    pages = fa.KVPages(i32([[0, -1], [0, -1], [1, -1]], dev), i32([2, 1], dev), 16)
    for granted in (None, i32([0] * 3, dev)):
        pairs = fa.resize_kv_pages(pages, i32([9, 9, 4], dev), i32([10, 10, 4], dev), granted=granted)
        assert reported(dev, 125)
        first = 0 if granted is not None else WAITS
        assert pages.table.tolist() == [[first, -1], [first, -1], [1, -1]] and pages.refs.tolist() == [2, 1] and pairs.tolist() == [[-1, -1]] * 3
    fa.resize_kv_pages(pages, i32([9, 9, 4], dev), i32([10, 10, 4], dev))
    assert reported(dev, 125)
    pairs = fa.resize_kv_pages(pages, i32([9, 9, 4], dev), i32([10, 10, 0], dev))
    assert pages.table.tolist() == [[1, -1], [0, -1], [-1, -1]] and pages.refs.tolist() == [1, 1] and pairs.tolist() == [[0, 1], [-1, -1], [-1, -1]]
    assert not reported(dev, 125)


def test_what_is_granted(cuda_device):
    dev = cuda_device
    for table, refs, held, wanted, granted in (
            ([[0, -1], [0, -1], [1, -1]], [2, 1], [9, 9, 4], [10, 10, 4], [9, 9, 4]),
            ([[0, -1], [0, -1], [1, -1]], [2, 1], [9, 9, 4], [10, 10, 0], [10, 10, 0]),
            ([[0, -1], [0, -1], [1, -1]], [2, 1, 0], [9, 9, 4], [10, 30, 6], [10, 16, 6]),        # (the last page is the copy; the keeper gets no other)
            ([[0, -1], [0, -1], [0, -1]], [3, 0], [9, 9, 9], [10, 10, 10], [10, 9, 9]),           # (one of two copies: the keeper waits for the other)
            ([[0, -1], [0, -1], [0, -1]], [3, 0], [9, 12, 9], [10, 12, 10], [10, 12, 9]),         # (one that does not write has it too)
            ([[0, -1], [0, -1], [1, -1], [1, -1]], [2, 2, 0], [9, 9, 3, 5], [10, 10, 4, 6], [10, 10, 3, 5]),
            ([[-1, -1, -1], [0, -1, -1]], [1, 0, 0], [0, 16], [48, 20], [32, 16]),                # (fresh pages alone)
            ([[0, -1, 2], [1, -1, -1]], [1, 1, 1, 0], [40, 16], [41, 17], [16, 17]),              # (a gap)
            ([[0, 1, -1]], [1, 1], [20, ], [25], [25]),
            ([[0, 1, -1]], [1, 1], [20, ], [3], [3]),
            ([[0, 1, -1]], [1, 1], [20, ], [0], [0])):
        model = Model(table, refs, 16)
        _, got = both(fa.KVPages(i32(table, dev), i32(refs, dev), 16), model, held, wanted, dev)
        assert got == granted
    # held beyond the table is cut first
    got = torch.zeros(1, dtype=torch.int32, device=dev)
    fa.resize_kv_pages(fa.KVPages(i32([[0, 1]], dev), i32([1, 1], dev), 16), i32([99], dev), i32([99], dev), granted=got)
    assert got.tolist() == [32]
    with pytest.raises(RuntimeError, match="code 2 .*site 124,"):
        fa.check_status(dev)


@pytest.mark.parametrize("B,width,pool,size", [(6, 3, 6, 16), (40, 5, 45, 16), (200, 9, 260, 48), (9, 40, 80, 16), (600, 3, 600, 32), (33, 70, 300, 64)])
@pytest.mark.parametrize("told", [True, False])
def test_nothing_that_is_held_is_lost(cuda_device, B, width, pool, size, told):
    """Rows that are forked, cut, grown and ended in a pool that is too small, the writers appending what was granted: every row reads back what it holds.
    Without `granted` the entries that must not be written to are marked."""
    dev, rng = cuda_device, random.Random(str((B, width)))
    model = Model([[-1] * width for _ in range(B)], [0] * pool, size)
    pages = fa.KVPages.empty(B, width, pool, size, device=dev)
    data = torch.full((pool, size), -1, dtype=torch.int64, device=dev)
    held, story, fresh, short, refused = [0] * B, [[] for _ in range(B)], 0, 0, 0
    for step in range(20):
        if step % 2 == 1:
            parents = [rng.choice([b, rng.randrange(B)]) for b in range(B)]
            pages, now = fa.fork_kv_pages(pages, i32(held, dev), i32(parents, dev))
            held = model.fork(held, parents)
            assert now.tolist() == held and pages.table.tolist() == model.table and pages.refs.tolist() == model.refs
            story = [list(story[a]) for a in parents]
        most = width * size
        wanted = [rng.choice([h, min(most, h + 1), min(most, h + 1), min(most, h + rng.randint(1, most // 3)), rng.randint(0, h) if rng.random() < 0.3 else h,
                              0 if rng.random() < 0.1 else h]) for h in held]
        pairs, room = both(pages, model, held, wanted, dev, told)
        fa.copy_kv_pages(data, pairs)
        short += sum(r < w for r, w in zip(room, wanted))
        refused += sum(r == h < w and h % size > 0 for h, r, w in zip(held, room, wanted))
        # (what is granted is never less than what is held and wanted: no row has a gap)
        assert all(min(h, w) <= r <= w for h, w, r in zip(held, wanted, room))
        where, what = [], []
        for b in range(B):
            story[b] = story[b][:room[b]]
            for t in range(held[b], room[b]):
                where.append(model.table[b][t // size] * size + t % size)
                what.append(fresh)
                story[b].append(fresh)
                fresh += 1
        assert len(set(where)) == len(where)                   # (no two rows write to one place)
        if where:
            data.view(-1)[torch.tensor(where, device=dev)] = torch.tensor(what, device=dev)
        held = room
        flat = data.view(-1).tolist()
        for b in range(B):
            assert [flat[model.table[b][t // size] * size + t % size] for t in range(held[b])] == story[b]
    assert short > refused > 0                                  # (the pool did run out, for copies too)


def test_a_captured_step_in_a_pool_that_runs_out(cuda_device):
    """Fork, resize, copy and the lengths that were granted in a graph; rows end between replays, and the others go on."""
    dev, rng = cuda_device, random.Random(8)
    B, width, size, pool = 12, 4, 16, 20
    model = Model([[b // 2] + [-1] * (width - 1) for b in range(B)], [2 if p < B // 2 else 0 for p in range(pool)], size)
    first = fa.KVPages(i32(model.table, dev), i32(model.refs, dev), size)
    second = fa.KVPages(torch.empty_like(first.table), first.refs, size)
    held, now, room = [9] * B, [i32([9] * B, dev), i32([0] * B, dev)], i32([0] * B, dev)
    parents, grow = i32(list(range(B)), dev), i32([1] * B, dev)
    data = torch.randint(0, 256, (pool, size), dtype=torch.uint8, device=dev)
    want = data.clone()
    kept = [t.clone() for t in (first.table, first.refs, now[0], data)]

    def step():
        fa.fork_kv_pages(first, now[0], parents, out=(second, now[1]))
        fa.copy_kv_pages(data, fa.resize_kv_pages(second, now[1], (now[1] + grow).clamp(min=0), granted=room))
        first.table.copy_(second.table)
        now[0].copy_(room)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t, x in zip((first.table, first.refs, now[0], data), kept):
        t.copy_(x)
    torch.cuda.synchronize()
    reported(dev, 125)
    short = 0
    for i in range(20):
        p = [rng.choice([b, b, rng.randrange(B)]) for b in range(B)]
        by = [rng.choice([1, 1, 5, 9, -100 if rng.random() < 0.2 else 1]) for _ in range(B)]
        held = model.fork(held, p)
        wanted = [max(0, min(h + n, width * size)) for h, n in zip(held, by)]
        by = [w - h for h, w in zip(held, wanted)]
        parents.copy_(i32(p, dev))
        grow.copy_(i32(by, dev))
        graph.replay()
        pairs, held, missing = model.resize(held, wanted)
        for a, b in pairs:
            if a >= 0:
                want[b] = want[a]
        assert first.table.tolist() == model.table and first.refs.tolist() == model.refs and now[0].tolist() == held and torch.equal(data, want)
        assert reported(dev, 125) == missing
        model.check()
        short += missing
    assert 0 < short < 20


def test_attention_where_a_copy_found_no_page(cuda_device):
    """What is held is attended to as before while there is no page, and after the copy was made; the row that keeps the page is not written to by the other."""
    dev = cuda_device
    H, G, D, size = 2, 4, 64, 16
    g = torch.Generator(device=dev).manual_seed(3)
    cache = fa.FP8KVCache.empty(2, size, H, D, device=dev, indexed=True)
    pages = fa.KVPages.empty(2, 2, 2, size, device=dev)
    def rows(n, s, h=H):
        return torch.randn(n, s, h, D, generator=g, device=dev).bfloat16()
    held, k, v, q = i32([9, 4], dev), rows(2, 9), rows(2, 9), rows(3, 1, G)
    fa.resize_kv_pages(pages, torch.zeros_like(held), held)
    fa.append_kv_fp8(cache, k, v, torch.zeros_like(held), page_table=pages.table, seqused_new=held)
    pages, held = fa.fork_kv_pages(pages, held, i32([0, 0, 1], dev))
    alone = fa.flash_attn_fp8_cache_func(q, cache, held, page_table=pages.table, causal=True)[0].clone()
    bytes_of = [t.view(torch.uint8).clone() for t in cache.tensors()]
    k1, v1 = rows(3, 1), rows(3, 1)
    # a caller who is not told appends to all, which changes nothing of what is held: the step can be done again
    pairs = fa.resize_kv_pages(pages, held, held + i32([1, 1, 0], dev))
    assert reported(dev, 125)
    fa.copy_kv_pages(cache, pairs)
    fa.append_kv_fp8(cache, k1, v1, held, page_table=pages.table, seqused_new=i32([1, 1, 0], dev))
    assert reported(dev, 121)
    assert all(torch.equal(t.view(torch.uint8), x) for t, x in zip(cache.tensors(), bytes_of))
    fa.flash_attn_fp8_cache_func(q, cache, held, page_table=pages.table, causal=True)
    assert reported(dev, 121)
    granted = torch.empty_like(held)
    pairs = fa.resize_kv_pages(pages, held, held + i32([1, 1, 0], dev), granted=granted)
    assert reported(dev, 125) and granted.tolist() == [9, 9, 4]
    fa.copy_kv_pages(cache, pairs)
    k, v = rows(3, 1), rows(3, 1)
    fa.append_kv_fp8(cache, k, v, held, page_table=pages.table, seqused_new=granted - held)
    assert all(torch.equal(t.view(torch.uint8), x) for t, x in zip(cache.tensors(), bytes_of))
    assert torch.equal(fa.flash_attn_fp8_cache_func(q, cache, granted, page_table=pages.table, causal=True)[0], alone)
    pairs = fa.resize_kv_pages(pages, held, i32([10, 10, 0], dev), granted=granted)
    assert granted.tolist() == [10, 10, 0] and pairs.tolist() == [[0, 1], [-1, -1], [-1, -1]]
    fa.copy_kv_pages(cache, pairs)
    fa.append_kv_fp8(cache, k, v, held, page_table=pages.table, seqused_new=granted - held)
    # the same tokens in caches of their own
    own = fa.FP8KVCache.empty(2, size, H, D, device=dev, indexed=True)
    for name, x in zip(("k", "v", "k_scale", "v_scale", "key_bounds", "bound_scale"), bytes_of):
        getattr(own, name).view(torch.uint8).copy_(x[:1].expand_as(x))
    fa.append_kv_fp8(own, k[:2], v[:2], held[:2])
    want = fa.flash_attn_fp8_cache_func(q[:2], own, granted[:2], causal=True)[0]
    assert torch.equal(fa.flash_attn_fp8_cache_func(q, cache, granted, page_table=pages.table, causal=True)[0][:2], want)
    fa.check_status(dev)


def test_a_loop_in_a_pool_that_runs_out(cuda_device):
    """The calls of a serving loop where there are too few pages: rows go on from others, end, are refused room and ask again.  Lists and results are those of caches
    that every row has to itself."""
    dev, rng = cuda_device, random.Random(6)
    H, G, D, size, width, pool, W, first = 2, 8, 64, 16, 8, 9, 4, 20
    g = torch.Generator().manual_seed(7)
    def rows(n, heads, s=1):
        return torch.randn(n, s, heads, D, generator=g).bfloat16().to(dev)
    cache = fa.FP8KVCache.empty(pool, size, H, D, device=dev, indexed=True, by_head=True)
    pages, held = fa.KVPages.empty(1, width, pool, size, device=dev), i32([0], dev)
    k0, v0 = rows(1, H, first), rows(1, H, first)
    fa.copy_kv_pages(cache, fa.resize_kv_pages(pages, held, held + first))
    fa.append_kv_fp8(cache, k0, v0, held, page_table=pages.table)
    pages, held = fa.fork_kv_pages(pages, held + first, i32([0] * W, dev))
    story, short, ended = [[] for _ in range(W)], 0, [False] * W
    for step in range(60):
        q, k, v = rows(W, G), rows(W, H), rows(W, H)
        here = held.tolist()
        end = [not e and h > first and rng.random() < 0.06 and not all(ended) for e, h in zip(ended, here)]
        wanted = [0 if e or now or h >= 90 else h + 1 for e, now, h in zip(ended, end, here)]
        ended = [w == 0 for w in wanted]
        room = torch.empty_like(held)
        fa.copy_kv_pages(cache, fa.resize_kv_pages(pages, held, i32(wanted, dev), granted=room))
        fa.append_kv_fp8(cache, k, v, held, page_table=pages.table, seqused_new=room - held)
        granted = room.tolist()
        missing = granted != wanted
        assert reported(dev, 125) == missing
        short += missing
        for b in range(W):
            assert granted[b] in (wanted[b], here[b])
            story[b] = [] if ended[b] else story[b] + [(k[b, 0], v[b, 0])] * (granted[b] - here[b])
            assert ended[b] or len(story[b]) + first == granted[b]
        lists = fa.select_kv_blocks(q, cache, room, 3, page_table=pages.table)
        out, lse = fa.flash_attn_fp8_blocks_func(q, cache, lists, room, page_table=pages.table, return_lse=True)
        fa.check_status(dev)
        if step % 7 == 6:
            own = fa.FP8KVCache.empty(W, width * size, H, D, size, device=dev, indexed=True)
            there = [0 if e else 1 for e in ended]
            fa.append_kv_fp8(own, k0.expand(W, -1, -1, -1).contiguous(), v0.expand(W, -1, -1, -1).contiguous(), i32([0] * W, dev), seqused_new=i32([first * t for t in there], dev))
            for i in range(max(len(s) for s in story)):
                t = [torch.stack([s[i][j] if i < len(s) else torch.zeros_like(k[0, 0]) for s in story])[:, None] for j in (0, 1)]
                fa.append_kv_fp8(own, *t, i32([first + i] * W, dev), seqused_new=i32([int(i < len(s)) for s in story], dev))
            mine = fa.select_kv_blocks(q, own, room, 3)
            want, want_lse = fa.flash_attn_fp8_blocks_func(q, own, mine, room, return_lse=True)
            assert torch.equal(lists, mine) and torch.equal(out, want) and torch.equal(lse, want_lse)
        held = room
        # (rows that ended begin again as another one, some time later)
        alive = [b for b in range(W) if not ended[b]]
        parents = [b if not ended[b] else rng.choice(alive) if alive and rng.random() < 0.3 else -1 for b in range(W)]
        pages, held = fa.fork_kv_pages(pages, held, i32(parents, dev))
        story = [list(story[a]) if a >= 0 else [] for a in parents]
        ended = [a < 0 for a in parents]
        if all(ended):
            break
    assert short > 5


def test_refusals_of_granted(cuda_device):
    dev = cuda_device
    p, n = fa.KVPages.empty(3, 4, 10, 16, device=dev), i32([0, 0, 0], dev)
    for bad in (n.clone().long(), n.clone()[:2], n.cpu(), n.clone()[None], torch.zeros(6, dtype=torch.int32, device=dev)[::2]):
        with pytest.raises(AssertionError, match="granted"):
            fa.resize_kv_pages(p, n, n + 1, granted=bad)
    for bad in (n, p.table.view(-1)[:3], p.refs[:3]):
        with pytest.raises(AssertionError, match="overlap"):
            fa.resize_kv_pages(p, n, n + 1, granted=bad)
    wanted = n + 1
    with pytest.raises(AssertionError, match="overlap"):
        fa.resize_kv_pages(p, n, wanted, granted=wanted)
    none = fa.KVPages(p.table[:0], p.refs, 16)
    assert fa.resize_kv_pages(none, n[:0], n[:0], granted=n.clone()[:0]).shape == (0, 2)
    assert not p.refs.any() and (p.table == -1).all()
    fa.check_status(dev)
