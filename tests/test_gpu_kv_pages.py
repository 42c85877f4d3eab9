"""Pages of a KV cache on the GPU: tables, reference counts and copies against plain loops.  Everything is whole numbers or bytes and is
compared for equality."""
import random

import pytest
import torch

import flash_attention_b200 as fa

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


class Model:
    """The same book-keeping as lists."""

    def __init__(self, table, refs, size):
        self.table, self.refs, self.size = [list(r) for r in table], list(refs), size

    def count(self, tokens):
        return -(-tokens // self.size)

    def resize(self, held, wanted):
        for row, h, w in zip(self.table, held, wanted):
            for j in range(self.count(min(h, w)), len(row)):
                if row[j] >= 0:
                    self.refs[row[j]] -= 1
                    row[j] = -1
        writes = [row[h // self.size] if w > h and h % self.size else -1 for row, h, w in zip(self.table, held, wanted)]
        copied = [p >= 0 and writes[:b].count(p) < self.refs[p] - 1 for b, p in enumerate(writes)]
        free = iter([p for p, r in enumerate(self.refs) if r == 0])
        pairs = []
        for b, (row, h, w) in enumerate(zip(self.table, held, wanted)):
            pair = [-1, -1]
            for j in range(self.count(w)):
                mine = copied[b] and j == h // self.size
                if row[j] < 0 or mine:
                    row[j] = next(free, -1)
                    if row[j] >= 0:
                        self.refs[row[j]] = 1
                    if mine and row[j] >= 0:
                        pair = [writes[b], row[j]]
            if copied[b]:
                self.refs[writes[b]] -= 1
            pairs.append(pair)
        return pairs

    def fork(self, held, parents):
        children = [parents.count(a) for a in range(len(self.table))]
        for a, (row, h) in enumerate(zip(self.table, held)):
            for j, p in enumerate(row):
                if p >= 0:
                    self.refs[p] += children[a] - 1 if j < self.count(h) else -1
        width = len(self.table[0])
        self.table = [[-1] * width if a < 0 else [p if j < self.count(held[a]) else -1 for j, p in enumerate(self.table[a])] for a in parents]
        return [0 if a < 0 else held[a] for a in parents]

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p, r in enumerate(self.refs) if r <= 0 and p < used]
        movers = [p for p, r in enumerate(self.refs) if r > 0 and p >= used]
        to = dict(zip(movers, holes))
        for p, q in to.items():
            self.refs[q], self.refs[p] = self.refs[p], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return [list(x) for x in to.items()], used

    def check(self):
        named = [p for row in self.table for p in row if p >= 0]
        assert self.refs == [named.count(p) for p in range(len(self.refs))] if len(self.refs) < 3000 else True


def pages_of(model, device):
    return fa.KVPages(i32(model.table, device), i32(model.refs, device), model.size)


def same(pages, model):
    assert pages.table.tolist() == model.table
    assert pages.refs.tolist() == model.refs


def made(rng, B, width, pool, size, beams=1):
    """Sequences of random lengths, those of a request sharing some pages; pages in any order."""
    order = list(range(pool))
    rng.shuffle(order)
    at = iter(order)
    table, held = [], []
    for _ in range(B // beams):
        n = rng.randint(0, (width - 1) * size)
        common = [next(at) for _ in range(rng.randint(0, -(-n // size)))]
        for _ in range(beams):
            row = common + [next(at) for _ in range(-(-n // size) - len(common))]
            table.append(row + [-1] * (width - len(row)))
            held.append(n)
    refs = [0] * pool
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return Model(table, refs, size), held


SHAPES = [(1, 1, 1, 16), (1, 3, 40, 16), (4, 5, 64, 48), (33, 7, 400, 64), (64, 40, 3000, 16), (300, 4, 1500, 128), (9, 100, 1001, 32)]


@pytest.mark.parametrize("B,width,pool,size", SHAPES)
@pytest.mark.parametrize("beams", [1, 3])
def test_growing_and_shrinking(cuda_device, B, width, pool, size, beams):
    rng = random.Random(str((B, width, beams)))
    model, held = made(rng, max(B // beams, 1) * beams if width > 1 else B, width, pool, size, beams if width > 1 else 1)
    pages = pages_of(model, cuda_device)
    for i in range(4):
        most = width * size
        wanted = [rng.choice([h, min(most, h + 1), 0, rng.randint(0, h), rng.randint(0, most), min(most, h + size + 1)]) for h in held]
        if sum(model.count(w) for w in wanted) + len(held) > pool:
            wanted = held
        pairs = fa.resize_kv_pages(pages, i32(held, cuda_device), i32(wanted, cuda_device))
        assert pairs.tolist() == model.resize(held, wanted)
        same(pages, model)
        model.check()
        held = [rng.randint(0, w) if rng.random() < 0.3 else w for w in wanted]       # (room that was not used)
    fa.check_status(cuda_device)


@pytest.mark.parametrize("B,width,pool,size", SHAPES[1:])
def test_forks_and_what_they_write_to(cuda_device, B, width, pool, size):
    """Beams: rows go on from others, grow, go on; the pages they write to become theirs."""
    rng = random.Random(str((B, width)))
    model, held = made(rng, B, width, 4 * pool, size)
    pages = pages_of(model, cuda_device)
    for i in range(5):
        rows = rng.choice([B, B, max(1, B // 2), min(2 * B, 300)])
        parents = [rng.choice([-1] + [rng.randrange(len(held)) for _ in range(6)]) for _ in range(rows)]
        pages, now = fa.fork_kv_pages(pages, i32(held, cuda_device), i32(parents, cuda_device))
        held = model.fork(held, parents)
        assert now.tolist() == held
        same(pages, model)
        model.check()
        wanted = [min(width * size, h + rng.choice([1, 1, 2])) for h in held]
        pairs = fa.resize_kv_pages(pages, now, i32(wanted, cuda_device))
        assert pairs.tolist() == model.resize(held, wanted)
        same(pages, model)
        held = wanted
    fa.check_status(cuda_device)


def test_the_last_sharer_keeps_the_page_if_nobody_else_has_it(cuda_device):
    model = Model([[5], [5], [2], [5]], [0, 0, 1, 0, 0, 3, 0, 0], 16)
    for wanted, copies in (([4, 4, 4, 4], 2), ([4, 4, 4, 3], 2), ([3, 4, 4, 3], 1), ([0, 4, 4, 4], 1), ([4, 0, 0, 0], 0)):
        m = Model(model.table, model.refs, 16)
        pages = pages_of(m, cuda_device)
        pairs = fa.resize_kv_pages(pages, i32([3] * 4, cuda_device), i32(wanted, cuda_device))
        assert pairs.tolist() == m.resize([3] * 4, wanted)
        same(pages, m)
        assert sum(p[0] >= 0 for p in pairs.tolist()) == copies


def test_forks_between_two_tables(cuda_device):
    """Two tables that take turns, in a captured graph with the resize and the copy."""
    dev, rng = cuda_device, random.Random(4)
    model, held = made(rng, 12, 8, 300, 16, 4)
    first = pages_of(model, dev)
    now = [i32(held, dev), i32(held, dev)]
    data = torch.randint(0, 256, (300, 16, 3), dtype=torch.uint8, device=dev)
    want = data.clone()
    second = fa.KVPages(torch.empty_like(first.table), first.refs, 16)
    parents = i32([0] * 12, dev)
    def step():
        a, h = fa.fork_kv_pages(first, now[0], parents, out=(second, now[1]))
        assert a is second and h is now[1]
        h1 = now[1] + 1
        fa.copy_kv_pages(data, fa.resize_kv_pages(second, now[1], h1))
        fa.fork_kv_pages(second, h1, torch.arange(12, dtype=torch.int32, device=dev), out=(first, now[0]))
    kept = first.table.clone(), first.refs.clone(), now[0].clone(), data.clone()
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
    for _ in range(6):
        p = [b // 4 * 4 + rng.randrange(4) for b in range(12)]
        parents.copy_(i32(p, dev))
        graph.replay()
        held = model.fork(held, p)
        pairs = model.resize(held, [h + 1 for h in held])
        for a, b in pairs:
            if a >= 0:
                want[b] = want[a]
        held = [h + 1 for h in held]
        same(first, model)
        assert now[0].tolist() == held and torch.equal(data, want)
    fa.check_status(dev)


def test_nothing_is_left(cuda_device):
    """More is wanted than there is: the last entries get nothing, which is reported; a copy that finds no page is not asked for."""
    model = Model([[0, -1, -1], [0, -1, -1], [-1, -1, -1]], [2, 0, 0, 0], 16)
    for held, wanted in (([0, 0, 0], [48, 48, 48]), ([9, 9, 0], [10, 10, 48]), ([0, 16, 0], [48, 17, 16])):
        m = Model(model.table, model.refs, 16)
        pages = pages_of(m, cuda_device)
        pairs = fa.resize_kv_pages(pages, i32(held, cuda_device), i32(wanted, cuda_device))
        want = m.resize(held, wanted)
        assert pairs.tolist() == want
        same(pages, m)
        with pytest.raises(RuntimeError, match="code 2 .*site 125,"):
            fa.check_status(cuda_device)
    m = Model([[0, 1, -1, 2], [0, 1, 2, -1]], [2, 2, 2], 16)
    pages = pages_of(m, cuda_device)
    assert fa.resize_kv_pages(pages, i32([40, 40], cuda_device), i32([41, 41], cuda_device)).tolist() == m.resize([40, 40], [41, 41])
    same(pages, m)
    with pytest.raises(RuntimeError, match="code 2 .*site 125,"):              # (a row with a gap among what it holds)
        fa.check_status(cuda_device)


@pytest.mark.parametrize("B,width,pool,size", SHAPES)
def test_compacting(cuda_device, B, width, pool, size):
    rng = random.Random(str((B, pool)))
    model, held = made(rng, B, width, pool, size)
    data = torch.randint(0, 256, (pool, 5), dtype=torch.uint8, device=cuda_device)
    before = [[data[p].tolist() for p in row if p >= 0] for row in model.table]
    for i in range(2):
        pages = pages_of(model, cuda_device)
        pairs, used = fa.compact_kv_pages(pages)
        want, n = model.compact()
        assert used.tolist() == [n] and pairs.tolist() == want + [[-1, -1]] * (pool // 2 - len(want))
        same(pages, model)
        assert max((p for row in model.table for p in row), default=-1) < n
        fa.copy_kv_pages(data, pairs)
        assert [[data[p].tolist() for p in row if p >= 0] for row in pages.table.tolist()] == before
    fa.check_status(cuda_device)


@pytest.mark.parametrize("pool,share", [(100_000, 0.5), (70_001, 0.01), (65_536, 1.0), (300_007, 0.9)])
def test_large_pools(cuda_device, pool, share):
    """Pools of which a warp sees many pages, rows that want thousands; against torch's own sums."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(pool)
    live = torch.rand(pool, generator=g, device=dev) < share
    pages_in = live.nonzero()[:, 0].to(torch.int32)
    n = len(pages_in) // 50 * 50
    table = torch.full((50, max(n // 50, 1) + 300), -1, dtype=torch.int32, device=dev)
    table[:, :n // 50] = pages_in[torch.randperm(len(pages_in), generator=g, device=dev)][:n].view(50, -1)
    refs = torch.zeros(pool, dtype=torch.int32, device=dev).index_add_(0, table[table >= 0].long(), torch.ones(n, dtype=torch.int32, device=dev))
    pages = fa.KVPages(table.clone(), refs.clone(), 16)
    held = torch.full((50,), n // 50 * 16, dtype=torch.int32, device=dev)
    wanted = held + 300 * 16 if share < 1 else held
    fa.resize_kv_pages(pages, held, wanted)
    fa.check_status(dev)
    free = (refs == 0).nonzero()[:, 0].to(torch.int32)
    if share < 1:
        assert torch.equal(pages.table[:, n // 50:], free[:15000].view(50, 300)) and torch.equal(pages.table[:, :n // 50], table[:, :n // 50])
        assert (pages.refs[free[:15000].long()] == 1).all() and (pages.refs == 0).sum() == len(free) - 15000
    pages = fa.KVPages(table.clone(), refs.clone(), 16)
    pairs, used = fa.compact_kv_pages(pages)
    n = int((refs > 0).sum())
    assert used.item() == n
    holes, movers = (refs[:n] == 0).nonzero()[:, 0], (refs[n:] > 0).nonzero()[:, 0] + n
    assert torch.equal(pairs[:len(holes)].long(), torch.stack([movers, holes], dim=1)) and (pairs[len(holes):] == -1).all()
    to = torch.arange(pool, device=dev)
    to[movers] = holes
    assert torch.equal(pages.table, torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1))
    assert (pages.refs[:n] > 0).all() and (pages.refs[n:] == 0).all()


def test_the_most_rows(cuda_device):
    rng = random.Random(7)
    table = [[b // 8 if j == 0 else -1 for j in range(2)] for b in range(4096)]
    model = Model(table, [8 if p < 512 else 0 for p in range(9000)], 16)
    pages = pages_of(model, cuda_device)
    held, wanted = [5] * 4096, [rng.choice([5, 6, 30, 0]) for _ in range(4096)]
    assert fa.resize_kv_pages(pages, i32(held, cuda_device), i32(wanted, cuda_device)).tolist() == model.resize(held, wanted)
    same(pages, model)
    parents = [rng.randrange(4096) for _ in range(5000)]
    pages, now = fa.fork_kv_pages(pages, i32(wanted, cuda_device), i32(parents, cuda_device))
    assert now.tolist() == model.fork(wanted, parents)
    same(pages, model)
    with pytest.raises(NotImplementedError, match="4096"):
        fa.resize_kv_pages(pages, now, now)
    fa.check_status(cuda_device)


def test_bad_numbers_are_reported(cuda_device):
    dev = cuda_device
    def pages():
        return fa.KVPages(i32([[0, 1], [2, -1]], dev), i32([1, 1, 1, 0, 0], dev), 16)
    p = pages()
    fa.resize_kv_pages(p, i32([-3, 3], dev), i32([5, 40], dev))            # (cut at the table's end)
    with pytest.raises(RuntimeError, match="code 2 .*site 124,"):
        fa.check_status(dev)
    assert p.table.tolist() == [[0, -1], [2, 1]] and p.refs.tolist() == [1, 1, 1, 0, 0]
    p = pages()
    p.table[1, 1] = 99
    fa.resize_kv_pages(p, i32([32, 16], dev), i32([32, 32], dev))
    with pytest.raises(RuntimeError, match="code 2 .*site 123,"):
        fa.check_status(dev)
    assert p.table.tolist() == [[0, 1], [2, 3]]
    p = pages()
    q, held = fa.fork_kv_pages(p, i32([32, 9], dev), i32([1, 7, -2, 0, 1], dev))
    with pytest.raises(RuntimeError, match="code 2 .*site 126,"):
        fa.check_status(dev)
    assert q.table.tolist() == [[2, -1], [-1, -1], [-1, -1], [0, 1], [2, -1]] and held.tolist() == [9, 0, 0, 32, 9] and q.refs.tolist() == [1, 1, 2, 0, 0]
    p = pages()
    p.table[0, 1] = 5
    p.refs[1] = 0
    fa.compact_kv_pages(p)
    with pytest.raises(RuntimeError, match="code 2 .*site 123,"):
        fa.check_status(dev)
    assert p.table.tolist() == [[0, 5], [1, -1]]
    x = torch.arange(10, device=dev).view(5, 2)
    fa.copy_kv_pages(x, i32([[0, 5], [1, 3], [6, 4], [-1, 2], [2, -1]], dev))
    with pytest.raises(RuntimeError, match="code 2 .*site 127,"):
        fa.check_status(dev)
    assert x.tolist() == [[0, 1], [2, 3], [4, 5], [2, 3], [8, 9]]


@pytest.mark.parametrize("H,D,size,block", [(1, 64, 16, 16), (3, 128, 48, 16), (8, 128, 64, 64), (2, 64, 256, 128)])
@pytest.mark.parametrize("by_head", [False, True])
def test_copies_of_an_8_bit_cache(cuda_device, H, D, size, block, by_head):
    """Keys, values, scales and index of a page move together; the others stay."""
    cache = fa.FP8KVCache.empty(20, size, H, D, block, device=cuda_device, indexed=True, by_head=by_head)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    parts = [cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale.view(torch.uint8), cache.v_scale.view(torch.uint8), cache.key_bounds.view(torch.uint8),
             cache.bound_scale.view(torch.uint8)]
    for t in parts:
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=cuda_device, dtype=torch.uint8))
    pairs = [[3, 7], [-1, -1], [0, 19], [5, 1], [-1, 4], [3, 2], [11, 11]]
    want = [t.clone() for t in parts]
    for t in want:
        for a, b in pairs:
            if a >= 0:
                t[b] = t[a]
    fa.copy_kv_pages(cache, i32(pairs, cuda_device))
    for t, w in zip(parts, want):
        assert torch.equal(t, w)
    fa.check_status(cuda_device)


def test_copies_of_any_tensors(cuda_device):
    """Types, odd sizes, views that leave gaps, many tensors in one call."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(2)
    def random_bytes(*shape):
        return torch.randint(0, 256, shape, generator=g, device=dev, dtype=torch.uint8)
    whole = [random_bytes(9, 7, 5, 33), random_bytes(9, 64, 4, 128), random_bytes(9, 12, 48), random_bytes(9, 3), random_bytes(9, 1, 1), random_bytes(9, 100_000),
             random_bytes(10, 16, 6, 64), random_bytes(9, 0), random_bytes(9, 4, 8, 4, 8), random_bytes(40), random_bytes(9, 65_536)]
    views = [whole[0][:, 1:6, :, 2:30], whole[1].transpose(1, 2), whole[2].view(torch.float32)[:, ::2], whole[3], whole[4], whole[5][:, 1:99_998],
             whole[6][1:, :, 2:4].permute(0, 2, 1, 3), whole[7], whole[8].permute(0, 3, 1, 2, 4)[:, 0], whole[9][1:37:4], whole[10].view(torch.bfloat16)]
    pairs = [[0, 8], [4, 2], [4, 3], [1, 5]]
    want = [t.clone() for t in whole]
    again = [want[0][:, 1:6, :, 2:30], want[1].transpose(1, 2), want[2].view(torch.float32)[:, ::2], want[3], want[4], want[5][:, 1:99_998],
             want[6][1:, :, 2:4].permute(0, 2, 1, 3), want[7], want[8].permute(0, 3, 1, 2, 4)[:, 0], want[9][1:37:4], want[10].view(torch.bfloat16)]
    for t in again:
        for a, b in pairs:
            t[b] = t[a].clone()
    fa.copy_kv_pages(views, i32(pairs, dev))
    for t, w in zip(whole, want):
        assert torch.equal(t, w)
    fa.check_status(dev)


@pytest.mark.parametrize("page", [65536, 40016, 16384, 131088])
def test_large_copies(cuda_device, page):
    """From 64 MB on pages that lie in one piece go another way; beside them tensors that do not, pairs that are none, pairs outside the pool."""
    dev, n = cuda_device, 5000
    g = torch.Generator(device=dev).manual_seed(page)
    flat = torch.randint(0, 256, (n, page // 16, 16), generator=g, device=dev, dtype=torch.uint8)
    small = torch.randn(n, 8, generator=g, device=dev)
    odd = torch.randint(0, 256, (n, 5), generator=g, device=dev, dtype=torch.uint8)
    apart = torch.randn(n, 6, 8, 4, generator=g, device=dev)[:, :, ::2]
    order = torch.randperm(n, generator=g, device=dev).to(torch.int32)
    pairs = order.view(n // 2, 2).clone()
    pairs[torch.rand(n // 2, generator=g, device=dev) < 0.4] = -1
    pairs[7] = i32([3, -1], dev)
    pairs[-1] = i32([int(order[-2]), int(order[-1])], dev)
    real = pairs.long()[(pairs >= 0).all(1)]
    tensors = [flat, small, odd, apart]
    want = [t.clone() for t in tensors]
    for w, t in zip(want, tensors):
        w[real[:, 1]] = t[real[:, 0]]
    fa.copy_kv_pages(tensors, pairs)
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)
    fa.check_status(dev)
    # the same again, and with pairs outside the pool among them
    pairs[11] = i32([n, 0], dev)
    pairs[13] = i32([0, 2 ** 31 - 1], dev)
    before = flat[0].clone()
    fa.copy_kv_pages(tensors, pairs)
    with pytest.raises(RuntimeError, match="code 2 .*site 127,"):
        fa.check_status(dev)
    real = pairs.long()[((pairs >= 0) & (pairs < n)).all(1)]
    for w in want:
        w[real[:, 1]] = w[real[:, 0]]
    for t, w in zip(tensors, want):
        assert torch.equal(t, w)
    assert torch.equal(flat[0], before) or (real[:, 1] == 0).any()


def test_copies_that_pass_32_bits(cuda_device):
    dev = cuda_device
    if torch.cuda.mem_get_info(dev)[0] < 12 * 2 ** 30:
        pytest.skip("not enough memory")
    x = torch.zeros(100_000, 64, 1024, dtype=torch.uint8, device=dev)
    x[7], x[99_990] = 3, 5
    fa.copy_kv_pages(x, i32([[7, 99_999], [99_990, 1]], dev))
    assert (x[99_999] == 3).all() and (x[1] == 5).all() and int(x[99_998].sum()) + int(x[0].sum()) == 0
    # (and by bulk copies)
    pairs = torch.full((2000, 2), -1, dtype=torch.int32, device=dev)
    pairs[1999] = i32([99_999, 99_997], dev)
    pairs[5] = i32([1, 2], dev)
    fa.copy_kv_pages(x, pairs)
    assert (x[99_997] == 3).all() and (x[2] == 5).all() and int(x[99_998].sum()) + int(x[0].sum()) == 0
    fa.check_status(dev)


def test_refusals(cuda_device):
    dev = cuda_device
    p = fa.KVPages.empty(3, 4, 10, 16, device=dev)
    n = i32([0, 0, 0], dev)
    for bad, match in ((fa.KVPages(p.table.long(), p.refs, 16), "table"), (fa.KVPages(p.table[:, ::2], p.refs, 16), "table"), (fa.KVPages(p.table.cpu(), p.refs, 16), "table"),
                       (fa.KVPages(p.table, p.refs[::2], 16), "refs"), (fa.KVPages(p.table, p.refs.float(), 16), "refs"), (fa.KVPages(p.table, p.refs[:0], 16), "refs"),
                       (fa.KVPages(p.table, p.refs.cpu(), 16), "CUDA"), (fa.KVPages(p.table[:, :0], p.refs, 16), "table"), (fa.KVPages(p.table, p.refs, 1 << 30), "too large")):
        for call in (lambda: fa.resize_kv_pages(bad, n, n), lambda: fa.fork_kv_pages(bad, n, n), lambda: fa.compact_kv_pages(bad)):
            with pytest.raises(AssertionError, match=match):
                call()
    with pytest.raises(ValueError, match="page_size"):
        fa.resize_kv_pages(fa.KVPages(p.table, p.refs, 0), n, n)
    for bad in (n[:2], n.long(), n.cpu(), n[None]):
        with pytest.raises(AssertionError, match="held"):
            fa.resize_kv_pages(p, bad, n)
        with pytest.raises(AssertionError, match="wanted"):
            fa.resize_kv_pages(p, n, bad)
        with pytest.raises(AssertionError, match="held"):
            fa.fork_kv_pages(p, bad, n)
    with pytest.raises(AssertionError, match="overlap"):
        fa.fork_kv_pages(p, n, n, out=(p, n.clone()))
    other = fa.KVPages(torch.empty_like(p.table), p.refs, 16)
    with pytest.raises(AssertionError, match="overlap"):
        fa.fork_kv_pages(p, n, n.clone(), out=(other, n))
    with pytest.raises(ValueError, match="refs"):
        fa.fork_kv_pages(p, n, n, out=(fa.KVPages.empty(3, 4, 10, 16, device=dev), n.clone()))
    with pytest.raises(AssertionError, match="out table"):
        fa.fork_kv_pages(p, n, n[:2], out=(other, n.clone()))
    with pytest.raises(AssertionError, match="no rows"):
        fa.compact_kv_pages(fa.KVPages(p.table[:0], p.refs, 16))
    x = torch.zeros(10, 4, device=dev)
    pair = i32([[0, 1]], dev)
    for bad in (pair[0], pair.long(), pair[:, :1]):
        with pytest.raises(AssertionError, match="pairs"):
            fa.copy_kv_pages(x, bad)
    with pytest.raises(AssertionError, match="as many pages"):
        fa.copy_kv_pages([x, x[:9]], pair)
    with pytest.raises(AssertionError, match="one CUDA device"):
        fa.copy_kv_pages([x, x.cpu()], pair)
    with pytest.raises(AssertionError, match="expanded"):
        fa.copy_kv_pages(x[:, :1].expand(10, 4), pair)
    with pytest.raises(AssertionError, match="expanded"):
        fa.copy_kv_pages(x[:1].expand(10, 4), pair)
    with pytest.raises(NotImplementedError, match="separate"):
        fa.copy_kv_pages(torch.zeros(10, 4, 4, 4, 4, device=dev)[:, ::2, ::2, ::2, ::2], pair)
    with pytest.raises(AssertionError, match="no tensors"):
        fa.copy_kv_pages([], pair)
    # nothing to do
    fa.copy_kv_pages(x, pair[:0])
    none = fa.KVPages(p.table[:0], p.refs, 16)
    assert fa.resize_kv_pages(none, n[:0], n[:0]).shape == (0, 2)
    q, held = fa.fork_kv_pages(none, n[:0], n[:0])
    assert q.table.shape == (0, 4) and held.shape == (0,)
    with pytest.raises(ValueError, match="no parents"):
        fa.fork_kv_pages(none, n[:0], n)
    fa.resize_kv_pages(p, n, n + 20)
    q, held = fa.fork_kv_pages(p, n + 20, n[:0])                                # (everything is given back)
    assert q.table.shape == (0, 4) and not p.refs.any()
    fa.check_status(dev)


def test_another_stream(cuda_device):
    dev, rng = cuda_device, random.Random(9)
    model, held = made(rng, 20, 6, 400, 16, 4)
    s = torch.cuda.Stream()
    for _ in range(10):
        m = Model(model.table, model.refs, 16)
        pages, h = pages_of(m, dev), i32(held, dev)
        parents = [rng.randrange(20) for _ in range(20)]
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            pages, h = fa.fork_kv_pages(pages, h, i32(parents, dev))
            pairs = fa.resize_kv_pages(pages, h, h + 1)
        torch.cuda.current_stream().wait_stream(s)
        now = m.fork(held, parents)
        assert pairs.tolist() == m.resize(now, [x + 1 for x in now])
        same(pages, m)
    fa.check_status(dev)


def test_a_beam_search_over_shared_pages(cuda_device):
    """The calls of a loop: a prompt appended once, forked into beams, each step forked, given room, copied, appended, blocks chosen and attended to.
    What every beam holds is what it would hold alone, and lists and results are those of a cache of its own."""
    dev, rng = cuda_device, random.Random(3)
    H, G, D, size, block, width, pool, W = 2, 8, 64, 32, 16, 8, 60, 4
    g = torch.Generator().manual_seed(5)
    cache = fa.FP8KVCache.empty(pool, size, H, D, block, device=dev, indexed=True, by_head=True)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0x7F)
    pages = fa.KVPages.empty(1, width, pool, size, device=dev)
    held = i32([0], dev)
    k, v = ((torch.randn(1, 75, H, D, generator=g)).bfloat16().to(dev) for _ in range(2))
    fa.copy_kv_pages(cache, fa.resize_kv_pages(pages, held, held + 75))
    fa.append_kv_fp8(cache, k, v, held, page_table=pages.table)
    held = held + 75
    story = [[(k[0, i], v[0, i]) for i in range(75)]] * W
    pages, held = fa.fork_kv_pages(pages, held, i32([0] * W, dev))
    for step in range(40):
        q, k, v = ((torch.randn(W, 1, n, D, generator=g)).bfloat16().to(dev) for n in (G, H, H))
        fa.copy_kv_pages(cache, fa.resize_kv_pages(pages, held, held + 1))
        fa.append_kv_fp8(cache, k, v, held, page_table=pages.table)
        held = held + 1
        story = [s + [(k[b, 0], v[b, 0])] for b, s in enumerate(story)]
        lists = fa.select_kv_blocks(q, cache, held, 4, page_table=pages.table)
        out, lse = fa.flash_attn_fp8_blocks_func(q, cache, lists, held, page_table=pages.table, return_lse=True)
        if step % 13 == 12:
            n = len(story[0])
            own = fa.FP8KVCache.empty(W, 128, H, D, block, device=dev, indexed=True)
            own.k.view(torch.uint8).zero_()
            for i in range(n):
                t = [torch.stack([s[i][j] for s in story])[:, None] for j in (0, 1)]
                fa.append_kv_fp8(own, *t, i32([i] * W, dev)) if i >= 75 else None
                if i == 74:
                    whole = [torch.stack([torch.stack([s[x][j] for x in range(75)]) for s in story]) for j in (0, 1)]
                    fa.append_kv_fp8(own, *whole, i32([0] * W, dev))
            for b in range(W):
                at = pages.table[b].long()
                for name in ("k", "v"):
                    got = getattr(cache, name).view(torch.uint8)[at[:-(-n // size)]].flatten(0, 1)[:n]
                    assert torch.equal(got, getattr(own, name).view(torch.uint8)[b, :n])
            mine = fa.select_kv_blocks(q, own, held, 4)
            ref, ref_lse = fa.flash_attn_fp8_blocks_func(q, own, mine, held, return_lse=True)
            assert torch.equal(lists, mine) and torch.equal(out, ref) and torch.equal(lse, ref_lse)
        parents = [rng.randrange(W) for _ in range(W)]
        pages, held = fa.fork_kv_pages(pages, held, i32(parents, dev))
        story = [story[a] for a in parents]
    # some end; the others are moved to the front of the pool and hold what they held
    wanted = held * i32([0, 1, 1, 0], dev)
    fa.resize_kv_pages(pages, held, wanted)
    before = [cache.k.view(torch.uint8)[pages.table[b, :4].long()].flatten(0, 1)[:int(held[b])].clone() for b in (1, 2)]
    pairs, used = fa.compact_kv_pages(pages)
    fa.copy_kv_pages(cache, pairs)
    assert int(pages.table.max()) < used.item() <= 8
    for b, x in zip((1, 2), before):
        assert torch.equal(cache.k.view(torch.uint8)[pages.table[b, :4].long()].flatten(0, 1)[:int(held[b])], x)
    fa.resize_kv_pages(pages, wanted, torch.zeros_like(wanted))
    assert not pages.refs.any() and (pages.table == -1).all()
    fa.check_status(dev)
