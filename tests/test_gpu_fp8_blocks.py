"""Chosen blocks of the 8-bit KV cache on the GPU: the index and the choice against the oracle's whole numbers, the
attention against 64 bits.

Index and lists are compared for equality: bounds are whole numbers, their scale is one product by a power of two, a score one fp32
product of a whole number below 2^24.  The attention's tolerances are those of the attention over the whole cache
(tests/test_gpu_fp8_cache.py): the weights and sums are made by the same steps."""
import math

import pytest
import torch

import flash_attention_b200 as fa
from oracle import fp8_blocks_oracle as orc
from tests.test_gpu_fp8_cache import fill, held_of, make_cache, tables_of

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def indexed(cache, value=77):
    """The cache with an index of anything in it."""
    pages, size, H, D = cache.k.shape
    cache.key_bounds = torch.full((pages, size // cache.block, H, 2, D), value, dtype=torch.int8, device=cache.k.device)
    cache.bound_scale = torch.full((pages, size // cache.block, H), float(value), device=cache.k.device)
    return cache


def by_head(cache):
    """The same cache with the tokens of a head side by side."""
    k, v = (t.view(torch.uint8).transpose(1, 2).contiguous().view(torch.float8_e4m3fn).transpose(1, 2) for t in (cache.k, cache.v))
    return fa.FP8KVCache(k, v, cache.k_scale, cache.v_scale, cache.key_bounds, cache.bound_scale)


def index_of(cache, tables, ranges):
    """What the index should hold: the oracle's bounds of the blocks that tokens [a, b) of each sequence lie in, the rest as it is."""
    bt, size = cache.block, cache.k.shape[1]
    bounds, scale = cache.key_bounds.cpu().clone(), cache.bound_scale.cpu().clone()
    values = cache.k.cpu().contiguous().view(torch.float8_e4m3fn).double()
    for table, (a, b) in zip(tables, ranges):
        for first in range(a // bt * bt, b, bt):
            if b <= a:
                continue
            page, off = table[first // size], first % size
            m = min(bt, b - first)
            bounds[page, off // bt], scale[page, off // bt] = orc.index(values[page, off:off + m], cache.k_scale[page, off // bt].cpu())
    return bounds, scale


def same_index(cache, want):
    assert torch.equal(cache.key_bounds.cpu(), want[0])
    got = cache.bound_scale.cpu()
    assert ((got == want[1]) | (got.isnan() & want[1].isnan())).all()


# ---- the index ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("H,D,size,block,paged,heads_first", [
    (1, 128, 16, 16, True, False), (8, 128, 64, 64, True, True), (3, 64, 96, 32, True, False), (2, 64, 128, 128, True, True),
    (2, 128, 256, 128, False, False), (5, 128, 48, 16, False, True)])
@pytest.mark.parametrize("held,fresh", [([0, 0, 0], [500, 1, 0]), ([130, 16, 64], [1, 1, 1]), ([127, 128, 0], [2, 333, 17])])
def test_index_gives_the_oracles_bounds(cuda_device, H, D, size, block, paged, heads_first, held, fresh):
    most = max(h + n for h, n in zip(held, fresh))
    per = -(-most // size)
    if not paged:
        size, per = per * size, 1
    tables = tables_of(3, per, 3 * per + 2, 1) if paged else [[b] for b in range(3)]
    cache = indexed(make_cache(3 * per + 2, size, H, D, block, 1, cuda_device))
    fill(cache, tables, [h + n for h, n in zip(held, fresh)], 2, spread=8.0, outlier=True)
    if heads_first:
        cache = by_head(cache)
    want = index_of(cache, tables, [(h, h + n) for h, n in zip(held, fresh)])
    fa.index_kv_fp8(cache, i32(held, cuda_device), max(fresh), page_table=i32(tables, cuda_device) if paged else None,
                    seqused_new=i32(fresh, cuda_device))
    torch.cuda.synchronize()
    fa.check_status(cuda_device)
    same_index(cache, want)


def test_index_of_every_byte(cuda_device):
    """All 256 codes: blocks of zeros (of both signs), of the smallest values, of the largest, with NaN of both signs."""
    cache = indexed(make_cache(4, 16, 1, 64, 16, 1, cuda_device))
    codes = torch.arange(256, dtype=torch.uint8)
    k = torch.zeros(4, 16, 1, 64, dtype=torch.uint8)
    k[0, :, 0] = codes[:127].repeat(9)[:1024].view(16, 64)
    k[1, :, 0] = torch.cat([codes[128:255]] * 9)[:1024].view(16, 64)
    k[2, 3, 0, 5] = 0x80
    k[3] = k[0]
    k[3, 15, 0, 63] = 0xFF
    cache.k.view(torch.uint8).copy_(k)
    cache.k_scale.copy_(torch.tensor([1.0, 2.0 ** -120, 0.0, 3.0]).view(4, 1, 1))
    table = i32([[0, 1, 2, 3]], cuda_device)
    want = index_of(cache, [[0, 1, 2, 3]], [(0, 64)])
    fa.index_kv_fp8(cache, i32([0], cuda_device), 64, page_table=table)
    same_index(cache, want)
    assert want[1].isnan().sum() == 1 and cache.bound_scale[2, 0, 0] == 0
    # without its last token the last block has no NaN; the one that is not looked at may be anything
    fa.index_kv_fp8(cache, i32([60], cuda_device), 3, page_table=table)
    same_index(cache, index_of(cache, [[0, 1, 2, 3]], [(60, 63)]))
    assert not cache.bound_scale.isnan().any()
    for byte in (0x01, 0x81, 0x08, 0x7E, 0xFE):
        cache.k.view(torch.uint8)[0] = byte
        want = index_of(cache, [[0, 1, 2, 3]], [(0, 1)])
        fa.index_kv_fp8(cache, i32([0], cuda_device), 1, page_table=table)
        same_index(cache, want)


def test_append_keeps_the_index(cuda_device):
    """Pieces and single tokens, scales that grow: after each call the index is the one of what the cache holds."""
    B, H, D, size, block = 3, 2, 128, 64, 32
    tables = tables_of(B, 4, 14, 2)
    cache = indexed(make_cache(14, size, H, D, block, 1, cuda_device))
    table = i32(tables, cuda_device)
    g = torch.Generator().manual_seed(3)
    held = [0, 0, 0]
    for S, fresh in ((70, [70, 3, 0]), (1, [1, 1, 1]), (1, [1, 0, 1]), (40, [40, 33, 5]), (1, [1, 1, 1])):
        k = (torch.randn(B, S, H, D, generator=g) * 8.0 ** torch.randn(B, S, 1, 1, generator=g)).bfloat16().to(cuda_device)
        before = cache.key_bounds.cpu().clone(), cache.bound_scale.cpu().clone()
        fa.append_kv_fp8(cache, k, k, i32(held, cuda_device), page_table=table, seqused_new=i32(fresh, cuda_device))
        ranges = [(h, h + n) for h, n in zip(held, fresh)]
        held = [h + n for h, n in zip(held, fresh)]
        got = cache.key_bounds, cache.bound_scale
        cache.key_bounds, cache.bound_scale = before
        want = index_of(cache, tables, ranges)
        cache.key_bounds, cache.bound_scale = got
        same_index(cache, want)
    fa.check_status(cuda_device)
    # and it bounds every key
    k, _ = held_of(cache, tables[0], held[0])
    for t in range(held[0]):
        page, off = tables[0][t // size], t % size // block
        hi, lo = (cache.key_bounds[page, off, :, i].cpu().double() * cache.bound_scale[page, off].cpu().double()[:, None] for i in (0, 1))
        assert (k[t] <= hi).all() and (k[t] >= lo).all()


def test_index_leaves_out_what_has_no_place(cuda_device):
    cache = indexed(make_cache(4, 32, 1, 64, 32, 1, cuda_device, nan=False))
    table = i32([[0, 1], [2, 7], [3, -1]], cuda_device)
    for held, site in (([64, 0, 0], 120), ([0, 33, 0], 121), ([0, 0, 40], 121), ([-5, 0, 0], 120), ([2 ** 31 - 1, 0, 0], 120), ([60, 0, 0], 120)):
        cache.bound_scale.fill_(-1.0)
        fa.index_kv_fp8(cache, i32(held, cuda_device), 5, page_table=table)
        with pytest.raises(RuntimeError, match=f"code 2 .*site {site},"):
            fa.check_status(cuda_device)
        assert cache.bound_scale[0, 0, 0] == -1 or held[0] == 0
        # (of tokens 60 .. 64 all but the last are there)
        assert (cache.bound_scale[1, 0, 0] != -1) == (held[0] == 60)
    fa.index_kv_fp8(cache, i32([0, 0, 0], cuda_device), 0, page_table=table)
    fa.index_kv_fp8(cache, i32([0, 0, 0], cuda_device), 32, page_table=table)
    fa.check_status(cuda_device)


# ---- the choice -----------------------------------------------------------------------------------------------

def setting(device, B, Sq, Hq, H, D, size, block, lens, fresh=None, paged=True, seed=1, spread=1.0, q_scale=1.0, heads_first=False, poke=None):
    """A filled and indexed cache, its tables, queries."""
    per = max(1, max(-(-n // size) for n in lens))
    if not paged:
        size, per = per * size, 1
    pages = B * per + 2
    tables = tables_of(B, per, pages, seed) if paged else [[b] for b in range(B)]
    cache = indexed(make_cache(pages, size, H, D, block, seed, device), value=0)
    fill(cache, tables, lens, seed, spread)
    if poke is not None:
        poke(cache, tables)
    cache.key_bounds, cache.bound_scale = (t.to(device) for t in index_of(cache, tables, [(0, n) for n in lens]))
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(B, Sq, Hq, D, generator=g) * q_scale).bfloat16()
    if heads_first:
        cache = by_head(cache)
    return cache, tables, q


def wide_table(tables, lens, size, device, paged=True):
    """Entries of the table behind the last page are anybody's."""
    if not paged:
        return None
    wide = [t + [10 ** 9, -7] for t in tables]
    for t, n in zip(wide, lens):
        for i in range(-(-n // size), len(t)):
            t[i] = 10 ** 9
    return i32(wide, device)


def lists_of(cache, tables, q, lens, fresh, chosen, rows, front, recent):
    """The oracle's lists, (B, query blocks, H, chosen)."""
    B, Sq, G, D = q.shape
    H, bt, size = cache.k.shape[2], cache.block, cache.k.shape[1]
    bounds, scale = cache.key_bounds.cpu(), cache.bound_scale.cpu()
    got = []
    for b in range(B):
        flat = torch.cat([bounds[p] for p in tables[b]]), torch.cat([scale[p] for p in tables[b]])
        n = Sq if fresh is None else fresh[b]
        for r0 in range(0, Sq, rows):
            r1 = min(n, r0 + rows)
            for h in range(H):
                if r1 <= r0:
                    got.append([-1] * chosen)
                    continue
                heads = slice(h * (G // H), (h + 1) * (G // H))
                got.append(orc.select(q[b, r0:r1, heads], flat[0][:, h], flat[1][:, h], lens[b] - n + r0, lens[b] - n + r1, bt, chosen, front, recent))
    return torch.tensor(got, dtype=torch.int32).view(B, -(-Sq // rows), H, chosen)


def choose(device, chosen, rows=1, front=1, recent=1, fresh=None, paged=True, poke_q=None, **kw):
    cache, tables, q = setting(device, fresh=fresh, paged=paged, **kw)
    if poke_q is not None:
        poke_q(q)
    lens, size = kw["lens"], cache.k.shape[1]
    table = wide_table(tables, lens, size, device, paged)
    got = fa.select_kv_blocks(q.to(device), cache, i32(lens, device), chosen, page_table=table,
                              seqused_q=None if fresh is None else i32(fresh, device), query_block=rows, front_blocks=front, recent_blocks=recent)
    torch.cuda.synchronize()
    fa.check_status(device)
    want = lists_of(cache, tables, q, lens, fresh, chosen, rows, front, recent)
    assert torch.equal(got.cpu(), want), f"{(got.cpu() != want).any(-1).sum()} of {want[..., 0].numel()} lists differ"
    return cache, tables, q, table, got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 16])
@pytest.mark.parametrize("lens,chosen", [([1], 2), ([0, 5, 300], 4), ([777, 128, 127, 129], 3), ([4100, 2049, 300, 129], 17)])
def test_choice_of_one_token(cuda_device, D, group, lens, chosen):
    choose(cuda_device, chosen, B=len(lens), Sq=1, Hq=2 * group, H=2, D=D, size=64, block=32, lens=lens)


@pytest.mark.parametrize("size,block,paged,heads_first", [(16, 16, True, False), (48, 16, True, True), (128, 64, True, False), (256, 128, True, True),
                                                          (64, 64, False, False)])
@pytest.mark.parametrize("Sq,rows", [(1, 1), (5, 1), (7, 3), (100, 64), (65, 1000)])
def test_choice_of_several_rows(cuda_device, size, block, paged, heads_first, Sq, rows):
    chosen = 3 + (min(rows, Sq) + block - 2) // block
    choose(cuda_device, chosen, rows=rows, B=3, Sq=Sq, Hq=6, H=2, D=128, size=size, block=block, lens=[1500, Sq + 3, 640], paged=paged,
           fresh=[Sq, max(1, Sq - 2), Sq // 2], heads_first=heads_first)


@pytest.mark.parametrize("front,recent,chosen", [(0, 1, 1), (0, 1, 5), (3, 4, 7), (2, 1, 8), (40, 30, 70)])
def test_blocks_that_are_always_chosen(cuda_device, front, recent, chosen):
    choose(cuda_device, chosen, front=front, recent=recent, B=3, Sq=2, Hq=4, H=2, D=64, size=32, block=16, lens=[1300, 33, 700], fresh=[2, 2, 1])


def test_rows_in_front_of_all_tokens(cuda_device):
    """More rows than tokens: the first ones stand at negative positions and see nothing."""
    choose(cuda_device, 4, B=3, Sq=6, Hq=4, H=2, D=64, size=32, block=16, lens=[3, 100, 0])
    choose(cuda_device, 9, rows=64, B=2, Sq=70, Hq=4, H=2, D=64, size=32, block=16, lens=[3, 500])


def test_equal_scores_go_to_the_lower_number(cuda_device):
    """Blocks that repeat, queries of zeros, scales of zero: most scores tie."""
    def repeat(cache, tables):
        k = cache.k.view(torch.uint8)
        for t in tables:
            for page in t[1:]:
                k[page] = k[t[0]]
                cache.k_scale[page] = cache.k_scale[t[0]]
    kw = dict(B=2, Sq=1, Hq=4, H=2, D=64, size=64, block=16, lens=[1280, 640])
    choose(cuda_device, 9, poke=repeat, **kw)
    choose(cuda_device, 9, poke_q=lambda q: q.zero_(), **kw)
    choose(cuda_device, 9, poke=lambda cache, tables: cache.k_scale.zero_(), **kw)


def test_scores_that_are_not_finite(cuda_device):
    """A block with a NaN comes first, scales as large as fp32 has them give infinite scores; queries that are not finite count as 0."""
    def poison(cache, tables):
        k = cache.k.view(torch.uint8)
        k[tables[0][3], 20, 1, 7] = 0x7F
        k[tables[0][9], 1, 0, 63] = 0xFF
        cache.k_scale[tables[0][5]] = 3e38
        cache.k_scale[tables[0][6]] = math.inf

    def poke_q(q):
        q[0, 0, 1, 3] = math.nan
        q[0, 0, 2, 4] = math.inf
        q[0, 0, 3, 5] = -math.inf
    kw = dict(B=1, Sq=1, Hq=4, H=2, D=64, size=32, block=32, lens=[1000])
    for chosen in (3, 4, 6, 12):
        choose(cuda_device, chosen, poke=poison, **kw)
        choose(cuda_device, chosen, poke=poison, poke_q=poke_q, **kw)
    choose(cuda_device, 5, poke_q=lambda q: q.fill_(math.nan), **kw)


@pytest.mark.parametrize("q_scale", [1e-38, 1e-30, 1e30])
def test_choice_by_small_and_large_queries(cuda_device, q_scale):
    choose(cuda_device, 7, B=2, Sq=3, Hq=8, H=2, D=128, size=64, block=32, lens=[1500, 900], q_scale=q_scale, spread=8.0)


def test_choice_among_many_blocks(cuda_device):
    """Tens of thousands of blocks, a list of thousands."""
    dev = cuda_device
    B, H, D, size, block, per = 2, 1, 64, 256, 16, 2500
    pages = B * per
    g = torch.Generator(device=dev).manual_seed(4)
    small = torch.zeros(pages, size, H, D, dtype=torch.uint8, device=dev)
    scale = torch.ones(pages, size // block, H, device=dev)
    cache = fa.FP8KVCache(small, small, scale, scale, torch.randint(-120, 121, (pages, size // block, H, 2, D), generator=g, device=dev).to(torch.int8),
                          torch.rand(pages, size // block, H, generator=g, device=dev) + 0.5)
    tables = torch.randperm(pages, generator=g, device=dev).view(B, per).to(torch.int32)
    q = torch.randn(B, 1, 4, D, generator=g, device=dev).bfloat16()
    lens = [per * size, per * size - 777]
    for chosen in (2, 100, 5000):
        got = fa.select_kv_blocks(q, cache, i32(lens, dev), chosen, page_table=tables)
        want = lists_of(cache, tables.tolist(), q.cpu(), lens, None, chosen, 1, 1, 1)
        assert torch.equal(got.cpu(), want)
    fa.check_status(dev)


# ---- attention over chosen blocks -------------------------------------------------------------------------------

def attend_both(device, lists, q, cache, tables, lens, fresh=None, rows=1, table=None, sink=None, **kw):
    B, Sq, G, D = q.shape
    H, bt = cache.k.shape[2], cache.block
    out = torch.full((B, Sq, G, D), 7.0, dtype=torch.bfloat16, device=device)
    lse = torch.full((B, G, Sq), 7.0, device=device)
    got, got_lse = fa.flash_attn_fp8_blocks_func(
        q.to(device), cache, lists.to(device), i32(lens, device), page_table=table, seqused_q=None if fresh is None else i32(fresh, device),
        query_block=rows, learnable_sink=None if sink is None else sink.to(device), return_lse=True, out=out, lse=lse, **kw)
    torch.cuda.synchronize()
    fa.check_status(device)
    assert got is out and got_lse is lse
    lists = lists.cpu().tolist()
    for b in range(B):
        n = Sq if fresh is None else fresh[b]
        k, v = held_of(cache, tables[b], lens[b])
        top = 1.0
        if lens[b] and n:
            top = float(q[b, :n].double().norm(dim=-1).max() * k[~k.isnan().any(-1)].norm(dim=-1).max()) * kw.get("softmax_scale", D ** -0.5)
        for s in range(n):
            place = lens[b] - n + s
            for h in range(H):
                g = slice(h * (G // H), (h + 1) * (G // H))
                keys = [t for t in orc.keys_of(lists[b][s // rows][h], bt) if t < lens[b]]
                args = dict(softmax_scale=kw.get("softmax_scale"), sink=None if sink is None else sink[g], softcap=kw.get("softcap", 0.0))
                want, want_lse = orc.attend(q[b, s, g], k[:, h], v[:, h], keys, place, **args)
                mag, _ = orc.attend(q[b, s, g], k[:, h], v[:, h].abs(), keys, place, **args)
                o, l = out[b, s, g].cpu().double(), lse[b, g, s].cpu().double()
                off = (o - want).abs()
                room = 2.0 ** -8 * (mag + want.abs()) + (2.0 ** -13 + math.expm1(2.0 * min(5.0, 2.0 ** -20 * top))) * mag + 1e-30
                assert (off <= room).all(), f"sequence {b}, row {s}, head {h}: {(off / room).max():.2f} of the room"
                sees = want_lse > -math.inf
                assert torch.equal(sees, l > -math.inf)
                room = 2.0 ** -18 * want_lse[sees].abs().clamp(min=1.0) + 2.0 ** -20 * top
                assert ((l[sees] - want_lse[sees]).abs() <= room).all()
        assert (out[b, n:] == 7.0).all() and (lse[b, :, n:] == 7.0).all()
    return out, lse


def chosen_and_attended(device, chosen, rows=1, sink=False, attn=None, **kw):
    cache, tables, q, table, lists = choose(device, chosen, rows=rows, **kw)
    s = torch.randn(q.shape[2], generator=torch.Generator().manual_seed(9)) * 2 if sink else None
    return attend_both(device, lists, q, cache, tables, kw["lens"], kw.get("fresh"), rows, table, s, **(attn or {}))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("lens,chosen", [([1], 2), ([0, 5], 3), ([777, 128, 127], 5), ([16, 2049, 300, 129], 19)])
def test_one_token(cuda_device, D, group, lens, chosen):
    chosen_and_attended(cuda_device, chosen, B=len(lens), Sq=1, Hq=2 * group, H=2, D=D, size=64, block=32, lens=lens)


@pytest.mark.parametrize("size,block,paged,heads_first", [(16, 16, True, True), (48, 16, True, False), (96, 32, True, True), (192, 64, True, False),
                                                          (256, 128, True, True), (16, 16, False, False), (128, 128, False, True)])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_and_blocks(cuda_device, size, block, paged, heads_first, D):
    kw = dict(B=3, Hq=8, H=2, D=D, size=size, block=block, lens=[700, 1030, 17], paged=paged, heads_first=heads_first, spread=8.0)
    chosen_and_attended(cuda_device, 5, Sq=1, **kw)
    chosen_and_attended(cuda_device, 6, Sq=17, rows=17, **{**kw, "lens": [700, 1030, 17]})


@pytest.mark.parametrize("Sq,group,rows", [(2, 4, 1), (5, 4, 1), (9, 2, 1), (8, 4, 4), (16, 2, 16), (33, 1, 32), (50, 4, 16), (70, 4, 64), (40, 8, 33), (130, 2, 100),
                                           (40, 16, 1), (20, 1, 7)])
def test_several_rows(cuda_device, Sq, group, rows):
    for D in (64, 128):
        chosen_and_attended(cuda_device, 4 + (rows + 14) // 16, rows=rows, B=2, Sq=Sq, Hq=2 * group, H=2, D=D, size=64, block=16, lens=[Sq + 700, Sq])


@pytest.mark.parametrize("Sq,rows", [(1, 1), (6, 1), (70, 64)])
@pytest.mark.parametrize("D", [64, 128])
def test_sink_and_softcap(cuda_device, Sq, rows, D):
    kw = dict(B=3, Sq=Sq, rows=rows, Hq=8, H=2, D=D, size=64, block=32, lens=[Sq + 600, Sq + 5, 0])
    chosen_and_attended(cuda_device, 6, sink=True, fresh=[Sq, Sq, Sq], **kw)
    chosen_and_attended(cuda_device, 6, attn=dict(softcap=20.0), q_scale=4.0, **kw)
    chosen_and_attended(cuda_device, 6, sink=True, attn=dict(softcap=5.0, softmax_scale=0.3), **kw)


@pytest.mark.parametrize("Sq,rows", [(1, 1), (6, 1), (6, 4), (70, 64)])
def test_padded_batches_and_rows_that_see_nothing(cuda_device, Sq, rows):
    for D in (64, 128):
        kw = dict(Sq=Sq, rows=rows, Hq=8, H=2, D=D, size=64, block=64)
        chosen_and_attended(cuda_device, 4, B=4, lens=[600, 40, max(1, Sq // 2), 0], fresh=[Sq, max(1, Sq - 3), Sq, Sq], **kw)
        chosen_and_attended(cuda_device, 4, B=3, lens=[600, 40, 7], fresh=[0, Sq, 1], **kw)


@pytest.mark.parametrize("B,Sq,rows,Hq,H,chosen", [(3, 1, 1, 4, 1, 60), (2, 4, 1, 8, 8, 40), (25, 1, 1, 8, 4, 20), (40, 1, 1, 4, 4, 80), (40, 6, 6, 16, 4, 80),
                                                   (40, 1, 1, 4, 4, 12), (80, 1, 1, 16, 8, 3), (1, 150, 1, 8, 4, 4)])
def test_calls_of_few_and_many_units(cuda_device, B, Sq, rows, Hq, H, chosen):
    """Few units, split among the CTAs of a cluster; a CTA a unit; shares dealt by the lengths and merged; whole units one after the other."""
    lens = [(331 * b) % (1500 if B < 60 else 300) + Sq for b in range(B)]
    chosen_and_attended(cuda_device, chosen, B=B, Sq=Sq, rows=rows, Hq=Hq, H=H, D=64, size=32, block=16, lens=lens)


@pytest.mark.parametrize("Sq,rows", [(1, 1), (3, 1), (70, 64)])
@pytest.mark.parametrize("D", [64, 128])
def test_lists_of_ones_own(cuda_device, Sq, rows, D):
    """Empty lists, lists that end early, entries behind the row, entries that do not ascend or lie outside the cache."""
    lens = [600, 90 + Sq, 300]
    cache, tables, q = setting(cuda_device, B=3, Sq=Sq, Hq=4, H=2, D=D, size=64, block=32, lens=lens)
    lists = torch.full((3, -(-Sq // rows), 2, 40), -1, dtype=torch.int32)
    lists[0, :, 0, :2] = i32([1, 4], "cpu")
    lists[0, :, 1, :40] = torch.arange(40)
    lists[1, :, 0, :6] = i32([0, 2, 1, 3, 5, 7], "cpu")
    lists[1, :, 1, :4] = i32([2, 2, 3, 4], "cpu")
    lists[2, :, 0, :4] = i32([3, 9, 2 ** 31 - 1, 4], "cpu")
    lists[2, :, 1, :3] = i32([-5, 0, 1], "cpu")
    table = wide_table(tables, lens, 64, cuda_device)
    attend_both(cuda_device, lists, q, cache, tables, lens, None, rows, table)
    sink = torch.randn(4, generator=torch.Generator().manual_seed(1))
    attend_both(cuda_device, lists, q, cache, tables, lens, None, rows, table, sink)


@pytest.mark.parametrize("Sq,rows", [(1, 1), (4, 2), (70, 64)])
def test_a_list_of_all_blocks_is_attention_over_the_whole(cuda_device, Sq, rows):
    lens = [900, 333]
    cache, tables, q = setting(cuda_device, B=2, Sq=Sq, Hq=8, H=2, D=128, size=64, block=64, lens=lens, spread=4.0)
    table = i32(tables, cuda_device)
    lists = fa.select_kv_blocks(q.to(cuda_device), cache, i32(lens, cuda_device), 20, page_table=table, query_block=rows)
    out, lse = fa.flash_attn_fp8_blocks_func(q.to(cuda_device), cache, lists, i32(lens, cuda_device), page_table=table, query_block=rows, return_lse=True)
    ref, ref_lse = fa.flash_attn_fp8_cache_func(q.to(cuda_device), cache, i32(lens, cuda_device), page_table=table, causal=True, return_lse=True)
    # (each is off by at most 2^-8 of the sums of magnitudes twice over: see the top of the file)
    mag, _ = fa.flash_attn_fp8_cache_func(q.to(cuda_device), fa.FP8KVCache(cache.k, (cache.v.view(torch.uint8) & 0x7F), cache.k_scale, cache.v_scale),
                                          i32(lens, cuda_device), page_table=table, causal=True)
    assert ((out.double() - ref.double()).abs() <= 2 * 2.0 ** -8 * (mag.double() * 1.01 + ref.double().abs()) + 1e-30).all()
    assert ((lse - ref_lse).abs() <= 2.0 ** -17 * ref_lse.abs().clamp(min=1.0) + 2.0 ** -18).all()
    fa.check_status(cuda_device)


@pytest.mark.parametrize("Sq,rows", [(1, 1), (70, 64)])
def test_blocks_that_are_not_chosen_may_hold_anything(cuda_device, Sq, rows):
    lens = [1000]
    cache, tables, q = setting(cuda_device, B=1, Sq=Sq, Hq=8, H=1, D=64, size=32, block=32, lens=lens)
    table = i32(tables, cuda_device)
    lists = fa.select_kv_blocks(q.to(cuda_device), cache, i32(lens, cuda_device), 6, page_table=table, query_block=rows)
    want = fa.flash_attn_fp8_blocks_func(q.to(cuda_device), cache, lists, i32(lens, cuda_device), page_table=table, query_block=rows)[0].clone()
    chosen = set(lists.flatten().tolist())
    for j in range(-(-lens[0] // 32)):
        if j not in chosen:
            cache.k.view(torch.uint8)[tables[0][j]] = 0x7F
            cache.v.view(torch.uint8)[tables[0][j]] = 0xFF
            cache.k_scale[tables[0][j]] = math.nan
            cache.v_scale[tables[0][j]] = math.nan
    got = fa.flash_attn_fp8_blocks_func(q.to(cuda_device), cache, lists, i32(lens, cuda_device), page_table=table, query_block=rows)[0]
    assert torch.equal(got, want)
    fa.check_status(cuda_device)


def test_bad_pages_are_reported(cuda_device):
    lens = [300]
    cache, tables, q = setting(cuda_device, B=1, Sq=1, Hq=4, H=2, D=64, size=64, block=32, lens=lens)
    table = i32(tables, cuda_device)
    table[0, 2] = 10 ** 9
    lists = fa.select_kv_blocks(q.to(cuda_device), cache, i32(lens, cuda_device), 3, page_table=table)
    with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
        fa.check_status(cuda_device)
    assert not ((lists == 4) | (lists == 5)).any()
    lists[..., 1] = 4
    fa.flash_attn_fp8_blocks_func(q.to(cuda_device), cache, lists, i32(lens, cuda_device), page_table=table)
    with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
        fa.check_status(cuda_device)
    lists[..., 1] = 3
    fa.flash_attn_fp8_blocks_func(q.to(cuda_device), cache, lists, i32(lens, cuda_device), page_table=table)
    fa.check_status(cuda_device)


# ---- calls as a program makes them --------------------------------------------------------------------------------

def step_of(cache, table, q, k, held, chosen, **kw):
    """One step of a serving loop: append, choose, attend."""
    fa.append_kv_fp8(cache, k, k, held, page_table=table)
    held.add_(k.shape[1])
    lists = fa.select_kv_blocks(q, cache, held, chosen, page_table=table)
    return lists, fa.flash_attn_fp8_blocks_func(q, cache, lists, held, page_table=table, return_lse=True, **kw)


def test_steps_of_a_serving_loop_in_a_graph(cuda_device):
    """Captured once, replayed over growing lengths: lists and results are those of the calls made one by one."""
    dev, room = cuda_device, [200, 61, 1000]           # (tokens that there are pages for)

    def start():
        cache, tables, _ = setting(dev, B=3, Sq=1, Hq=8, H=2, D=128, size=32, block=16, lens=room, seed=5)
        return cache, i32(tables, dev)
    g = torch.Generator().manual_seed(6)
    steps = [[(torch.randn(3, 1, n, 128, generator=g)).bfloat16().to(dev) for n in (8, 2)] for _ in range(5)]
    lens = [n - 10 for n in room]
    cache, table = start()
    held = i32(lens, dev)
    want = []
    for q, k in steps:
        lists, (out, lse) = step_of(cache, table, q, k, held, 6)
        want.append((lists.clone(), out.clone(), lse.clone()))
    cache, table = start()
    held = i32(lens, dev)
    q, k = (t.clone() for t in steps[0])
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale, cache.key_bounds, cache.bound_scale)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step_of(cache, table, q, k, held, 6)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lists, (out, lse) = step_of(cache, table, q, k, held, 6)
    for t, x in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_scale, cache.v_scale, cache.key_bounds, cache.bound_scale), before):
        t.copy_(x)
    held.copy_(i32(lens, dev))
    for (q1, k1), (l1, o1, e1) in zip(steps, want):
        q.copy_(q1)
        k.copy_(k1)
        graph.replay()
        assert torch.equal(lists, l1) and torch.equal(out, o1) and torch.equal(lse, e1)
    fa.check_status(dev)


def test_two_streams_at_once_and_the_same_bits_each_time(cuda_device):
    dev, lens = cuda_device, [3000, 1200]
    made = [setting(dev, B=2, Sq=n, Hq=8, H=2, D=128, size=64, block=32, lens=lens, seed=n) for n in (1, 70)]
    def call(i):
        cache, tables, q = made[i]
        q, rows, table = q.to(dev), (1, 64)[i], i32(tables, dev)
        lists = fa.select_kv_blocks(q, cache, i32(lens, dev), 20, page_table=table, query_block=rows)
        return lists, fa.flash_attn_fp8_blocks_func(q, cache, lists, i32(lens, dev), page_table=table, query_block=rows)[0]
    want = [[t.clone() for t in call(i)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        for lists, out in got[i]:
            assert torch.equal(lists, want[i][0]) and torch.equal(out, want[i][1])
    fa.check_status(dev)


def test_strided_queries_and_outputs(cuda_device):
    dev, lens = cuda_device, [700, 90]
    cache, tables, q = setting(dev, B=2, Sq=3, Hq=4, H=2, D=64, size=32, block=32, lens=lens)
    table, used = i32(tables, dev), i32(lens, dev)
    want_l = fa.select_kv_blocks(q.to(dev), cache, used, 5, page_table=table)
    want = fa.flash_attn_fp8_blocks_func(q.to(dev), cache, want_l, used, page_table=table)[0]
    wide = torch.zeros(2, 3, 12, 64, dtype=torch.bfloat16, device=dev)
    wide[:, :, 4:8] = q.to(dev)
    odd = torch.zeros(2 * 3 * 4 * 65 + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, 3, 4, 65)[..., 1:]
    odd.copy_(q)
    out = torch.zeros(2, 3, 8, 64, dtype=torch.bfloat16, device=dev)
    into = torch.full((2, 3, 2, 5), 9, dtype=torch.int32, device=dev)
    for view in (wide[:, :, 4:8], odd):
        lists = fa.select_kv_blocks(view, cache, used, 5, page_table=table, out=into)
        assert lists is into and torch.equal(lists, want_l)
        # lists may be a view as well
        spread = torch.full((2, 3, 2, 10), 3, dtype=torch.int32, device=dev)[..., ::2]
        spread.copy_(lists)
        out.zero_()
        got = fa.flash_attn_fp8_blocks_func(view, cache, spread, used, page_table=table, out=out[:, :, 2:6])[0]
        assert torch.equal(got, want) and (out[:, :, :2] == 0).all() and (out[:, :, 6:] == 0).all()
    fa.check_status(dev)


def test_offsets_that_pass_32_bits(cuda_device):
    """A pool of more than 2^32 bytes, the pages in use at its end."""
    dev = cuda_device
    pages, size, H, D = 70000, 64, 8, 128
    if torch.cuda.mem_get_info(dev)[0] < 16 * 2 ** 30:
        pytest.skip("not enough memory")
    raw = torch.zeros(pages, size, H, D, dtype=torch.uint8, device=dev)
    scale = torch.ones(pages, 1, H, device=dev)
    cache = fa.FP8KVCache(raw, raw, scale, scale, torch.zeros(pages, 1, H, 2, D, dtype=torch.int8, device=dev), torch.zeros(pages, 1, H, device=dev))
    small = fa.FP8KVCache(*(t[-20:].clone() for t in (raw, raw, scale, scale, cache.key_bounds, cache.bound_scale)))
    g = torch.Generator(device=dev).manual_seed(2)
    bytes_ = torch.randint(0, 0x70, (20, size, H, D), generator=g, device=dev, dtype=torch.uint8) | (torch.randint(0, 2, (20, size, H, D), generator=g, device=dev, dtype=torch.uint8) << 7)
    raw[-20:] = bytes_
    small.k.copy_(bytes_)
    small.v = small.k
    q = torch.randn(1, 1, 32, D, generator=g, device=dev).bfloat16()
    got = []
    for c, table in ((cache, torch.arange(pages - 20, pages)), (small, torch.arange(20))):
        table = table.to(dev, torch.int32)[None]
        fa.index_kv_fp8(c, i32([0], dev), 20 * size, page_table=table)
        lists = fa.select_kv_blocks(q, c, i32([20 * size - 3], dev), 7, page_table=table)
        got.append((c.key_bounds[-20:], lists, fa.flash_attn_fp8_blocks_func(q, c, lists, i32([20 * size - 3], dev), page_table=table)[0]))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    fa.check_status(dev)


def test_refusals_on_the_gpu(cuda_device):
    dev, lens = cuda_device, [300, 90]
    cache, tables, q = setting(dev, B=2, Sq=3, Hq=4, H=2, D=64, size=32, block=32, lens=lens)
    table, used, q = i32(tables, dev), i32(lens, dev), q.to(dev)
    bare = fa.FP8KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale)
    lists = fa.select_kv_blocks(q, cache, used, 5, page_table=table)
    with pytest.raises(AssertionError, match="no index"):
        fa.select_kv_blocks(q, bare, used, 5, page_table=table)
    with pytest.raises(AssertionError, match="no index"):
        fa.index_kv_fp8(bare, used, 3, page_table=table)
    half = fa.FP8KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.key_bounds)
    with pytest.raises(AssertionError, match="no index"):
        fa.append_kv_fp8(half, q[:, :, :2], q[:, :, :2], used, page_table=table)
    for name, bad in (("key_bounds", cache.key_bounds.view(torch.uint8)), ("key_bounds", cache.key_bounds[..., :1, :]), ("key_bounds", cache.key_bounds[:-1]),
                      ("bound_scale", cache.bound_scale.double()), ("bound_scale", cache.bound_scale.cpu())):
        c = fa.FP8KVCache(cache.k, cache.v, cache.k_scale, cache.v_scale, cache.key_bounds, cache.bound_scale)
        setattr(c, name, bad)
        for call in (lambda: fa.select_kv_blocks(q, c, used, 5, page_table=table), lambda: fa.index_kv_fp8(c, used, 1, page_table=table)):
            with pytest.raises(AssertionError, match=name):
                call()
    for kw, match in ((dict(num_blocks=0), "must be positive"), (dict(query_block=0), "must be positive"), (dict(recent_blocks=0), "must be positive"),
                      (dict(front_blocks=-1), "not negative"), (dict(front_blocks=5), "no room"), (dict(num_blocks=2, query_block=3), "no room"),
                      (dict(num_blocks=1), "no room")):
        with pytest.raises(ValueError, match=match):
            fa.select_kv_blocks(q, cache, used, page_table=table, **{"num_blocks": 5, **kw})
    with pytest.raises(AssertionError, match="out shape"):
        fa.select_kv_blocks(q, cache, used, 5, page_table=table, out=lists[..., :4])
    with pytest.raises(AssertionError, match="q dtype"):
        fa.select_kv_blocks(q.half(), cache, used, 5, page_table=table)
    for bad in (lists[:1], lists[:, :2], lists[:, :, :1], lists.long(), lists.cpu(), lists[..., 0], lists[..., :0]):
        with pytest.raises(AssertionError, match="blocks"):
            fa.flash_attn_fp8_blocks_func(q, cache, bad, used, page_table=table)
    with pytest.raises(AssertionError, match="blocks"):
        fa.flash_attn_fp8_blocks_func(q, cache, lists, used, page_table=table, query_block=2)
    with pytest.raises(ValueError, match="query_block"):
        fa.flash_attn_fp8_blocks_func(q, cache, lists, used, page_table=table, query_block=0)
    with pytest.raises(TypeError, match="blocks"):
        fa.flash_attn_fp8_blocks_func(q, cache, None, used, page_table=table)
    with pytest.raises(NotImplementedError, match="53248"):
        fa.select_kv_blocks(q, cache, used, 5, page_table=torch.zeros(2, 60000, dtype=torch.int32, device=dev))
    # empty calls
    assert fa.select_kv_blocks(q[:0], cache, used[:0], 5, page_table=table[:0]).shape == (0, 3, 2, 5)
    assert fa.select_kv_blocks(q[:, :0], cache, used, 5, page_table=table).shape == (2, 0, 2, 5)
    assert fa.flash_attn_fp8_blocks_func(q[:, :0], cache, lists[:, :0], used, page_table=table)[0].shape == (2, 0, 4, 64)
    fa.check_status(dev)
