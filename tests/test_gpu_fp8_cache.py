"""The 8-bit KV cache on the GPU: appending against the oracle, attention over it against 64 bits.

Tolerances.  Appended bytes and scales are the oracle's: rotation, scale and quotient are the same correctly rounded fp32 steps
(the rounding to e4m3 is exact in 64 bits), so they are compared for equality; q is rounded to bf16 once from those.
Attention: one output element is sum p v / sum p.  The weights are rounded to no fewer than 8 significant bits (2^-8 of
each at most, half a step of bf16), scores are fp32 sums of exact products, so |error| <= 2^-8 sum p |v| / sum p, plus the output's
own rounding of 2^-8 |out|, plus fp32 noise, for which 2^-13 sum p |v| is room.  A score itself is an fp32 sum of D <= 128
products of at most |q| |k| scale = T together: 2^-24 of T for each addition, sqrt(128) < 16 of them where signs differ, so it
is off by delta = 2^-20 T, a weight by the factor e^delta, and the quotient of two sums of weights by e^2delta: another
(e^2delta - 1) sum p |v| / sum p.  (T is 10 in an ordinary case and this is nothing; with T in the thousands it is as much as the
rest, with T in the millions, as in the test of far scores, fp32 scores tell only the largest ones apart.)  lse: fp32 sums and hardware
exponentials, 2^-18 of max(1, |lse|), and the same delta.  Weights keep their bits down to 2^-14 (many rows: 2^-20) of
the largest: no case here has an element that is made by smaller ones alone."""
import math

import pytest
import torch

import flash_attention_b200 as fa
from oracle import fp8_cache_oracle as orc

pytestmark = pytest.mark.gpu


def make_cache(pages, size, H, D, block, seed, device, nan=True):
    """A pool of random bytes (NaN where nothing is held yet: everything here, to begin with) and odd scales."""
    g = torch.Generator().manual_seed(seed)
    c = fa.FP8KVCache.empty(pages, size, H, D, block, device=device)
    for t in (c.k, c.v):
        t.view(torch.uint8).copy_(torch.full(t.shape, 0x7F, dtype=torch.uint8) if nan else
                                  torch.randint(0, 0x78, t.shape, generator=g, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.full(t.shape, math.nan) if nan else torch.rand(t.shape, generator=g))
    return c


def fill(cache, tables, lens, seed, spread=1.0, outlier=False):
    """Random keys and values for the first lens[b] tokens of every sequence: e4m3 values of a maximum / 448 scale."""
    g = torch.Generator().manual_seed(seed)
    pages, size, H, D = cache.k.shape
    bt = cache.block
    for t, sc, strong in ((cache.k, cache.k_scale, outlier), (cache.v, cache.v_scale, False)):
        values, scales = t.cpu().view(torch.uint8).clone(), sc.cpu().clone()
        for b, n in enumerate(lens):
            for first in range(0, n, bt):
                m = min(bt, n - first)
                x = torch.randn(m, H, D, generator=g) * (spread ** torch.randn(1, H, 1, generator=g))
                if strong:
                    x[..., ::16] *= 8
                s = x.abs().amax(dim=(0, 2)) / 448
                page, off = tables[b][first // size], first % size
                values[page, off:off + m] = (x / s[None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                scales[page, off // bt] = s
        t.view(torch.uint8).copy_(values)
        sc.copy_(scales)


def held_of(cache, table, n):
    """float64 keys and values (n, H, D) of a sequence."""
    got = []
    for t, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = t.cpu().view(torch.float8_e4m3fn).double() * sc.cpu().double().repeat_interleave(cache.block, dim=1)[..., None]
        got.append(torch.cat([x[p] for p in table])[:n])
    return got


def tables_of(B, per, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * per].view(B, per).tolist()


def rope(rows, dim, dtype=torch.float32, seed=0):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / max(1, dim // 2))
    return ang.cos().to(dtype), ang.sin().to(dtype)


# ---- append ---------------------------------------------------------------------------------------------------

APPENDS = [
    # B, S, H, D, page, block, paged, held, fresh, rotary, interleaved, Hq, table dtype
    (1, 1, 1, 128, 16, 16, True, [0], None, 128, False, 4, torch.float32),
    (3, 1, 8, 128, 64, 64, True, [0, 63, 64], None, 128, False, 32, torch.bfloat16),
    (3, 1, 2, 64, 48, 16, True, [47, 48, 15], [1, 0, 1], 32, True, 2, torch.float32),
    (2, 4, 3, 128, 128, 128, True, [126, 0], None, 128, True, 6, torch.float32),
    (2, 7, 2, 64, 96, 32, True, [30, 96], [7, 3], 64, False, 2, torch.float32),
    (2, 16, 2, 128, 32, 32, False, [16, 3], None, 0, False, 0, torch.float32),
    (1, 333, 2, 128, 192, 64, True, [1], None, 64, False, 3, torch.float32),
    (2, 129, 1, 128, 256, 128, True, [127, 255], [129, 1], 128, False, 5, torch.float32),
    (2, 50, 4, 64, 64, 64, True, [60, 0], [50, 9], 16, True, 4, torch.bfloat16),
    (2, 300, 2, 128, 16, 16, True, [5, 31], [300, 17], 128, False, 2, torch.float32),
    (1, 500, 2, 64, 512, 128, False, [12], None, 64, True, 9, torch.float32),
    # queries enough for four heads a thread, the last group of a row with fewer
    (2, 3300, 1, 128, 256, 128, True, [3, 0], [3300, 1000], 128, False, 6, torch.float32),
    (1, 9000, 1, 64, 128, 64, False, [0], None, 32, True, 9, torch.bfloat16),
]


def append_both(cuda_device, case, seed, scale=1.0, poke=None):
    B, S, H, D, size, block, paged, held, fresh, rotary, interleaved, Hq, dt = case
    per = max(-(-(h + S) // size) for h in held)
    if not paged:
        size, per = per * size, 1
    pages = B * per + 2
    tables = tables_of(B, per, pages, seed) if paged else [[b] for b in range(B)]
    cache = make_cache(pages, size, H, D, block, seed, cuda_device)
    fill(cache, tables, held, seed)
    g = torch.Generator().manual_seed(seed + 1)
    # the three tensors of a projection lie side by side
    qkv = (torch.randn(B, S, Hq + 2 * H, D, generator=g) * scale).bfloat16()
    if poke:
        poke(qkv[:, :, Hq:])
    cos, sin = rope(max(held) + S, rotary, dt) if rotary else (None, None)
    want = {n: getattr(cache, n).cpu().float().double() for n in ("k", "v", "k_scale", "v_scale")}
    want_q = qkv[:, :, :Hq].clone()
    for b in range(B):
        n = S if fresh is None else fresh[b]
        k, v = qkv[b, :n, Hq:Hq + H].float(), qkv[b, :n, Hq + H:].float()
        if rotary:
            k = orc.rotate(k, cos, sin, held[b], interleaved)
            if Hq:
                want_q[b] = orc.rotate(qkv[b, :, :Hq], cos, sin, held[b], interleaved).bfloat16()
        orc.append(want["k"], want["k_scale"], k, held[b], tables[b], block)
        orc.append(want["v"], want["v_scale"], v, held[b], tables[b], block)
    dev = qkv.to(cuda_device)
    q = fa.append_kv_fp8(cache, dev[:, :, Hq:Hq + H], dev[:, :, Hq + H:],
                         torch.tensor(held, dtype=torch.int32, device=cuda_device),
                         page_table=torch.tensor(tables, dtype=torch.int32, device=cuda_device) if paged else None,
                         seqused_new=None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device=cuda_device),
                         rotary_cos=cos.to(cuda_device) if rotary else None, rotary_sin=sin.to(cuda_device) if rotary else None,
                         rotary_interleaved=interleaved, q=dev[:, :, :Hq] if rotary and Hq else None)
    torch.cuda.synchronize()
    fa.check_status(cuda_device)
    for name in ("k", "v", "k_scale", "v_scale"):
        got = getattr(cache, name).cpu().float().double()
        same = (got == want[name]) | (got.isnan() & want[name].isnan())
        assert same.all(), f"{name}: {(~same).sum()} of {same.numel()} differ, first at {(~same).nonzero()[0].tolist()}"
    if rotary and Hq:
        assert torch.equal(q.cpu(), want_q)
    else:
        assert q is None


@pytest.mark.parametrize("case", APPENDS)
def test_append_gives_the_oracles_bytes(cuda_device, case):
    append_both(cuda_device, case, seed=3)


@pytest.mark.parametrize("scale", [1e-30, 1e-3, 40.0, 1e30])
def test_append_of_small_and_large_values(cuda_device, scale):
    """The block's scale grows by far (or not at all) beside what it holds."""
    append_both(cuda_device, APPENDS[1], seed=4, scale=scale)
    append_both(cuda_device, APPENDS[6], seed=5, scale=scale)


def test_append_of_values_that_are_not_finite(cuda_device):
    def poke(kv):
        kv[0, 0, 0, 5] = math.inf
        kv[0, 0, -1, 7] = -math.inf
        kv[-1, -1, -1, 9] = math.nan
        kv[-1, 0, 0] = 0
    append_both(cuda_device, APPENDS[5], seed=6, poke=poke)
    append_both(cuda_device, APPENDS[0][:9] + (0, False, 0, torch.float32), seed=7, poke=poke)


def test_tokens_one_by_one_leave_what_they_leave_at_once(cuda_device):
    """(values of one scale: where a scale grows, small values are rounded twice)"""
    g = torch.Generator().manual_seed(8)
    k = torch.randn(2, 70, 2, 128, generator=g).clamp(-3.4, 3.4).bfloat16()
    k[:, 0] = 3.4375                                 # every block's largest... of the first block: the rest follows
    k[:, 32] = 3.4375
    k[:, 64] = 3.4375
    k = k.to(cuda_device)
    caches = [make_cache(2, 96, 2, 128, 32, 1, cuda_device) for _ in range(2)]
    at = lambda n: torch.full((2,), n, dtype=torch.int32, device=cuda_device)
    fa.append_kv_fp8(caches[0], k, k, at(0))
    for i in range(70):
        fa.append_kv_fp8(caches[1], k[:, i:i + 1], k[:, i:i + 1], at(i))
    fa.check_status(cuda_device)
    for name in ("k", "v", "k_scale", "v_scale"):
        a, b = (getattr(c, name).view(torch.uint8) for c in caches)
        assert torch.equal(a, b)


def test_append_leaves_out_what_has_no_place(cuda_device):
    """Positions behind the cache's end, pages outside the pool, positions without a row in the tables: reported, the rest
    written."""
    cache = make_cache(4, 32, 1, 64, 32, 1, cuda_device)
    k = torch.randn(3, 2, 1, 64, device=cuda_device, dtype=torch.bfloat16)
    table = torch.tensor([[0, 1], [2, 7], [3, -1]], dtype=torch.int32, device=cuda_device)
    before = [getattr(cache, n).view(torch.uint8).clone() for n in ("k", "v")]
    for held, site in (([63, 0, 0], 120), ([0, 33, 0], 121), ([0, 0, 40], 121), ([-5, 0, 0], 120), ([2 ** 31 - 1, 0, 0], 120)):
        fa.append_kv_fp8(cache, k, k, torch.tensor(held, dtype=torch.int32, device=cuda_device), page_table=table)
        with pytest.raises(RuntimeError, match=f"code 2 .*site {site},"):
            fa.check_status(cuda_device)
    # sequence 1 held 33 in a page outside the pool and wrote nothing there; page 1 (of sequence 0) got its one token
    assert torch.equal(cache.k.view(torch.uint8)[1, :31], before[0][1, :31])
    assert not torch.equal(cache.k.view(torch.uint8)[1, 31], before[0][1, 31])
    cos, sin = (t.to(cuda_device) for t in rope(3, 64))
    fa.append_kv_fp8(cache, k[:1], k[:1], torch.tensor([2], dtype=torch.int32, device=cuda_device), page_table=table[:1],
                     rotary_cos=cos, rotary_sin=sin)
    with pytest.raises(RuntimeError, match="code 2 .*site 122,"):
        fa.check_status(cuda_device)
    fa.append_kv_fp8(cache, k, k, torch.tensor([1, 2, 3], dtype=torch.int32, device=cuda_device), page_table=table)
    fa.check_status(cuda_device)


def test_append_to_a_pool_of_another_order_and_from_unaligned_views(cuda_device):
    """(page, head, token) pools are views; k and v that are no 16-byte pieces are copied."""
    g = torch.Generator().manual_seed(9)
    k = torch.randn(1, 40, 2, 64, generator=g).bfloat16().to(cuda_device)
    plain = make_cache(3, 32, 2, 64, 16, 1, cuda_device)
    other = make_cache(3, 32, 2, 64, 16, 1, cuda_device)
    for n in ("k", "v"):
        t = torch.full((3, 2, 32, 64), 0x7F, dtype=torch.uint8, device=cuda_device).view(torch.float8_e4m3fn)
        setattr(other, n, t.transpose(1, 2))
    odd = torch.empty(40 * 2 * 65 + 1, device=cuda_device, dtype=torch.bfloat16)[1:].view(1, 40, 2, 65)[..., 1:]
    odd.copy_(k)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=cuda_device)
    at = torch.tensor([7], dtype=torch.int32, device=cuda_device)
    for c in (plain, other):
        c.k_scale.zero_()
        c.v_scale.zero_()
    fa.append_kv_fp8(plain, k, k, at, page_table=table)
    fa.append_kv_fp8(other, odd, odd, at, page_table=table)
    fa.check_status(cuda_device)
    for n in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(plain, n).contiguous().view(torch.uint8), getattr(other, n).contiguous().view(torch.uint8))


# ---- attention ------------------------------------------------------------------------------------------------

def attend_both(device, B, Sq, Hq, H, D, size, block, lens, fresh=None, paged=True, spread=1.0, seed=1, outlier=False, splits=0,
                q_scale=1.0, **kw):
    per = max(1, max(-(-n // size) for n in lens))
    if not paged:
        size, per = per * size, 1
    pages = B * per + 2
    tables = tables_of(B, per, pages, seed) if paged else [[b] for b in range(B)]
    cache = make_cache(pages, size, H, D, block, seed, device)
    fill(cache, tables, lens, seed, spread, outlier)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(B, Sq, Hq, D, generator=g) * q_scale).bfloat16()
    sink = torch.randn(Hq, generator=g) * 2 if kw.pop("sink", False) else None
    # entries of the table behind the last page are anybody's
    wide = [t + [10 ** 9, -7] for t in tables]
    for t, n in zip(wide, lens):
        for i in range(-(-n // size), len(t)):
            t[i] = 10 ** 9
    out = torch.full((B, Sq, Hq, D), 7.0, dtype=torch.bfloat16, device=device)
    lse = torch.full((B, Hq, Sq), 7.0, device=device)
    got, got_lse = fa.flash_attn_fp8_cache_func(
        q.to(device), cache, torch.tensor(lens, dtype=torch.int32, device=device),
        page_table=torch.tensor(wide, dtype=torch.int32, device=device) if paged else None,
        seqused_q=None if fresh is None else torch.tensor(fresh, dtype=torch.int32, device=device),
        learnable_sink=None if sink is None else sink.to(device), num_splits=splits, return_lse=True, out=out, lse=lse, **kw)
    torch.cuda.synchronize()
    fa.check_status(device)
    assert got is out and got_lse is lse
    args = dict(softmax_scale=kw.get("softmax_scale"), causal=kw.get("causal", False), window=kw.get("window_size", (None, None)),
                sink=sink, softcap=kw.get("softcap", 0.0))
    for b in range(B):
        n = Sq if fresh is None else fresh[b]
        k, v = held_of(cache, tables[b], lens[b])
        want, want_lse = orc.attend(q[b], k, v, n, **args)
        mag, _ = orc.attend(q[b], k, v.abs(), n, **args)
        o, l = out[b, :n].cpu().double(), lse[b, :, :n].cpu().double()
        top = 1.0
        if k.shape[0]:
            top = float((q[b, :n].double().norm(dim=-1).max() if n else 0.0) * k.norm(dim=-1).max()) * (kw.get("softmax_scale") or D ** -0.5)
        off = (o - want).abs()
        room = 2.0 ** -8 * (mag + want.abs()) + (2.0 ** -13 + math.expm1(2.0 * min(5.0, 2.0 ** -20 * top))) * mag + 1e-30
        assert (off <= room).all(), f"sequence {b}: {(off / room).max():.2f} of the room at {(off / room).argmax()}"
        sees = want_lse > -math.inf
        assert torch.equal(sees, l > -math.inf)
        room = 2.0 ** -18 * want_lse[sees].abs().clamp(min=1.0) + 2.0 ** -20 * top
        assert ((l[sees] - want_lse[sees]).abs() <= room).all(), f"lse off by {(l[sees] - want_lse[sees]).abs().max():.2e}, room {room.min():.2e}"
        # rows behind the last one stay as they were
        assert (out[b, n:] == 7.0).all() and (lse[b, :, n:] == 7.0).all()
    return out, lse


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("lens", [[1], [0, 5], [777, 128, 127], [16, 2049, 300, 129]])
def test_one_token(cuda_device, D, group, lens):
    attend_both(cuda_device, len(lens), 1, 2 * group, 2, D, 64, 64, lens, causal=True)


@pytest.mark.parametrize("size,block,paged", [(16, 16, True), (48, 16, True), (32, 32, True), (96, 32, True), (128, 64, True),
                                              (192, 64, True), (256, 128, True), (384, 128, True), (128, 16, True), (16, 16, False),
                                              (64, 64, False), (128, 128, False)])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_and_blocks(cuda_device, size, block, paged, D):
    attend_both(cuda_device, 3, 1, 8, 2, D, size, block, [500, 1030, 17], paged=paged, causal=True, spread=8.0)
    attend_both(cuda_device, 2, 40, 8, 2, D, size, block, [500, 333], paged=paged, causal=True, spread=8.0)


@pytest.mark.parametrize("Sq,group", [(2, 4), (3, 3), (4, 4), (5, 4), (8, 4), (7, 5), (33, 1), (9, 8), (64, 2), (130, 4), (257, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_rows(cuda_device, Sq, group, causal):
    attend_both(cuda_device, 2, Sq, 2 * group, 2, 128, 64, 64, [Sq + 300, Sq], causal=causal)
    attend_both(cuda_device, 2, Sq, 2 * group, 2, 64, 64, 64, [Sq + 300, Sq], causal=causal)


@pytest.mark.parametrize("window", [(0, 0), (15, None), (127, 0), (200, 3), (None, 5)])
@pytest.mark.parametrize("Sq,group", [(1, 4), (4, 4), (70, 4)])
def test_windows(cuda_device, window, Sq, group):
    for D in (64, 128):
        attend_both(cuda_device, 3, Sq, 2 * group, 2, D, 64, 32, [Sq + 700, Sq + 128, Sq], window_size=window,
                    causal=window[1] is None, spread=4.0)


@pytest.mark.parametrize("Sq,group", [(1, 4), (6, 2), (70, 4)])
@pytest.mark.parametrize("D", [64, 128])
def test_sink_and_softcap(cuda_device, Sq, group, D):
    lens = [Sq + 300, Sq + 5, 0]
    attend_both(cuda_device, 3, Sq, 2 * group, 2, D, 64, 32, lens, causal=True, sink=True, fresh=[Sq, Sq, Sq])
    attend_both(cuda_device, 3, Sq, 2 * group, 2, D, 64, 32, lens, causal=True, softcap=20.0, q_scale=4.0)
    attend_both(cuda_device, 3, Sq, 2 * group, 2, D, 64, 32, lens, window_size=(40, 0), sink=True, softcap=5.0)


@pytest.mark.parametrize("Sq,group", [(1, 4), (6, 2), (70, 4)])
def test_padded_batches_and_rows_that_see_nothing(cuda_device, Sq, group):
    """Rows behind seqused_q are left alone; with fewer keys than rows the first rows see nothing."""
    for D in (64, 128):
        attend_both(cuda_device, 4, Sq, 2 * group, 2, D, 64, 64, [300, 40, max(1, Sq // 2), 0], fresh=[Sq, max(1, Sq - 3), Sq, Sq], causal=True)
        attend_both(cuda_device, 3, Sq, 2 * group, 2, D, 64, 64, [300, 40, 7], fresh=[0, Sq, 1], causal=True)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 128])
@pytest.mark.parametrize("Sq,group,D", [(1, 8, 128), (5, 4, 128), (1, 4, 64), (60, 4, 128), (60, 4, 64)])
def test_splits(cuda_device, splits, Sq, group, D):
    attend_both(cuda_device, 2, Sq, group * 2, 2, D, 64, 64, [Sq + 1500, Sq + 100], causal=True, splits=splits, sink=True)
    attend_both(cuda_device, 2, Sq, group * 2, 2, D, 64, 64, [Sq + 1500, Sq + 100], splits=splits, window_size=(300, 0))


@pytest.mark.parametrize("Sq", [1, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_strong_channels_and_unequal_blocks(cuda_device, Sq, D):
    """Scores far apart, keys of a few strong channels, values whose blocks differ by orders of magnitude."""
    attend_both(cuda_device, 2, Sq, 8, 2, D, 64, 16, [Sq + 900, Sq + 40], causal=True, spread=30.0, outlier=True, q_scale=6.0)
    attend_both(cuda_device, 2, Sq, 8, 2, D, 64, 16, [Sq + 900, Sq + 40], causal=True, q_scale=1e-3)
    attend_both(cuda_device, 1, Sq, 8, 2, D, 64, 16, [Sq + 900], causal=True, q_scale=30.0, softmax_scale=1.0)


def test_many_sequences(cuda_device):
    lens = [(37 * b) % 700 for b in range(150)]
    attend_both(cuda_device, 150, 1, 4, 1, 128, 32, 32, lens, causal=True)
    attend_both(cuda_device, 150, 2, 8, 2, 64, 32, 32, lens, causal=True)


def test_a_prompt_appended_and_attended_step_by_step(cuda_device):
    """The calls of a serving loop: a ragged batch of prompts in two pieces, then tokens one by one, one graph for the steps;
    attention of all rows against the oracle over what the cache holds."""
    B, H, G, D, size, block = 3, 2, 8, 128, 32, 32
    lens, steps = [90, 41, 7], 6
    per = -(-(max(lens) + steps) // size)
    tables = tables_of(B, per, B * per + 1, 5)
    table = torch.tensor(tables, dtype=torch.int32, device=cuda_device)
    cache = make_cache(B * per + 1, size, H, D, block, 5, cuda_device)
    g = torch.Generator().manual_seed(6)
    T = max(lens) + steps
    q, k, v = ((torch.randn(B, T, n, D, generator=g)).bfloat16().to(cuda_device) for n in (G, H, H))
    cos, sin = (t.to(cuda_device) for t in rope(T, D))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    outs = [[] for _ in range(B)]
    held = [0] * B
    turned = [[] for _ in range(B)]
    for piece in (max(lens) // 2, max(lens) - max(lens) // 2):
        n = [max(0, min(piece, lens[b] - held[b])) for b in range(B)]
        part = [torch.stack([torch.cat([x[b, held[b]:held[b] + n[b]], x[b, :piece - n[b]]]) for b in range(B)]) for x in (q, k, v)]
        qr = fa.append_kv_fp8(cache, part[1], part[2], i32(held), page_table=table, seqused_new=i32(n), rotary_cos=cos, rotary_sin=sin, q=part[0])
        held = [h + m for h, m in zip(held, n)]
        out, _ = fa.flash_attn_fp8_cache_func(qr, cache, i32(held), page_table=table, seqused_q=i32(n), causal=True)
        for b in range(B):
            outs[b].append(out[b, :n[b]].clone())
            turned[b].append(qr[b, :n[b]].clone())
    # one step, captured, the lengths counted on the device
    at = i32(held)
    one = [torch.zeros(B, 1, x.shape[2], D, dtype=torch.bfloat16, device=cuda_device) for x in (q, k, v)]

    def step():
        qr = fa.append_kv_fp8(cache, one[1], one[2], at, page_table=table, rotary_cos=cos, rotary_sin=sin, q=one[0])
        at.add_(1)
        return qr, fa.flash_attn_fp8_cache_func(qr, cache, at, page_table=table, causal=True, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t, x in zip(one, (q, k, v)):
            t.copy_(torch.stack([x[b, held[b]] for b in range(B)])[:, None])
        step()
        at.sub_(1)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        qr, (out, _) = step()
    for i in range(steps):
        for t, x in zip(one, (q, k, v)):
            t.copy_(torch.stack([x[b, lens[b] + i] for b in range(B)])[:, None])
        graph.replay()
        for b in range(B):
            outs[b].append(out[b].clone())
            turned[b].append(qr[b].clone())
    torch.cuda.synchronize()
    fa.check_status(cuda_device)
    for b in range(B):
        n = lens[b] + steps
        kk, vv = held_of(cache, tables[b], n)
        # (an early row met scales that grew later: blocks of one magnitude keep theirs within a factor of two, which a token
        # of the same distribution raises without moving the bytes that stay above 2^-6)
        want, _ = orc.attend(torch.cat(turned[b]).cpu(), kk, vv, n, causal=True)
        mag, _ = orc.attend(torch.cat(turned[b]).cpu(), kk, vv.abs(), n, causal=True)
        off = (torch.cat(outs[b]).cpu().double() - want).abs()
        assert (off <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -11 * mag).all()


def test_another_stream_and_strided_operands(cuda_device):
    """q and out as slices of larger tensors, on a side stream, the pool in (page, head, token) order."""
    cache = make_cache(4, 64, 2, 128, 64, 1, cuda_device)
    tables = [[2, 0], [3, 1]]
    fill(cache, tables, [100, 65], 1)
    moved = fa.FP8KVCache(*(getattr(cache, n).transpose(1, 2).contiguous().transpose(1, 2) for n in ("k", "v")), cache.k_scale, cache.v_scale)
    table = torch.tensor(tables, dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([100, 65], dtype=torch.int32, device=cuda_device)
    for Sq in (1, 33):
        big = torch.randn(2, Sq, 24, 128, device=cuda_device).bfloat16()
        want, _ = fa.flash_attn_fp8_cache_func(big[:, :, 8:16].contiguous(), cache, lens, page_table=table, causal=True)
        torch.cuda.synchronize()
        room = torch.zeros(2, Sq, 24, 128, device=cuda_device, dtype=torch.bfloat16)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fa.flash_attn_fp8_cache_func(big[:, :, 8:16], moved, lens, page_table=table, causal=True, out=room[:, :, 8:16])
        side.synchronize()
        fa.check_status(cuda_device)
        assert torch.equal(room[:, :, 8:16], want)
        assert not room[:, :, :8].any() and not room[:, :, 16:].any()


def test_same_call_gives_the_same_bits(cuda_device):
    cache = make_cache(40, 64, 2, 128, 64, 1, cuda_device)
    tables = [list(range(20)), list(range(20, 40))]
    fill(cache, tables, [1280, 700], 1)
    table = torch.tensor(tables, dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([1280, 700], dtype=torch.int32, device=cuda_device)
    for Sq in (1, 4, 200):
        q = torch.randn(2, Sq, 8, 128, device=cuda_device).bfloat16()
        a = [fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, return_lse=True) for _ in range(8)]
        torch.cuda.synchronize()
        fa.check_status(cuda_device)
        for out, lse in a[1:]:
            assert torch.equal(out, a[0][0]) and torch.equal(lse, a[0][1])


def test_bad_pages_are_reported(cuda_device):
    """A page outside the pool stands for keys and values of zero."""
    cache = make_cache(3, 64, 1, 128, 64, 1, cuda_device)
    fill(cache, [[0, 1]], [128], 1)
    lens = torch.tensor([128], dtype=torch.int32, device=cuda_device)
    for Sq in (1, 40):
        q = torch.randn(1, Sq, 4, 128, device=cuda_device).bfloat16()
        for bad in (3, -1, 10 ** 9):
            got, _ = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=torch.tensor([[0, bad]], dtype=torch.int32, device=cuda_device))
            with pytest.raises(RuntimeError, match="code 2 .*site 121,"):
                fa.check_status(cuda_device)
            k, v = held_of(cache, [0], 64)
            z = torch.zeros_like(k)
            want, _ = orc.attend(q[0].cpu(), torch.cat([k, z]), torch.cat([v, z]), Sq)
            mag, _ = orc.attend(q[0].cpu(), torch.cat([k, z]), torch.cat([v, z]).abs(), Sq)
            assert ((got[0].cpu().double() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -13 * mag).all()


@pytest.mark.parametrize("B,Sq,Hq,H,D,size,block,n", [(4, 1, 64, 8, 128, 128, 128, 40000), (8, 1, 32, 8, 128, 64, 64, 9999), (6, 4, 32, 8, 128, 16, 16, 12345),
                                                      (6, 1, 32, 8, 64, 32, 32, 12345), (3, 7, 16, 4, 128, 64, 64, 30001), (4, 2, 64, 8, 64, 64, 64, 20000),
                                                      (1, 200, 32, 8, 128, 128, 128, 20000), (2, 333, 16, 2, 64, 64, 64, 9999)])
@pytest.mark.parametrize("splits", [0, 1, 5])
def test_long_contexts_on_a_full_gpu(cuda_device, B, Sq, Hq, H, D, size, block, n, splits):
    """Every SM busy with several tiles in flight, three times in a row: the same bits, and those of the oracle (on the GPU here)."""
    per = -(-n // size)
    cache = make_cache(B * per, size, H, D, block, 1, "cpu", nan=False)
    cache = fa.FP8KVCache(*(getattr(cache, f).to(cuda_device) for f in ("k", "v", "k_scale", "v_scale")))
    g = torch.Generator(device=cuda_device).manual_seed(1)
    for x, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x.copy_((torch.randn(x.shape, generator=g, device=cuda_device) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn))
        sc.mul_(0.02).add_(0.005)
    order = torch.randperm(B * per, generator=g, device=cuda_device).view(B, per)
    q = torch.randn(B, Sq, Hq, D, generator=g, device=cuda_device).bfloat16()
    lens = torch.tensor([n - 7 * b for b in range(B)], dtype=torch.int32, device=cuda_device)
    got = [fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=order.int(), causal=True, num_splits=splits, return_lse=True) for _ in range(3)]
    torch.cuda.synchronize()
    fa.check_status(cuda_device)
    for out, lse in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(lse, got[0][1])
    k, v = cache.dequantize()
    for b in (0, B - 1):
        kb, vb = (x[order[b]].flatten(0, 1)[:int(lens[b])].double() for x in (k, v))
        want, want_lse = orc.attend(q[b], kb, vb, Sq, causal=True)
        mag, _ = orc.attend(q[b], kb, vb.abs(), Sq, causal=True)
        off = (got[0][0][b].double() - want).abs()
        # 2^-8 of each weight in the worst case.  Thousands of independent roundings do not add up like that: the output's own have a root
        # mean square below 2^-8 / sqrt(3) of it, those of the weights (2^-9 of each at most) one below 2^-9 sqrt(sum p^2 v^2), and with values of
        # random signs that root is the size of an output.  So the norm is off by less than 2^-8 of it, which a wrong scale of one tile is not.
        assert (off <= 2.0 ** -8 * (mag + want.abs())).all()
        assert off.norm() <= 2.0 ** -8 * want.norm()
        assert (got[0][1][b].double() - want_lse).abs().max() <= 2.0 ** -18 * want_lse.abs().max()


@pytest.mark.parametrize("B,Sq,Hq,H,D,n", [(1, 64, 8, 2, 128, 64), (1, 200, 8, 2, 64, 1000), (1, 130, 16, 1, 128, 5000), (3, 150, 8, 4, 128, 1500), (9, 100, 16, 4, 64, 700),
                                           (2, 600, 16, 8, 128, 600), (1, 33, 8, 8, 128, 9000), (2, 40, 40, 1, 128, 300)])
def test_rows_of_a_cta_and_splits(cuda_device, B, Sq, Hq, H, D, n):
    """Many rows, few or many CTAs, short or long: tiles of 128 and of 256 rows, with and without splits."""
    attend_both(cuda_device, B, Sq, Hq, H, D, 64, 64, [n - 17 * b for b in range(B)], fresh=[Sq - 11 * b for b in range(B)], causal=True)
    attend_both(cuda_device, B, Sq, Hq, H, D, 64, 64, [n - 17 * b for b in range(B)], window_size=(300, 20))


@pytest.mark.parametrize("softcap", [0.5, 2.0, 8.0, 50.0])
@pytest.mark.parametrize("Sq", [1, 70])
def test_soft_caps_below_and_above_the_scores(cuda_device, Sq, softcap):
    """Scores of a few units: warps whose scores are all well below the cap, all above, and both."""
    for D, q_scale in ((64, 1.0), (128, 3.0)):
        attend_both(cuda_device, 2, Sq, 8, 2, D, 64, 64, [Sq + 700, Sq + 5], causal=True, softcap=softcap, q_scale=q_scale)


@pytest.mark.parametrize("B,Sq,Hq,H", [(9, 3, 24, 12), (9, 1, 14, 7), (9, 2, 11, 11), (70, 4, 8, 8), (9, 40, 24, 12)])
@pytest.mark.parametrize("splits", [0, 2])
def test_sequences_without_rows_or_keys_between_others(cuda_device, B, Sq, Hq, H, splits):
    lens = [(b * 211) % 900 if b % 4 else 0 for b in range(B)]
    fresh = [0 if b % 3 == 1 else max(1, Sq - b % 3) for b in range(B)]
    attend_both(cuda_device, B, Sq, Hq, H, 64, 32, 32, lens, fresh=fresh, causal=True, splits=splits)
    attend_both(cuda_device, B, Sq, Hq, H, 128, 32, 32, lens, fresh=[0] * (B - 1) + [1], causal=True, splits=splits)


def batch_of(device, B, n, H=2, D=128, size=64, seed=1):
    """A cache of B sequences of n tokens, its table."""
    per = -(-n // size)
    cache = make_cache(B * per + 1, size, H, D, 64, seed, "cpu")
    cache = fa.FP8KVCache(*(getattr(cache, f).to(device) for f in ("k", "v", "k_scale", "v_scale")))
    tables = tables_of(B, per, B * per + 1, seed)
    fill(cache, tables, [n] * B, seed)
    return cache, torch.tensor(tables, dtype=torch.int32, device=device)


@pytest.mark.parametrize("Sq", [1, 6, 100])
@pytest.mark.parametrize("splits", [1, 3])
def test_a_chosen_split_count_gives_the_bits_of_the_entry_alone(cuda_device, Sq, splits):
    cache, table = batch_of(cuda_device, 5, 1000)
    lens = torch.tensor([1000, 3, 640, 641, 129], dtype=torch.int32, device=cuda_device)
    q = torch.randn(5, Sq, 8, 128, device=cuda_device).bfloat16()
    out, lse = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, num_splits=splits, return_lse=True)
    for b in range(5):
        o, l = fa.flash_attn_fp8_cache_func(q[b:b + 1], cache, lens[b:b + 1], page_table=table[b:b + 1], causal=True, num_splits=splits, return_lse=True)
        assert torch.equal(o[0], out[b]) and torch.equal(l[0], lse[b])
    fa.check_status(cuda_device)


def test_keys_that_no_row_sees_may_be_anything(cuda_device):
    """NaN bytes and NaN scales in front of a window and behind the last token; pages of the table there that do not exist."""
    cache, table = batch_of(cuda_device, 2, 1000)
    lens = torch.tensor([950, 700], dtype=torch.int32, device=cuda_device)
    for Sq, Hq in ((1, 8), (6, 8), (50, 8), (200, 8)):
        for cap in (0.0, 10.0):
            q = torch.randn(2, Sq, Hq, 128, device=cuda_device).bfloat16()
            args = dict(page_table=table, window_size=(100, 0), softcap=cap, return_lse=True)
            want = fa.flash_attn_fp8_cache_func(q, cache, lens, **args)
            bad = fa.FP8KVCache(cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone())
            gone = table.clone()
            for b, n in enumerate([950, 700]):
                first = max(0, n - Sq - 100)       # row 0 stands at n - Sq and sees 100 keys in front of it
                for i, page in enumerate(table[b].tolist()):
                    seen_lo, seen_hi = max(0, first - 64 * i), min(64, n - 64 * i)
                    if seen_hi <= 0 or seen_lo >= 64:
                        gone[b, i] = -5
                        bad.k_scale[page] = bad.v_scale[page] = math.nan
                        seen_lo, seen_hi = 64, 64
                    for t in (bad.k, bad.v):
                        t[page, :seen_lo].view(torch.uint8).fill_(0x7F)
                        t[page, max(0, seen_hi):].view(torch.uint8).fill_(0x7F)
            args["page_table"] = gone
            got = fa.flash_attn_fp8_cache_func(q, bad, lens, **args)
            fa.check_status(cuda_device)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_calls_on_two_streams_at_once(cuda_device):
    """Workspaces and results of calls that run side by side are their own."""
    cache, table = batch_of(cuda_device, 4, 2000)
    lens = torch.tensor([2000, 1500, 77, 1999], dtype=torch.int32, device=cuda_device)
    sizes = [(1, 4, 0), (5, 4, 0), (120, 8, 0), (1, 4, 4), (120, 8, 3)]
    qs = [[torch.randn(4, Sq, Hq, 128, device=cuda_device).bfloat16() for _ in range(2)] for Sq, Hq, _ in sizes]
    run = lambda q, sp: fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, num_splits=sp)[0]
    want = [[run(q, size[2]) for q in pair] for pair, size in zip(qs, sizes)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for i, (pair, size) in enumerate(zip(qs, sizes)):
            for j in (0, 1):
                with torch.cuda.stream(streams[j]):
                    got[j].append((i, run(pair[j], size[2])))
    torch.cuda.synchronize()
    fa.check_status(cuda_device)
    for j in (0, 1):
        for i, out in got[j]:
            assert torch.equal(out, want[i][j])


@pytest.mark.parametrize("Sq,splits", [(1, 0), (6, 0), (1, 3), (90, 0), (90, 2)])
def test_a_replayed_graph_reads_the_lengths_anew(cuda_device, Sq, splits):
    cache, table = batch_of(cuda_device, 4, 1500)
    q = torch.randn(4, Sq, 8, 128, device=cuda_device).bfloat16()
    lens = torch.tensor([1, 1, 1, 1], dtype=torch.int32, device=cuda_device)
    rows = torch.tensor([Sq] * 4, dtype=torch.int32, device=cuda_device)
    out, lse = torch.zeros_like(q), torch.zeros(4, 8, Sq, device=cuda_device)
    run = lambda **kw: fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, seqused_q=rows, causal=True, num_splits=splits, return_lse=True, **kw)
    run()
    torch.cuda.synchronize()
    graph, twin = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(out=out, lse=lse)
    with torch.cuda.graph(twin):
        again = run()
    for new, n in (([1500, 3, 0, 900], [Sq, 1, Sq, 0]), ([64, 1499, 1024, 1], [Sq] * 4), ([0, 0, 0, 0], [Sq] * 4), ([1500] * 4, [Sq, 0, 0, Sq])):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        rows.copy_(torch.tensor(n, dtype=torch.int32))
        want = run()
        out.zero_()
        lse.zero_()
        graph.replay()
        twin.replay()
        fa.check_status(cuda_device)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        for a, w in zip(again, want):
            assert torch.equal(a, w)


def test_offsets_that_pass_32_bits(cuda_device):
    """Pages 2^31 + 2^20 bytes apart: the bytes and the results of a compact pool."""
    far = (1 << 31) + (1 << 20)
    compact = make_cache(3, 256, 2, 128, 64, 1, cuda_device)
    room = [torch.empty(2 * far + 256 * 2 * 128, dtype=torch.uint8, device=cuda_device) for _ in range(2)]
    wide = fa.FP8KVCache(*(t.as_strided((3, 256, 2, 128), (far, 256, 128, 1)) for t in room), torch.empty_like(compact.k_scale), torch.empty_like(compact.v_scale))
    k, v = (torch.randn(1, 600, 2, 128, device=cuda_device).bfloat16() for _ in range(2))
    table = torch.tensor([[2, 1, 0]], dtype=torch.int32, device=cuda_device)
    for c in (compact, wide):
        c.k_scale.zero_()
        c.v_scale.zero_()
        for x in (c.k, c.v):
            for page in range(3):
                x[page].view(torch.uint8).fill_(0x7F)
        fa.append_kv_fp8(c, k, v, torch.zeros(1, dtype=torch.int32, device=cuda_device), page_table=table)
        fa.append_kv_fp8(c, k[:, :1], v[:, :1], torch.full((1,), 600, dtype=torch.int32, device=cuda_device), page_table=table)
    for a, b in ((compact.k, wide.k), (compact.v, wide.v)):
        assert all(torch.equal(a[p].view(torch.uint8), b[p]) for p in range(3))
    lens = torch.tensor([601], dtype=torch.int32, device=cuda_device)
    for Sq in (1, 100):
        q = torch.randn(1, Sq, 4, 128, device=cuda_device).bfloat16()
        got = [fa.flash_attn_fp8_cache_func(q, c, lens, page_table=table, causal=True)[0] for c in (compact, wide)]
        assert torch.equal(*got)
    fa.check_status(cuda_device)


def test_operands_that_start_between_pieces_are_copied(cuda_device):
    """Contiguous, but two bytes behind a 16-byte boundary."""
    cache, table = batch_of(cuda_device, 1, 200)
    lens = torch.tensor([150], dtype=torch.int32, device=cuda_device)
    for Sq in (1, 40):
        q = torch.randn(1, Sq, 8, 128, device=cuda_device).bfloat16()
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=cuda_device)[1:].view(q.shape)
        odd.copy_(q)
        got = [fa.flash_attn_fp8_cache_func(x, cache, lens, page_table=table, causal=True)[0] for x in (q, odd)]
        assert torch.equal(*got)
        twin = fa.FP8KVCache(*(getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")))
        for c, x in ((cache, q), (twin, odd)):
            fa.append_kv_fp8(c, x[:, :, :2], x[:, :, 2:4].contiguous(), lens, page_table=table)
        assert torch.equal(cache.k.view(torch.uint8), twin.k.view(torch.uint8)) and torch.equal(cache.v.view(torch.uint8), twin.v.view(torch.uint8))


def test_refusals_on_the_gpu(cuda_device):
    cache, table = batch_of(cuda_device, 2, 100)
    lens = torch.tensor([90, 80], dtype=torch.int32, device=cuda_device)
    q = torch.zeros(2, 1, 8, 128, dtype=torch.bfloat16, device=cuda_device)
    ok = dict(page_table=table)
    call = lambda q=q, cache=cache, lens=lens, **kw: fa.flash_attn_fp8_cache_func(q, cache, lens, **dict(ok, **kw))
    for bad in (dict(q=q.half()), dict(q=q[:, :, :3]), dict(q=q[:1]), dict(lens=lens.long()), dict(lens=lens[:1]), dict(page_table=table.long()),
                dict(page_table=table[:1]), dict(seqused_q=lens.cpu()), dict(out=q[..., :64]), dict(out=torch.zeros(2, 1, 8, 132, dtype=q.dtype, device=cuda_device)[..., 4:]),
                dict(lse=torch.zeros(2, 1, 8, device=cuda_device)), dict(learnable_sink=torch.zeros(3, device=cuda_device)), dict(softcap=-1.0),
                dict(softcap=math.inf), dict(softmax_scale=0.0), dict(num_splits=129), dict(num_splits=-1)):
        with pytest.raises((AssertionError, ValueError, TypeError, RuntimeError, NotImplementedError)):
            call(**bad)
    k = torch.zeros(2, 3, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    cos = torch.zeros(200, 64, device=cuda_device)
    put = lambda k=k, v=k, lens=lens, **kw: fa.append_kv_fp8(cache, k, v, lens, **dict(ok, **kw))
    for bad in (dict(k=k.float()), dict(v=k[:, :2]), dict(k=k[:, :, :1], v=k[:, :, :1]), dict(lens=lens.float()), dict(seqused_new=lens[:1]), dict(q=k),
                dict(rotary_cos=cos), dict(rotary_cos=cos, rotary_sin=cos.bfloat16()), dict(rotary_cos=cos[:, :4], rotary_sin=cos[:, :4]),
                dict(rotary_cos=cos.cpu(), rotary_sin=cos.cpu()), dict(rotary_cos=cos, rotary_sin=cos, q=k[:, :1]), dict(page_table=None, k=k.repeat(9, 1, 1, 1), v=k.repeat(9, 1, 1, 1), lens=lens.repeat(9))):
        with pytest.raises((AssertionError, ValueError, TypeError, RuntimeError, NotImplementedError)):
            put(**bad)
    torch.cuda.synchronize()
    fa.check_status(cuda_device)


def test_blocks_whose_scale_is_zero(cuda_device):
    """Keys and values of zero, among others, next to masked keys."""
    cache, table = batch_of(cuda_device, 1, 600)
    g = torch.Generator().manual_seed(3)
    for t in (cache.k_scale, cache.v_scale):
        t.mul_((torch.rand(t.shape, generator=g) < 0.6).to(t))
    lens = torch.tensor([590], dtype=torch.int32, device=cuda_device)
    k, v = held_of(cache, table[0].tolist(), 590)
    assert (k.abs().amax(dim=-1) == 0).any() and (v.abs().amax(dim=-1) == 0).any()
    for Sq in (1, 6, 90):
        for kw in (dict(causal=True), dict(window_size=(70, 0)), dict(causal=True, softcap=10.0)):
            q = torch.randn(1, Sq, 8, 128, generator=g).bfloat16()
            out, lse = fa.flash_attn_fp8_cache_func(q.to(cuda_device), cache, lens, page_table=table, return_lse=True, **kw)
            fa.check_status(cuda_device)
            args = dict(causal=kw.get("causal", False), window=kw.get("window_size", (None, None)), softcap=kw.get("softcap", 0.0))
            want, want_lse = orc.attend(q[0], k, v, Sq, **args)
            mag, _ = orc.attend(q[0], k, v.abs(), Sq, **args)
            assert ((out[0].cpu().double() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -13 * mag).all()
            assert ((lse[0].cpu().double() - want_lse).abs() <= 2.0 ** -17 * want_lse.abs().clamp(min=1.0)).all()


def test_lengths_beyond_the_end_count_as_the_end(cuda_device):
    cache, table = batch_of(cuda_device, 2, 256)
    for Sq in (1, 50):
        q = torch.randn(2, Sq, 8, 128, device=cuda_device).bfloat16()
        call = lambda n: fa.flash_attn_fp8_cache_func(q, cache, torch.tensor(n, dtype=torch.int32, device=cuda_device), page_table=table, causal=True, return_lse=True)
        for a, b in zip(call([2 ** 31 - 1, -5]), call([256, 0])):
            assert torch.equal(a, b)
        fa.check_status(cuda_device)


def test_more_than_a_million_rows(cuda_device):
    cache, table = batch_of(cuda_device, 1, 200)
    lens = torch.tensor([200], dtype=torch.int32, device=cuda_device)
    q = torch.randn(1, 40000, 32, 128, device=cuda_device, dtype=torch.bfloat16)
    out, lse = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, num_splits=1, return_lse=True)
    for a, b in ((0, 4096), (20000, 20001 + 64), (39936, 40000)):
        o, l = fa.flash_attn_fp8_cache_func(q[:, a:b], cache, lens, page_table=table, num_splits=1, return_lse=True)
        assert torch.equal(o, out[:, a:b]) and torch.equal(l, lse[:, :, a:b])
    fa.check_status(cuda_device)


@pytest.mark.parametrize("Sq", [1, 70])
def test_soft_cap_of_small_scores(cuda_device, Sq):
    """Scores far below the cap are the scores: lse of one key is its score, to the room of a score itself."""
    for n in (1, 3):
        attend_both(cuda_device, 6, Sq, 8, 2, 128, 64, 64, [n] * 6, softcap=50.0, spread=8.0, seed=5)
        attend_both(cuda_device, 6, Sq, 8, 2, 64, 64, 64, [n] * 6, softcap=50.0, spread=8.0, seed=6)


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("Sq,group", [(1, 4), (6, 2), (70, 4)])
def test_sinks_that_are_switched_off(cuda_device, Sq, group, splits):
    """A sink of -inf adds nothing: a row that sees no key either gets zeros and -inf, the others what they get without sinks."""
    Hq = 2 * group
    off = torch.arange(Hq) % 3 == 0
    sink = torch.where(off, -math.inf, torch.linspace(-2.0, 2.0, Hq))
    cache, table = batch_of(cuda_device, 4, 1000)
    lens = torch.tensor([1000, 0, max(1, Sq // 2), Sq], dtype=torch.int32, device=cuda_device)
    q = torch.randn(4, Sq, Hq, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device)
    call = lambda **kw: fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, causal=True, num_splits=splits, return_lse=True, **kw)
    out, lse = (x.cpu() for x in call(learnable_sink=sink.to(cuda_device)))
    plain, plain_lse = (x.cpu() for x in call())
    fa.check_status(cuda_device)
    assert torch.equal(out[:, :, off], plain[:, :, off]) and torch.equal(lse[:, off], plain_lse[:, off])
    blind = plain_lse[:, 0] == -math.inf                    # (B, Sq): alike for all heads
    assert blind[1].all() and blind[2, :Sq - max(1, Sq // 2)].all() and not blind[0].any()
    assert not out[blind].any()
    # the sink alone, times log2 e and times ln 2: two products and two constants off by 2^-24 each
    alone = sink[None, :, None].expand_as(lse).transpose(1, 2)[blind]
    got = lse.transpose(1, 2)[blind]
    assert torch.equal(got == -math.inf, alone == -math.inf)
    live = alone > -math.inf
    assert ((got - alone)[live].abs() <= 2.0 ** -22 * alone[live].abs()).all()


@pytest.mark.parametrize("Sq", [1, 6, 70])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_rows_of_nan_beside_a_sink(cuda_device, Sq, splits):
    """A sequence whose keys are all NaN: out and lse are NaN, with a sink too; its neighbour is what it was."""
    cache, table = batch_of(cuda_device, 2, 300)
    for page in table[0].tolist():
        cache.k[page].view(torch.uint8).fill_(0x7F)
    lens = torch.tensor([300, 290], dtype=torch.int32, device=cuda_device)
    q = torch.randn(2, Sq, 8, 128, device=cuda_device).bfloat16()
    for sink in (None, torch.linspace(-1.0, 1.0, 8, device=cuda_device)):
        out, lse = fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, learnable_sink=sink, num_splits=splits, return_lse=True)
        fa.check_status(cuda_device)
        assert out[0].isnan().all() and lse[0].isnan().all()
        assert out[1].isfinite().all() and lse[1].isfinite().all()


def test_an_expired_wait_takes_the_place_of_a_bad_index(cuda_device):
    """A bad index stopped nothing; behind it a wait that runs out is what the caller has to know.  The first expired wait stays."""
    word = fa.interface.DeviceStatus.word(cuda_device)
    expire = lambda: fa.lib().fa4_nvfp4_debug_wait_expiry(word.data_ptr(), 5_000_000, None)
    for before, after in ((0x02780503, "site 99,"), (0, "site 99,"), (0x01640700, "site 100, launch epoch 7,")):
        word.fill_(before)
        assert expire() == 0
        with pytest.raises(RuntimeError, match=f"code 1 .*bounded wait expired.*{after}"):
            fa.check_status(cuda_device)
        fa.check_status(cuda_device)


@pytest.mark.parametrize("byte", [0x7E, 0xFE, 0x7F])
@pytest.mark.parametrize("softcap", [0.0, 3.0, 10.0, 50.0])
def test_bytes_that_no_row_sees_leave_the_bits(cuda_device, byte, softcap):
    """The largest values, of either sign, and NaN in front of the window and behind the last token, in blocks that are seen too."""
    cache, table = batch_of(cuda_device, 2, 1000)
    lens = [950, 700]
    n = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    for Sq in (1, 6, 50, 200):
        q = torch.randn(2, Sq, 8, 128, generator=torch.Generator().manual_seed(Sq)).bfloat16().to(cuda_device)
        call = lambda c: fa.flash_attn_fp8_cache_func(q, c, n, page_table=table, window_size=(100, 0), softcap=softcap, return_lse=True)
        want = call(cache)
        bad = fa.FP8KVCache(cache.k.clone(), cache.v.clone(), cache.k_scale, cache.v_scale)
        for b, m in enumerate(lens):
            first = max(0, m - Sq - 100)
            for i, page in enumerate(table[b].tolist()):
                for t in (bad.k, bad.v):
                    t[page, :min(64, max(0, first - 64 * i))].view(torch.uint8).fill_(byte)
                    t[page, min(64, max(0, m - 64 * i)):].view(torch.uint8).fill_(byte)
        got = call(bad)
        fa.check_status(cuda_device)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def attend_values(device, cache, table, lens, q, **kw):
    """A call against 64 bits, in the room that the head of this file derives (and half a step of the smallest bf16 values, 2^-134)."""
    n = torch.tensor(lens, dtype=torch.int32, device=device)
    out, lse = fa.flash_attn_fp8_cache_func(q.to(device), cache, n, page_table=table, return_lse=True, **kw)
    torch.cuda.synchronize()
    fa.check_status(device)
    args = dict(causal=kw.get("causal", False), window=kw.get("window_size", (None, None)), softcap=kw.get("softcap", 0.0))
    for b, m in enumerate(lens):
        k, v = held_of(cache, table[b].tolist(), m)
        want, want_lse = orc.attend(q[b], k, v, q.shape[1], **args)
        mag, _ = orc.attend(q[b], k, v.abs(), q.shape[1], **args)
        top = float(q[b].double().norm(dim=-1).max() * k.norm(dim=-1).max()) * q.shape[-1] ** -0.5
        off = (out[b].cpu().double() - want).abs()
        room = 2.0 ** -8 * (mag + want.abs()) + (2.0 ** -13 + math.expm1(2.0 * min(5.0, 2.0 ** -20 * top))) * mag + 2.0 ** -134
        assert (off <= room).all(), f"sequence {b}: {(off / room).max():.3g} of the room, first at {(~(off <= room)).nonzero()[0].tolist()}"
        assert ((lse[b].cpu().double() - want_lse).abs() <= 2.0 ** -18 * want_lse.abs().clamp(min=1.0) + 2.0 ** -20 * top).all()


def cache_of_scales(device, exponent, seed=2):
    """Two sequences of 1000 tokens: values up to 200 x 2^exponent or twice that."""
    cache, table = batch_of(device, 2, 1000)
    g = torch.Generator().manual_seed(seed)
    cache.v.copy_((torch.randn(cache.v.shape, generator=g) * 100).clamp(-200, 200).to(torch.float8_e4m3fn))
    cache.v_scale.copy_(2.0 ** (exponent + torch.randint(0, 2, cache.v_scale.shape, generator=g)))
    return cache, table


@pytest.mark.parametrize("exponent", [-120, -110, 100, 115])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_many_rows_on_value_scales_at_the_ends_of_their_range(cuda_device, exponent, splits):
    """(hundreds of keys of much the same weight, and few that outweigh the others)"""
    cache, table = cache_of_scales(cuda_device, exponent)
    for q_scale in (0.1, 1.0, 4.0):
        q = (torch.randn(2, 70, 8, 128, generator=torch.Generator().manual_seed(4)) * q_scale).bfloat16()
        attend_values(cuda_device, cache, table, [1000, 640], q, causal=True, num_splits=splits)


@pytest.mark.parametrize("exponent", [-19, -25, -35, -60])
@pytest.mark.parametrize("D,splits,softcap", [(128, 0, 0.0), (64, 0, 0.0), (128, 3, 0.0), (128, 1, 20.0)])
def test_small_values_in_front_of_large_ones(cuda_device, exponent, D, splits, softcap):
    """A causal prompt whose values grow: an early row's result is right to its own values, whatever the rows beside it see."""
    cache = make_cache(16, 32, 2, D, 16, 1, cuda_device)
    tables = tables_of(2, 7, 16, 1)
    fill(cache, tables, [200, 200], 1)
    table = torch.tensor(tables, dtype=torch.int32, device=cuda_device)
    g = torch.Generator().manual_seed(3)
    for b in range(2):
        for i in range(13):
            cache.v_scale[tables[b][i // 2], i % 2] = 2.0 ** max(-120, -8 + (2 * exponent if i == 0 else exponent if i < 3 else 0))
    for q_scale in (1.0, 4.0):
        attend_values(cuda_device, cache, table, [200, 197], (torch.randn(2, 197, 8, D, generator=g) * q_scale).bfloat16(), causal=True,
                      num_splits=splits, softcap=softcap)
        attend_values(cuda_device, cache, table, [200, 197], (torch.randn(2, 197, 8, D, generator=g) * q_scale).bfloat16(), window_size=(20, 0),
                      num_splits=splits, softcap=softcap)


@pytest.mark.parametrize("splits", [0, 2, 3, 16])
def test_parts_of_the_largest_values_are_merged(cuda_device, splits):
    """Values up to 2^127 or so: the sum of the parts of a row lies beyond fp32, their mean does not."""
    cache, table = cache_of_scales(cuda_device, 118)
    for q_scale in (0.1, 1.0):
        q = (torch.randn(2, 70, 8, 128, generator=torch.Generator().manual_seed(4)) * q_scale).bfloat16()
        attend_values(cuda_device, cache, table, [1000, 640], q, causal=True, num_splits=splits)
    cache.v.fill_(200.0)
    attend_values(cuda_device, cache, table, [1000, 640], q, causal=True, num_splits=splits)


@pytest.mark.parametrize("exponent", [-120, -110, 100, 115, 118])
@pytest.mark.parametrize("Sq", [1, 6])
@pytest.mark.parametrize("splits", [0, 1, 3])
def test_few_rows_on_value_scales_at_the_ends_of_their_range(cuda_device, Sq, exponent, splits):
    cache, table = cache_of_scales(cuda_device, exponent)
    for q_scale in (0.1, 1.0, 4.0):
        q = (torch.randn(2, Sq, 8, 128, generator=torch.Generator().manual_seed(4)) * q_scale).bfloat16()
        attend_values(cuda_device, cache, table, [1000, 640], q, causal=True, num_splits=splits)
    # blocks of values 2^80 from the others, whose keys weigh as much
    for b in range(2):
        cache.v_scale[table[b, 2:4].long()] = 2.0 ** (exponent + (80 if exponent < 0 else -80))
    attend_values(cuda_device, cache, table, [1000, 640], torch.randn(2, Sq, 8, 128, generator=torch.Generator().manual_seed(5)).bfloat16(), num_splits=splits)


def test_scales_and_soft_caps_at_the_ends_of_fp32(cuda_device):
    """Beyond them refused (a cap that fp32 rounds to 0 would be no cap); inside a cap far from the scores is none, or cuts all of them."""
    cache, table = batch_of(cuda_device, 1, 200)
    lens = torch.tensor([200], dtype=torch.int32, device=cuda_device)
    largest = float(held_of(cache, table[0].tolist(), 200)[1].abs().max())
    for Sq in (1, 40):
        q = torch.randn(1, Sq, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device)
        call = lambda **kw: fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, return_lse=True, **kw)
        for kw in (dict(softcap=1e300), dict(softcap=1e-300), dict(softmax_scale=1e300), dict(softmax_scale=1e-300), dict(softmax_scale=1e-20, softcap=1e20)):
            with pytest.raises(ValueError, match="must be"):
                call(**kw)
        plain, even = call(), call(softmax_scale=1e-30)
        far, near = call(softcap=1e30), call(softcap=1e-30)
        fa.check_status(cuda_device)
        # scores of a few units, 2^-20 of them and the weights' own 2^-8 apart
        assert ((far[1] - plain[1]).abs() <= 2.0 ** -18 * plain[1].abs().clamp(min=1.0)).all()
        assert ((far[0].float() - plain[0].float()).abs() <= 2.0 ** -6 * largest).all()
        # every weight alike
        assert ((near[1] - math.log(200)).abs() <= 2.0 ** -18 * math.log(200)).all() and torch.equal(near[1], even[1])
        assert ((near[0].float() - even[0].float()).abs() <= 2.0 ** -6 * largest).all()


def test_an_expanded_output_is_refused(cuda_device):
    cache, table = batch_of(cuda_device, 2, 100)
    lens = torch.tensor([90, 80], dtype=torch.int32, device=cuda_device)
    for Sq in (2, 40):
        q = torch.zeros(2, Sq, 8, 128, dtype=torch.bfloat16, device=cuda_device)
        for i in range(3):
            shape = [1 if j == i else n for j, n in enumerate(q.shape)]
            with pytest.raises(AssertionError, match="out must not be expanded"):
                fa.flash_attn_fp8_cache_func(q, cache, lens, page_table=table, out=torch.zeros(shape, dtype=q.dtype, device=cuda_device).expand(q.shape))
