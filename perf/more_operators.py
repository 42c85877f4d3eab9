"""Long contexts in the 8-bit KV cache: attention over chosen blocks of it, and the pages it is kept in.  What is timed, on
which inputs, what one pass cannot do without, and the operators in their plain form.

A case is a dict of plain values.  ``op`` names what a pass does:

* ``index``    bounds of the keys of the blocks that new tokens went to;
* ``sparse``   the choice of blocks by those bounds, then attention over the chosen ones;
* ``beam``     one step of a beam search: rows forked, room for a token made, shared pages that are written to copied;
* ``turnover`` sequences that end, begin, grow and lose drafted tokens in one call, and the copies it asks for;
* ``compact``  used pages moved to the front of the pool.

The cache is a pool of pages (``page`` tokens each) of e4m3 values with one fp32 scale for each ``block`` tokens and kv head; it
lies as (page, head, token) where ``by_head``, else as (page, token, head).  Sizes are those of this repository's
configurations and tests, or generic.
"""
import math
import random

import torch

own = False


def listed():
    return [
        # one decode step of a serving batch: the blocks that the new tokens went to
        {"name": "index_step", "op": "index", "B": 64, "S": 1, "held": 8192, "Hkv": 8, "D": 128, "page": 64, "block": 64,
         "ragged": True, "by_head": False},
        # prompts of a document's length that have just been written
        {"name": "index_prompt", "op": "index", "B": 4, "S": 32768, "held": 0, "Hkv": 8, "D": 128, "page": 128, "block": 64,
         "ragged": True, "by_head": True},
        # one token of one sequence: latency is everything
        {"name": "sparse_one", "op": "sparse", "B": 1, "Sq": 1, "Sk": 8192, "Hq": 32, "Hkv": 8, "D": 128, "page": 64, "block": 64,
         "chosen": 16, "rows": 1, "ragged": False, "by_head": True, "sink": False, "softcap": 0.0},
        # one decode step of a serving batch, every sequence with a length of its own
        {"name": "sparse_step", "op": "sparse", "B": 32, "Sq": 1, "Sk": 32768, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "block": 64, "chosen": 32, "rows": 1, "ragged": True, "by_head": True, "sink": False, "softcap": 0.0},
        # drafted tokens to be verified, small blocks, head dim 64, a sink and a soft cap, tokens of a page side by side
        {"name": "sparse_draft", "op": "sparse", "B": 8, "Sq": 5, "Sk": 12289, "Hq": 32, "Hkv": 8, "D": 64, "page": 48, "block": 16,
         "chosen": 67, "rows": 1, "ragged": True, "by_head": False, "sink": True, "softcap": 30.0},
        # a few very long contexts
        {"name": "sparse_long", "op": "sparse", "B": 4, "Sq": 1, "Sk": 262144, "Hq": 64, "Hkv": 8, "D": 128, "page": 128,
         "block": 64, "chosen": 64, "rows": 1, "ragged": False, "by_head": True, "sink": False, "softcap": 0.0},
        # a chunk of a long prompt: every 64 queries choose together
        {"name": "sparse_chunk", "op": "sparse", "B": 1, "Sq": 2048, "Sk": 65536, "Hq": 32, "Hkv": 8, "D": 128, "page": 128,
         "block": 64, "chosen": 64, "rows": 64, "ragged": False, "by_head": True, "sink": False, "softcap": 0.0},
        # one step of a beam search of one request
        {"name": "beam_one", "op": "beam", "B": 4, "beams": 4, "held": 777, "Hkv": 8, "D": 128, "page": 64, "block": 64,
         "spare": 64},
        # the same for a batch of requests
        {"name": "beam_batch", "op": "beam", "B": 128, "beams": 8, "held": 2048, "Hkv": 8, "D": 128, "page": 128, "block": 128,
         "spare": 512},
        # a serving batch between two steps: some sequences end, some begin, some lose their drafted tokens
        {"name": "turnover_batch", "op": "turnover", "B": 256, "beams": 2, "held": 4096, "Hkv": 8, "D": 128, "page": 64,
         "block": 64, "spare": 4096},
        # a pool that is given back: a tenth of it in use, all over the place
        {"name": "compact_small", "op": "compact", "B": 8, "beams": 1, "held": 512, "Hkv": 8, "D": 64, "page": 32, "block": 32,
         "spare": 600},
        # the same with half of a large pool in use
        {"name": "compact_large", "op": "compact", "B": 64, "beams": 1, "held": 8192, "Hkv": 8, "D": 128, "page": 64, "block": 64,
         "spare": 4096},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (16, 16), (8, 1), (12, 4)])
    D = rng.choice([128, 128, 128, 64])
    block = rng.choice([16, 32, 64, 64, 128])
    page = block * rng.choice([1, 1, 2, 3])
    op = rng.choice(["index", "sparse", "sparse", "sparse", "beam", "turnover", "compact"])
    by_head = rng.random() < 0.6
    if op == "index":
        S = rng.choice([1, 1, _log(rng, 2, 32768)])
        return {"op": op, "B": _log(rng, 1, max(1, min(128, 131072 // S))), "S": S, "held": rng.choice([0, _log(rng, 1, 8192)]),
                "Hkv": Hkv, "D": D, "page": page, "block": block, "ragged": rng.random() < 0.5, "by_head": by_head}
    if op == "sparse":
        Sk = _log(rng, 64, 131072)
        rows = rng.choice([1, 1, 1, 16, 64, 100])
        chosen = _log(rng, 3 + 128 // block, 64)
        if rows == 1:
            B, Sq = _log(rng, 1, max(1, min(48, 1048576 // Sk))), min(Sk, rng.choice([1, 1, 1, 2, 4, 7]))
        else:
            B, Sq = rng.choice([1, 1, 2]), min(Sk, _log(rng, 9, 2048))
            chosen = max(chosen, 3 + (rows + block - 2) // block)
        return {"op": op, "B": B, "Sq": Sq, "Sk": Sk, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "block": block,
                "chosen": chosen, "rows": rows, "ragged": rng.random() < 0.5, "by_head": by_head,
                "sink": rng.random() < 0.2, "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}
    beams = 1 if op == "compact" else rng.choice([1, 2, 4, 5])
    held = _log(rng, 1, 8192)
    B = beams * _log(rng, 1, max(1, min(128, 262144 // held) // beams))
    # (room for what begins anew, and for a page more of everybody)
    spare = _log(rng, 8, 2048) + B + (-(-held // page) * (B // 8 + 1) if op == "turnover" else 0)
    return {"op": op, "B": B, "beams": beams, "held": held, "Hkv": Hkv, "D": D, "page": page, "block": block, "spare": spare}


def _key(case):
    return repr(sorted((k, v) for k, v in case.items() if k != "name"))


# ---- inputs -----------------------------------------------------------------------------------------------------

def _lengths(case):
    """(keys or tokens of every sequence, new tokens or queries of every sequence): by the case alone."""
    rng = random.Random(_key(case))
    new = case["S"] if case["op"] == "index" else case["Sq"]
    top = case["held"] if case["op"] == "index" else case["Sk"]
    held, fresh = [], []
    for b in range(case["B"]):
        if case["ragged"] and b > 0:
            n = new if new == 1 else rng.randint(max(1, new // 3), new)
            low = 0 if case["op"] == "index" else max(n, top // 4)
            held.append(rng.randint(min(low, top), top))
            fresh.append(n)
        else:
            held.append(top)
            fresh.append(new)
    return held, fresh


def _cached(case, pages, gen, keys_only=False):
    """A pool as it is met: keys of a block have something in common and a few strong channels, values of unequal blocks.  The scale of a
    block is the smallest power of two that leaves its values at most 448."""
    dev, D, H, size, bt = gen.device, case["D"], case["Hkv"], case["page"], case["block"]
    got = {}
    for name in ("k",) if keys_only else ("k", "v"):
        x = torch.randn(pages, H, size // bt, bt, D, generator=gen, device=dev)
        if name == "k":
            x += torch.randn(pages, H, size // bt, 1, D, generator=gen, device=dev)
            x[..., :: D // 4] *= 3.0
        else:
            x *= 0.25 + torch.rand(pages, H, size // bt, 1, 1, generator=gen, device=dev)
        significand, exponent = torch.frexp(x.abs().amax(dim=(3, 4), keepdim=True))
        scale = torch.ldexp(torch.ones_like(significand), exponent - 9 + (significand > 0.875).int())
        x = (x / scale).to(torch.float8_e4m3fn).view(pages, H, size, D).transpose(1, 2)
        got[name] = x if case.get("by_head") else x.contiguous()
        got[name + "_scale"] = scale.view(pages, H, size // bt).transpose(1, 2).contiguous()
    return got


def _tables(case, seed):
    """Pages as they are in the middle of serving: beams of a request share the pages of its prompt.  (table, refs, held, pages)"""
    rng = random.Random(repr((_key(case), seed)))
    size, B, W = case["page"], case["B"], case["beams"]
    fix = random.Random(_key(case))                   # (what the work goes by is the case's alone)
    held, need = [], 0
    for r in range(B // W):
        n = case["held"] if r == 0 else fix.randint(max(1, case["held"] // 4), case["held"])
        prompt = fix.randint(0, n)
        held += [n] * W
        need += prompt // size + W * (-(-n // size) - prompt // size)
    pages = need + case["spare"]
    width = -(-(case["held"] + 2 * size) // size)
    order = list(range(pages))
    rng.shuffle(order)
    at = iter(order)
    fix = random.Random(_key(case))
    table = []
    for r in range(B // W):
        n = case["held"] if r == 0 else fix.randint(max(1, case["held"] // 4), case["held"])
        prompt = fix.randint(0, n)
        common = [next(at) for _ in range(prompt // size)]
        for _ in range(W):
            row = common + [next(at) for _ in range(-(-n // size) - len(common))]
            table.append(row + [-1] * (width - len(row)))
    refs = [0] * pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    return table, refs, held, pages


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] in ("beam", "turnover", "compact"):
        table, refs, held, pages = _tables(case, seed)
        rng = random.Random(seed)
        B, W, size = case["B"], case["beams"], case["page"]
        # one piece of memory, so that a pass starts from the same with one copy
        book = torch.tensor([p for row in table for p in row] + refs + held, **i32)
        state = {"case": case, "book": book, "shape": (B, len(table[0]), pages), **_cached(case, pages, gen)}
        if case["op"] == "beam":
            state["parents"] = torch.tensor([b // W * W + rng.randrange(W) for b in range(B)], **i32)
        elif case["op"] == "turnover":
            # by turns: grows by one, ends, begins anew as a prompt of other length, loses up to four tokens
            wanted = [n + 1 if b % 8 < 5 else 0 if b % 8 == 5 else rng.randint(1, case["held"]) if b % 8 == 6 else max(0, n - rng.randint(1, 4))
                      for b, n in enumerate(held)]
            state["now"] = torch.tensor([0 if b % 8 == 6 else n for b, n in enumerate(held)], **i32)
            state["wanted"] = torch.tensor(wanted, **i32)
        return state
    held, fresh = _lengths(case)
    index = case["op"] == "index"
    most = max(h + (n if index else 0) for h, n in zip(held, fresh))
    per = -(-most // case["page"])
    pages = case["B"] * per + 3
    state = {"case": case, **_cached(case, pages, gen, keys_only=index)}
    # pages in any order, three that nobody owns
    state["table"] = torch.randperm(pages, generator=gen, device=dev)[: case["B"] * per].view(case["B"], per).to(torch.int32)
    state["fresh"] = torch.tensor(fresh, **i32) if case["ragged"] and max(fresh) > 1 else None
    bounds = (pages, case["page"] // case["block"], case["Hkv"], 2, case["D"])
    state["bounds"] = torch.zeros(bounds, dtype=torch.int8, device=dev)
    state["bound_scale"] = torch.zeros(bounds[:3], device=dev)
    if index:
        state["held"] = torch.tensor(held, **i32)
        state["v"], state["v_scale"] = state["k"], state["k_scale"]        # (an index is one of keys)
        return state
    state["used"] = torch.tensor(held, **i32)
    q = torch.randn(case["B"], case["Sq"], case["Hq"], case["D"], generator=gen, device=dev)
    state["q"] = (q + torch.randn(case["B"], 1, case["Hq"], case["D"], generator=gen, device=dev)).to(torch.bfloat16)
    state["sink"] = torch.randn(case["Hq"], generator=gen, device=dev) if case["sink"] else None
    # rows of padding are nobody's: they come in as zeros and stay so
    state["out"] = torch.zeros(case["B"], case["Sq"], case["Hq"], case["D"], device=dev, dtype=torch.bfloat16)
    state["lse"] = torch.zeros(case["B"], case["Hq"], case["Sq"], device=dev)
    # what a page held before is anything, behind the last token too
    for b, n in enumerate(held):
        flat = torch.arange(n, per * case["page"], device=dev)
        page = state["table"][b].long()[flat // case["page"]]
        for name in ("k", "v"):
            state[name].view(torch.uint8)[page, flat % case["page"]] = 0x7F
    start = torch.zeros_like(state["used"])
    _index(state, case, start, state["used"].long(), max(held))
    return state


# ---- a pass -----------------------------------------------------------------------------------------------------

def _cache(state):
    import flash_attention_b200 as fa
    return fa, fa.FP8KVCache(state["k"], state["v"], state["k_scale"], state["v_scale"], state.get("bounds"), state.get("bound_scale"))


def run(state):
    case = state["case"]
    if case["op"] == "index":
        if own:
            fa, cache = _cache(state)
            fa.index_kv_fp8(cache, state["held"], case["S"], page_table=state["table"], seqused_new=state["fresh"])
        else:
            fresh = state["fresh"].long() if state["fresh"] is not None else torch.full_like(state["held"], case["S"]).long()
            _index(state, case, state["held"], fresh, case["S"])
        return {"bounds": state["bounds"], "scale": state["bound_scale"]}
    if case["op"] == "sparse":
        if own:
            fa, cache = _cache(state)
            blocks = fa.select_kv_blocks(state["q"], cache, state["used"], case["chosen"], page_table=state["table"],
                                         seqused_q=state["fresh"], query_block=case["rows"])
            out, lse = fa.flash_attn_fp8_blocks_func(
                state["q"], cache, blocks, state["used"], page_table=state["table"], seqused_q=state["fresh"],
                query_block=case["rows"], learnable_sink=state["sink"], softcap=case["softcap"], return_lse=True,
                out=state["out"], lse=state["lse"])
        else:
            blocks = _select(state, case)
            out, lse = _attend(state, case, blocks)
        return {"blocks": blocks, "out": out, "lse": lse}
    # (the pages are changed in place: a pass works on a copy)
    B, width, pages = state["shape"]
    book = state["book"].clone()
    table, refs, held = book[: B * width].view(B, width), book[B * width: B * width + pages], book[B * width + pages:]
    size = case["page"]
    if own:
        fa, cache = _cache(state)
        kept = fa.KVPages(table, refs, size)
    if case["op"] == "beam":
        if own:
            kept, held = fa.fork_kv_pages(kept, held, state["parents"])
            pairs = fa.resize_kv_pages(kept, held, held + 1)
            table = kept.table
        else:
            table, held = _fork(table, refs, held, state["parents"].long(), size)
            table, pairs = _resize(table, refs, held.long(), held.long() + 1, size)
    elif case["op"] == "turnover":
        if own:
            pairs = fa.resize_kv_pages(kept, state["now"], state["wanted"])
        else:
            table, pairs = _resize(table, refs, state["now"].long(), state["wanted"].long(), size)
    else:
        if own:
            pairs, used = fa.compact_kv_pages(kept)
        else:
            table, refs, pairs, used = _compact(table, refs)
    if own:
        fa.copy_kv_pages(cache, pairs)
    else:
        _copy(state, pairs)
    got = {"table": table, "refs": refs, "pairs": pairs, "k": state["k"], "v": state["v"], "k_scale": state["k_scale"],
           "v_scale": state["v_scale"]}
    return {**got, "used": used} if case["op"] == "compact" else {**got, "held": held}


# ---- the plain forms ------------------------------------------------------------------------------------------

def _index(state, case, held, fresh, most):
    """The bounds of all blocks that tokens held .. held + fresh - 1 (at most `most`) lie in, over the tokens that are there then."""
    bt, size, H, D = case["block"], case["page"], case["Hkv"], case["D"]
    held = held.long()
    B, per = state["table"].shape
    n = min((most + bt - 2) // bt + 1, per * size // bt)
    blk = (held // bt)[:, None] + torch.arange(n, device=held.device)
    used = (blk * bt < (held + fresh)[:, None]) & (fresh > 0)[:, None] & (blk < per * size // bt)
    seq, at = used.nonzero(as_tuple=True)
    for piece in torch.arange(len(seq), device=seq.device).split(16384):
        b, j = seq[piece], blk[seq[piece], at[piece]]
        page, in_page = state["table"].long()[b, j * bt // size], j % (size // bt)
        tok = in_page[:, None] * bt + torch.arange(bt, device=held.device)
        x = state["k"].view(torch.uint8)[page[:, None], tok].view(torch.float8_e4m3fn).float()          # (blocks, bt, H, D)
        there = (j[:, None] * bt + torch.arange(bt, device=held.device) < (held + fresh)[b][:, None])[:, :, None, None]
        bad = (x.isnan() & there).any(dim=3).any(dim=1)
        hi, lo = torch.where(there, x, -math.inf).amax(1), torch.where(there, x, math.inf).amin(1)          # (blocks, H, D)
        top = torch.maximum(hi.abs(), lo.abs()).amax(-1)
        unit = torch.where(top > 0, torch.frexp(torch.where(top > 0, top, 1.0))[1] - 7, -15)
        step = torch.ldexp(torch.ones_like(top), unit)
        hi, lo = torch.ceil(hi / step[..., None]), torch.floor(lo / step[..., None])
        both = torch.where(bad[..., None, None], 0.0, torch.stack([hi, lo], dim=2)).to(torch.int8)
        state["bounds"][page, in_page] = both
        state["bound_scale"][page, in_page] = torch.where(bad, math.nan, state["k_scale"][page, in_page] * step)


def _places(state, case):
    """Of every sequence and query block: its rows, the first one's position, the end of what its last row sees."""
    used = state["used"].long()
    fresh = state["fresh"].long() if state["fresh"] is not None else torch.full_like(used, case["Sq"])
    q0 = torch.arange(0, case["Sq"], case["rows"], device=used.device)
    rows = (fresh[:, None] - q0).clamp(0, case["rows"])
    first = (used - fresh)[:, None] + q0
    end = torch.where(rows > 0, torch.minimum((first + rows).clamp(min=0), used[:, None]), 0)
    return rows, first, end


def _grouped(state, case):
    """Queries as (B, query blocks, H, rows of the block, group, D), rows that are not there as zeros."""
    q, Q = state["q"], case["rows"]
    B, Sq, G, D = q.shape
    n = -(-Sq // Q)
    x = torch.zeros(B, n * Q, G, D, device=q.device)
    x[:, :Sq] = q.float()
    x = x.view(B, n, Q, case["Hkv"], G // case["Hkv"], D).permute(0, 1, 3, 2, 4, 5)
    there = torch.arange(Q, device=q.device) < _places(state, case)[0][..., None]
    return torch.where(there[:, :, None, :, None, None], x, 0.0), there


def _select(state, case):
    bt, size, D, K = case["block"], case["page"], case["D"], case["chosen"]
    x = _grouped(state, case)[0].flatten(3, 4).double()                              # (B, n, H, rows, D)
    x = torch.where(x.isfinite(), x, 0.0)
    exponent = (torch.frexp(x.abs().amax(dim=(3, 4)))[1] - 1).clamp(min=-100)
    x = torch.round(torch.ldexp(x, 14 - exponent[..., None, None]))
    part = torch.stack([x.clamp(min=0).sum(3), (-x).clamp(min=0).sum(3)], dim=3)           # (B, n, H, 2, D), whole numbers
    shift = (torch.frexp(part.amax(dim=(3, 4)))[1] - 7).clamp(min=0)[..., None, None]
    half = torch.floor(torch.ldexp(torch.ones_like(part), shift - 1))
    part = torch.floor(torch.ldexp(part + half, -shift)).clamp(max=127)
    part[..., 1, :] *= -1
    table = state["table"].long()
    bounds = state["bounds"][table].flatten(1, 2).permute(0, 2, 3, 4, 1)                  # (B, H, 2, D, blocks)
    scale = state["bound_scale"][table].flatten(1, 2).permute(0, 2, 1)                    # (B, H, blocks)
    # (sums of whole numbers below 2^24: exact in fp32)
    score = part.flatten(3, 4).float().transpose(1, 2) @ bounds.flatten(2, 3).float()     # (B, H, n, blocks)
    score = (score * scale[:, :, None]).transpose(1, 2)                                   # (B, n, H, blocks)
    score = torch.where(score.isnan(), math.inf, score)
    rows, first, end = _places(state, case)
    j = torch.arange(score.shape[-1], device=score.device)
    seen = j * bt < end[..., None]
    always = seen & ((j < 1) | (j >= (first.clamp(min=0) // bt)[..., None]))
    rank = torch.where(always, 0, torch.where(seen, 1, 2))[:, :, None].expand_as(score)
    order = torch.argsort(score, dim=-1, descending=True, stable=True)
    order = order.gather(-1, torch.argsort(rank.gather(-1, order), dim=-1, stable=True))[..., :K]
    none = len(j)
    blocks = torch.where(rank.gather(-1, order) < 2, order, none).sort(dim=-1)[0]
    blocks = torch.where(blocks < none, blocks, -1).to(torch.int32)
    return torch.nn.functional.pad(blocks, (0, K - blocks.shape[-1]), value=-1)


def _attend(state, case, blocks):
    bt, size, D, Sq, Q, H = case["block"], case["page"], case["D"], case["Sq"], case["rows"], case["Hkv"]
    q, there = _grouped(state, case)
    B, n, _, _, group, _ = q.shape
    dev = q.device
    key = (blocks.long()[..., None] * bt + torch.arange(bt, device=dev)).flatten(3)          # (B, n, H, keys)
    key = torch.where(blocks.repeat_interleave(bt, dim=-1) >= 0, key, 1 << 40)
    rows, first, end = _places(state, case)
    row_end = torch.minimum((first[..., None] + 1 + torch.arange(Q, device=dev)).clamp(min=0), state["used"].long()[:, None, None])
    see = key[:, :, :, None] < row_end[:, :, None, :, None]                                    # (B, n, H, rows, keys)
    read = torch.where(key < end[:, :, None, None], key, 0)
    page = state["table"].long()[torch.arange(B, device=dev)[:, None, None, None], read // size]
    head = torch.arange(H, device=dev)[:, None]

    def gathered(name):
        x = state[name].view(torch.uint8)[page, read % size, head].view(torch.float8_e4m3fn).float()
        return x * state[name + "_scale"][page, read % size // bt, head][..., None]

    s = q.flatten(3, 4) @ gathered("k").transpose(-1, -2)                                       # (B, n, H, rows x group, keys)
    s = s.view(B, n, H, Q, group, -1) * (1.0 / math.sqrt(D))
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    s = s.masked_fill(~see[:, :, :, :, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    sink = state["sink"].view(1, 1, H, 1, group, 1) if state["sink"] is not None else None
    if sink is not None:
        top = torch.maximum(top, sink)
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.exp(sink - top)
    v = torch.where((key < end[:, :, None, None])[..., None], gathered("v"), 0.0)
    o = (p.flatten(3, 4) @ v).view(B, n, H, Q, group, D) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)                                                   # (B, n, H, rows, group)
    o = o.permute(0, 1, 3, 2, 4, 5).reshape(B, n * Q, H * group, D)[:, :Sq].to(torch.bfloat16)
    lse = lse.permute(0, 2, 4, 1, 3).reshape(B, H * group, n * Q)[..., :Sq]
    there = there.view(B, n * Q)[:, :Sq]
    return torch.where(there[..., None, None], o, state["out"]), torch.where(there[:, None], lse, state["lse"])


def _fork(table, refs, held, parents, size):
    """Row b of the new table is row parents[b] of the old one as far as it holds tokens."""
    width, dev = table.shape[1], table.device
    children = torch.zeros_like(held).index_add_(0, parents, torch.ones_like(held))
    kept = torch.arange(width, device=dev) < (-(-held.long() // size))[:, None]
    change = torch.where(kept, children[:, None] - 1, -1) * (table >= 0)
    refs.index_add_(0, table.clamp(min=0).flatten().long(), change.flatten().to(refs.dtype))
    return torch.where(kept, table, -1)[parents], held[parents]


def _resize(table, refs, held, wanted, size):
    """Every row keeps the pages of what it holds, gives back those behind, and gets pages for `wanted` tokens; where it is about to write
    into a page that others name too it gets a copy: (table, pairs of pages to copy)."""
    B, width = table.shape
    dev, table = table.device, table.long()
    j = torch.arange(width, device=dev)
    keep = -(-wanted // size)
    drop = (table >= 0) & (j >= (-(-torch.minimum(held, wanted) // size))[:, None])
    refs.index_add_(0, table.clamp(min=0).flatten(), -drop.flatten().to(refs.dtype))
    table = torch.where(drop, -1, table)
    at = (held // size).clamp(max=width - 1)
    page = table.gather(1, at[:, None])[:, 0]
    writes = (wanted > held) & (held % size != 0) & (page >= 0)
    page = torch.where(writes, page, -1)
    earlier = ((page[:, None] == page) & writes[:, None]).tril(-1).sum(1)
    copies = writes & (earlier < refs[page.clamp(min=0)] - 1)
    refs.index_add_(0, page.clamp(min=0), -copies.to(refs.dtype))
    lacks = (table < 0) & (j < keep[:, None])
    lacks.scatter_(1, at[:, None], lacks.gather(1, at[:, None]) | copies[:, None])
    # free pages, the lowest first, to entries in order
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1
    pages = torch.full((len(refs) + 1,), -1, dtype=torch.long, device=dev)
    pages.scatter_(0, torch.where(free, rank, len(refs)), torch.where(free, torch.arange(len(refs), device=dev), -1))
    order = (torch.cumsum(lacks.flatten(), 0) - 1).view(B, width).clamp(0, len(refs))
    given = torch.where(lacks, pages[order], -1)
    refs.index_add_(0, given.clamp(min=0).flatten(), (given >= 0).flatten().to(refs.dtype))
    table = torch.where(lacks, given, table)
    new = table.gather(1, at[:, None])[:, 0]
    done = copies & (new >= 0)
    pairs = torch.stack([torch.where(done, page, -1), torch.where(done, new, -1)], dim=1)
    return table.to(torch.int32), pairs.to(torch.int32)


def _compact(table, refs):
    """(table, refs, pairs of pages to copy, pages in use)"""
    n, dev = len(refs), refs.device
    live = refs > 0
    used = live.sum()
    i = torch.arange(n, device=dev)
    hole, mover = ~live & (i < used), live & (i >= used)
    pairs = torch.full((n // 2 + 1, 2), -1, dtype=torch.long, device=dev)
    for column, which in ((0, mover), (1, hole)):
        pairs[:, column].scatter_(0, torch.where(which, torch.cumsum(which, 0) - 1, n // 2), torch.where(which, i, -1))
    pairs = pairs[: n // 2]
    to = i.scatter(0, torch.where(mover, i, 0), torch.where(mover, pairs[(torch.cumsum(mover, 0) - 1).clamp(0, n // 2 - 1), 1], 0)) if n > 1 else i
    to = torch.where(mover, to, i)
    table = torch.where(table >= 0, to[table.clamp(min=0).long()], -1).to(torch.int32)
    moved = torch.zeros_like(refs).index_add_(0, to, refs)
    return table, moved, pairs.to(torch.int32), used.to(torch.int32).view(1)


def _copy(state, pairs):
    pairs = pairs.long()[pairs[:, 0] >= 0]
    for name in ("k", "v", "k_scale", "v_scale"):
        x = state[name].view(torch.uint8) if name in ("k", "v") else state[name]
        x[pairs[:, 1]] = x[pairs[:, 0]]


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    bt, size, D, H = case["block"], case["page"], case["D"], case["Hkv"]
    if case["op"] == "index":
        blocks = tokens = 0
        for h, n in zip(*_lengths(case)):
            blocks += (h + n - 1) // bt - h // bt + 1
            tokens += h + n - h // bt * bt
        return {"bytes": H * (tokens * D + blocks * (2 * D + 8)), "flops": 2 * tokens * H * D}
    if case["op"] == "sparse":
        G, read, flops = case["Hq"], 0, 0
        for n, rows in zip(*_lengths(case)):
            read += -(-n // bt) * H * (2 * D + 4) + rows * G * (4 * D + 4)
            keys = 0
            for r0 in range(0, rows, case["rows"]):
                q = min(case["rows"], rows - r0)
                end = n - rows + r0 + q
                flops += 4 * D * H * -(-end // bt)
                if end > case["chosen"] * bt:
                    here = case["chosen"] * bt - (-end % bt)
                    flops += 4 * D * G * (q * here - q * (q - 1) // 2)
                else:
                    here = end
                    flops += 4 * D * G * (q * end - q * (q - 1) // 2)
                keys += here
            # (query blocks may choose the same: no more than there is, no less than one chooses)
            read += min(n, keys) * H * 2 * D
        return {"bytes": read, "flops": flops}
    table, refs, held, pages = _tables(case, 0)
    B, width = len(table), len(table[0])
    page_bytes = 2 * size * H * D + 2 * size // bt * H * 4
    books = 4 * (2 * B * width + 2 * pages)
    if case["op"] == "compact":
        # (pages in use lie anywhere: half of those beyond the front, on average)
        used = sum(r > 0 for r in refs)
        moved = used * (pages - used) / pages
    elif case["op"] == "beam":
        # (of the beams that write into a page with others, all but one; parents are drawn evenly)
        W = case["beams"]
        moved = sum(1 for h in held if h % size) * max(0.0, 1 - (1 - (1 - 1 / W) ** W))
    else:
        moved = 0
    return {"bytes": books + 2 * moved * page_bytes, "flops": 0}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] not in ("index", "sparse"):
        return None                                    # (numbers of pages, and bytes that are moved)
    state = prepare(case, seed)
    held, fresh = _lengths(case)
    bt, size, D, H = case["block"], case["page"], case["D"], case["Hkv"]
    table = state["table"].long()
    per = size // bt
    if case["op"] == "index":
        scale = state["bound_scale"].double().clone()
        for b in range(case["B"]):
            j0, end = held[b] // bt, held[b] + fresh[b]
            j1 = (end - 1) // bt + 1
            j = torch.arange(j0, j1, device=table.device)
            page, at = table[b][j // per], j % per
            x = state["k"].view(torch.uint8)[page[:, None], at[:, None] * bt + torch.arange(bt, device=table.device)]
            x = x.view(torch.float8_e4m3fn).double().abs()
            x[(j[:, None] * bt + torch.arange(bt, device=table.device)) >= end] = 0
            top = x.amax(dim=(1, 3))
            scale[page, at] = state["k_scale"][page, at].double() * torch.where(top > 0, torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -9))) - 6), 2.0 ** -15)
        return {"bounds": None, "scale": scale}
    Sq, Q, G, K = case["Sq"], case["rows"], case["Hq"], case["chosen"]
    if case["B"] * -(-Sq // Q) * H > 1200:
        return None
    out, lse = state["out"].double(), state["lse"].double()
    for b in range(case["B"]):
        n, rows = held[b], fresh[b]
        j = torch.arange(-(-n // bt), device=out.device)
        page, at = table[b][j // per], j % per
        bounds, scales = state["bounds"][page, at].double(), state["bound_scale"][page, at]                  # (blocks, H, 2, D), (blocks, H)
        for r0 in range(0, rows, Q):
            r1 = min(rows, r0 + Q)
            first, end = n - rows + r0, n - rows + r1
            blocks = -(-end // bt)
            for h in range(H):
                g = slice(h * (G // H), (h + 1) * (G // H))
                q = state["q"][b, r0:r1, g].double()
                # which blocks
                exponent = max(-100, math.frexp(q.abs().max().item())[1] - 1) if q.abs().max() > 0 else -100
                whole = torch.round(q * 2.0 ** (14 - exponent)).long()
                up, down = whole.clamp(min=0).sum(dim=(0, 1)), (-whole).clamp(min=0).sum(dim=(0, 1))
                most = max(up.max().item(), down.max().item())
                s = max(0, most.bit_length() - 7)
                half = 1 << s >> 1
                up, down = ((up + half) >> s).clamp(max=127).double(), ((down + half) >> s).clamp(max=127).double()
                dot = bounds[:blocks, h, 0] @ up - bounds[:blocks, h, 1] @ down
                score = (dot.float() * scales[:blocks, h]).tolist()
                score = [math.inf if x != x else x for x in score]
                must = [i for i in range(blocks) if i == 0 or i >= first // bt]
                rest = sorted((i for i in range(1, min(blocks, first // bt))), key=lambda i: (-score[i], i))
                mine = sorted(must + rest[: max(0, K - len(must))])
                # attention over them
                key = (torch.tensor(mine, device=out.device)[:, None] * bt + torch.arange(bt, device=out.device)).flatten()
                key = key[key < end]
                pg = table[b][key // size]

                def values(name):
                    x = state[name].view(torch.uint8)[pg, key % size, h].view(torch.float8_e4m3fn).double()
                    return x * state[name + "_scale"][pg, key % size // bt, h].double()[:, None]

                x = torch.einsum("rgd,kd->rgk", q, values("k")) / math.sqrt(D)
                if case["softcap"]:
                    x = case["softcap"] * torch.tanh(x / case["softcap"])
                place = torch.arange(first, end, device=out.device)
                x = x.masked_fill((key > place[:, None])[:, None], -math.inf)
                if case["sink"]:
                    x = torch.cat([x, state["sink"][g].double()[None, :, None].expand(r1 - r0, -1, 1)], dim=2)
                total = torch.logsumexp(x, dim=2)
                weight = torch.exp(x - total[..., None])[..., : len(key)]
                out[b, r0:r1, g] = torch.einsum("rgk,kd->rgd", weight, values("v"))
                lse[b, g, r0:r1] = total.T
    return {"blocks": None, "out": out, "lse": lse}
