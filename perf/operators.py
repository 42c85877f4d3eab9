"""The 8-bit KV cache of a serving loop: appending keys and values to it, and attention over it.  What is timed, on which
inputs, what one pass cannot do without, and the operators in their plain form.

A case is a dict of plain values.  ``op`` names the operator:

* ``append``  keys and values of new tokens into the cache, keys and queries rotated on the way;
* ``attend``  queries of the last tokens of every sequence against the cache.

The cache is a pool of pages (``page`` tokens each, found through a page table), or contiguous (``page`` 0).  It holds e4m3
values and one fp32 scale for each ``block`` tokens and kv head.  Sizes are those of this repository's configurations and
tests, or generic.
"""
import math
import random

import torch

own = False


def listed():
    return [
        # one token of one sequence: latency is everything
        {"name": "append_one", "op": "append", "B": 1, "S": 1, "held": 776, "Hq": 32, "Hkv": 8, "D": 128, "page": 0,
         "block": 64, "ragged": False, "rotary": 128, "interleaved": False},
        # one decode step of a serving batch, every sequence at a place of its own
        {"name": "append_step", "op": "append", "B": 64, "S": 1, "held": 4096, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "block": 64, "ragged": True, "rotary": 128, "interleaved": False},
        # a padded batch of prompt pieces of odd lengths behind what the cache holds, half of the head rotated
        {"name": "append_ragged", "op": "append", "B": 6, "S": 777, "held": 333, "Hq": 16, "Hkv": 4, "D": 64, "page": 16,
         "block": 16, "ragged": True, "rotary": 32, "interleaved": True},
        # a whole prompt: the largest append
        {"name": "append_prompt", "op": "append", "B": 2, "S": 8192, "held": 0, "Hq": 32, "Hkv": 8, "D": 128, "page": 128,
         "block": 128, "ragged": False, "rotary": 128, "interleaved": False},
        # one token of one sequence against a short context: latency is everything
        {"name": "attend_one", "op": "attend", "B": 1, "Sq": 1, "Sk": 777, "Hq": 32, "Hkv": 8, "D": 128, "page": 0,
         "block": 64, "ragged": False, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
        # one decode step of a serving batch: every sequence with a length of its own, small pages
        {"name": "attend_step", "op": "attend", "B": 32, "Sq": 1, "Sk": 8192, "Hq": 32, "Hkv": 8, "D": 128, "page": 64,
         "block": 64, "ragged": True, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
        # a few long contexts
        {"name": "attend_long", "op": "attend", "B": 4, "Sq": 1, "Sk": 65536, "Hq": 64, "Hkv": 8, "D": 128, "page": 128,
         "block": 128, "ragged": False, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
        # drafted tokens to be verified, the smallest pages
        {"name": "attend_draft", "op": "attend", "B": 8, "Sq": 5, "Sk": 4099, "Hq": 32, "Hkv": 8, "D": 128, "page": 16,
         "block": 16, "ragged": True, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
        # a sliding-window layer with sinks, head dim 64, a step of drafted tokens
        {"name": "attend_window_d64", "op": "attend", "B": 16, "Sq": 2, "Sk": 4096, "Hq": 64, "Hkv": 8, "D": 64, "page": 32,
         "block": 32, "ragged": True, "causal": True, "window": 1023, "sink": True, "softcap": 0.0},
        # pieces of prompts of unequal lengths, with a soft cap
        {"name": "attend_pieces", "op": "attend", "B": 3, "Sq": 333, "Sk": 2048, "Hq": 16, "Hkv": 4, "D": 128, "page": 64,
         "block": 64, "ragged": True, "causal": True, "window": -1, "sink": False, "softcap": 30.0},
        # a chunk of a long prompt against what the cache holds so far
        {"name": "attend_chunk", "op": "attend", "B": 1, "Sq": 1024, "Sk": 16384, "Hq": 32, "Hkv": 8, "D": 128, "page": 128,
         "block": 128, "ragged": False, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
        # a whole prompt: the largest call
        {"name": "attend_prompt", "op": "attend", "B": 1, "Sq": 8192, "Sk": 8192, "Hq": 64, "Hkv": 8, "D": 128, "page": 128,
         "block": 128, "ragged": False, "causal": True, "window": -1, "sink": False, "softcap": 0.0},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 4), (16, 16), (8, 1), (12, 4)])
    D = rng.choice([128, 128, 128, 64])
    block = rng.choice([16, 32, 64, 128])
    page = rng.choice([0, block, block, 2 * block, 3 * block])
    if rng.random() < 0.35:
        S = rng.choice([1, 1, 1, _log(rng, 2, 8192)])
        B = _log(rng, 1, max(1, min(128, 16384 // S)))
        rotary = rng.choice([0, D, D, D // 2])
        return {"op": "append", "B": B, "S": S, "held": rng.choice([0, _log(rng, 1, 8192)]), "Hq": Hq, "Hkv": Hkv, "D": D,
                "page": page, "block": block, "ragged": rng.random() < 0.5, "rotary": rotary,
                "interleaved": rng.random() < 0.5}
    Sk = _log(rng, 64, 65536)
    few = rng.random() < 0.6
    B = _log(rng, 1, max(1, min(64, (262144 if few else 16384) // Sk)))
    Sq = rng.choice([1, 1, 1, 2, 4, 7]) if few else _log(rng, 9, max(9, min(Sk, 2_000_000_000 // (Sk * B * Hq))))
    Sq = min(Sq, Sk)
    return {"op": "attend", "B": B, "Sq": Sq, "Sk": Sk, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "block": block,
            "ragged": rng.random() < 0.5, "causal": Sq == 1 or rng.random() < 0.85,
            "window": rng.choice([-1, -1, -1, _log(rng, 16, Sk)]), "sink": rng.random() < 0.2,
            "softcap": rng.choice([0.0, 0.0, 0.0, 30.0])}


def _lengths(case):
    """(keys or tokens of every sequence, new tokens or queries of every sequence): by the case alone."""
    rng = random.Random(_key(case))
    new = case["S"] if case["op"] == "append" else case["Sq"]
    top = case["held"] if case["op"] == "append" else case["Sk"]
    held, fresh = [], []
    for b in range(case["B"]):
        if case["ragged"]:
            n = new if new == 1 or b == 0 else rng.randint(max(1, new // 3), new)
            low = 0 if case["op"] == "append" else max(n, top // 16)
            held.append(top if b == 0 else rng.randint(min(low, top), top))
            fresh.append(n)
        else:
            held.append(top)
            fresh.append(new)
    return held, fresh


def _key(case):
    return repr(sorted((k, v) for k, v in case.items() if k != "name"))


def _pool(case, tokens):
    """(pages, tokens of a page, pages of a sequence) of the cache; a contiguous one has a page for every sequence."""
    if case["page"] == 0:
        size = -(-tokens // case["block"]) * case["block"]
        return case["B"], size, 1
    per = -(-tokens // case["page"])
    return case["B"] * per + 3, case["page"], per


def _cached(case, pages, size, gen):
    """A cache as it is met: normal keys with a few strong channels, values of unequal blocks; scales maximum / 448."""
    dev, D, H = gen.device, case["D"], case["Hkv"]
    got = []
    for strong in (True, False):
        x = torch.randn(pages, size, H, D, generator=gen, device=dev)
        if strong:
            x[..., :: D // 4] *= 4.0
        x = x.view(pages, size // case["block"], case["block"], H, D)
        if not strong:
            x *= 0.25 + torch.rand(pages, size // case["block"], 1, H, 1, generator=gen, device=dev)
        scale = x.abs().amax(dim=(2, 4)) / torch.full((), 448.0, device=dev)
        x = (x / scale[:, :, None, :, None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
        got += [x.view(pages, size, H, D), scale.contiguous()]
    return got


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    held, fresh = _lengths(case)
    append = case["op"] == "append"
    pages, size, per = _pool(case, max(h + (n if append else 0) for h, n in zip(held, fresh)))
    k, k_scale, v, v_scale = _cached(case, pages, size, gen)
    state = {"case": case, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "table": None}
    if case["page"]:
        # pages in any order, three that nobody owns
        order = torch.randperm(pages, generator=gen, device=dev)[: case["B"] * per]
        state["table"] = order.view(case["B"], per).to(torch.int32)
    B, H, G, D = case["B"], case["Hkv"], case["Hq"], case["D"]
    i32 = dict(dtype=torch.int32, device=dev)
    if append:
        S = case["S"]
        state["held"] = torch.tensor(held, **i32)
        state["fresh"] = torch.tensor(fresh, **i32) if case["ragged"] else None
        # what a projection leaves: q, k and v of a token side by side
        qkv = torch.randn(B, S, G + 2 * H, D, generator=gen, device=dev, dtype=torch.bfloat16)
        state["q"], state["k_new"], state["v_new"] = qkv[:, :, :G], qkv[:, :, G:G + H], qkv[:, :, G + H:]
        state["cos"] = state["sin"] = None
        if case["rotary"]:
            half = case["rotary"] // 2
            freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
            angle = torch.arange(max(held) + S, device=dev, dtype=torch.float64)[:, None] * freq
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
    else:
        state["used"] = torch.tensor(held, **i32)
        state["fresh"] = torch.tensor(fresh, **i32) if case["ragged"] and case["Sq"] > 1 else None
        state["q"] = torch.randn(B, case["Sq"], G, D, generator=gen, device=dev, dtype=torch.bfloat16)
        state["sink"] = torch.randn(G, generator=gen, device=dev) if case["sink"] else None
        # rows of padding are nobody's: they come in as zeros and stay so
        state["out"] = torch.zeros(B, case["Sq"], G, D, device=dev, dtype=torch.bfloat16)
        state["lse"] = torch.zeros(B, G, case["Sq"], device=dev)
        # what a page held before is anything, behind the last token too
        for b, n in enumerate(held):
            flat = torch.arange(n, per * size, device=dev)
            page = state["table"][b].long()[flat // size] if case["page"] else torch.full_like(flat, b)
            for name in ("k", "v"):
                state[name].view(torch.uint8)[page, flat % size] = 0x7F
    return state


def run(state):
    case = state["case"]
    if own:
        import flash_attention_b200 as fa
        cache = fa.FP8KVCache(state["k"], state["v"], state["k_scale"], state["v_scale"])
    if case["op"] == "append":
        if own:
            q = fa.append_kv_fp8(cache, state["k_new"], state["v_new"], state["held"],
                                 page_table=state["table"], seqused_new=state["fresh"],
                                 rotary_cos=state["cos"], rotary_sin=state["sin"],
                                 rotary_interleaved=case["interleaved"],
                                 q=state["q"] if case["rotary"] else None)
        else:
            q = _append(state, case)
        got = {"k": state["k"], "v": state["v"], "k_scale": state["k_scale"], "v_scale": state["v_scale"]}
        return {**got, "q": q} if case["rotary"] else got
    if own:
        out, lse = fa.flash_attn_fp8_cache_func(
            state["q"], cache, seqused_k=state["used"], page_table=state["table"], seqused_q=state["fresh"],
            causal=case["causal"], window_size=(case["window"] if case["window"] >= 0 else None, None),
            learnable_sink=state["sink"], softcap=case["softcap"], return_lse=True, out=state["out"], lse=state["lse"])
        return {"out": out, "lse": lse}
    return _attend(state, case)


# ---- the plain forms ------------------------------------------------------------------------------------------

def _rotate(x, cos, sin, interleaved):
    """x (B, S, H, D) in fp32, cos and sin (B, S, rotary / 2)."""
    half = cos.shape[-1]
    c, s = cos[:, :, None], sin[:, :, None]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([y, x[..., 2 * half:]], dim=-1)


def _append(state, case):
    k, v, q = state["k_new"].float(), state["v_new"].float(), None
    B, S, H, D = k.shape
    dev, bt, size = k.device, case["block"], state["k"].shape[1]
    held = state["held"].long()
    fresh = state["fresh"].long() if state["fresh"] is not None else torch.full_like(held, S)
    if case["rotary"]:
        at = (held[:, None] + torch.arange(S, device=dev)).clamp(max=state["cos"].shape[0] - 1)
        cos, sin = state["cos"][at], state["sin"][at]
        k = _rotate(k, cos, sin, case["interleaved"])
        q = _rotate(state["q"].float(), cos, sin, case["interleaved"]).to(torch.bfloat16)
    # the blocks that get tokens, whole: those of sequence b start at its first one
    blocks = (S + bt - 2) // bt + 1
    first = held // bt
    tok = first[:, None] * bt + torch.arange(blocks * bt, device=dev)              # places in the sequence
    new = (tok >= held[:, None]) & (tok < (held + fresh)[:, None])
    old = (tok < held[:, None])
    src = (tok - held[:, None]).clamp(0, S - 1)
    touched = new.view(B, blocks, bt).any(-1)
    if state["table"] is not None:
        page = state["table"].long().gather(1, (tok // size).clamp(max=state["table"].shape[1] - 1))
    else:
        page = torch.arange(B, device=dev)[:, None].expand_as(tok)
    rows = (page * size + tok % size).clamp(max=state["k"].shape[0] * size - 1).view(B, blocks, bt)
    seq, blk = touched.nonzero(as_tuple=True)
    rows, old, new = rows[seq, blk], old.view(B, blocks, bt)[seq, blk], new.view(B, blocks, bt)[seq, blk]
    src = src.view(B, blocks, bt)[seq, blk]
    for name, x in (("k", k), ("v", v)):
        values, scales = state[name].view(torch.uint8).view(-1, H, D), state[name + "_scale"].view(-1, H)
        x = x[seq[:, None], src]                                                    # (n, bt, H, D)
        fine = x.isfinite() & new[:, :, None, None]
        top = torch.where(fine, x.abs(), 0.0).amax(dim=(1, 3))
        significand, exponent = torch.frexp(top)                                     # top = significand 2^exponent
        exponent = (exponent - 9 + (significand > 0.875).int()).clamp(-120, 120)     # 448 = .875 2^9
        need = torch.where(top > 0, torch.ldexp(torch.ones_like(top), exponent), 2.0 ** -120)
        before = scales[rows[:, 0] // bt]
        kept = old.any(1)[:, None]
        scale = torch.where(kept, torch.maximum(before, need), need)
        was = values[rows].view(torch.float8_e4m3fn).float()
        again = torch.where(kept, before / scale, 1.0)[:, None, :, None]
        y = torch.where(fine, x / scale[:, None, :, None], math.nan).clamp(-448.0, 448.0)
        y = torch.where(new[:, :, None, None], y, torch.where(old[:, :, None, None], was * again, was))
        values[rows] = y.to(torch.float8_e4m3fn).view(torch.uint8)
        scales[rows[:, 0] // bt] = scale
    return q


def _attend(state, case):
    q, used = state["q"].float(), state["used"].long()
    B, Sq, G, D = q.shape
    H, bt, dev = case["Hkv"], case["block"], q.device

    def gathered(values, scales):
        x = values.float().view(values.shape[0], -1, bt, H, D) * scales[:, :, None, :, None]
        x = x.view(values.shape)
        x = x[state["table"].long()].flatten(1, 2) if state["table"] is not None else x
        return x[:, :case["Sk"]].permute(0, 2, 1, 3)                                 # (B, H, Sk, D)

    k, v = gathered(state["k"], state["k_scale"]), gathered(state["v"], state["v_scale"])
    j = torch.arange(k.shape[2], device=dev)
    live = j < used[:, None]                                                         # (B, Sk)
    v = torch.where(live[:, None, :, None], v, 0.0)
    s = q.view(B, Sq, H, G // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, -1, D) @ k.transpose(2, 3)
    s = s.view(B, G, Sq, -1) * (1.0 / math.sqrt(D))
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    fresh = state["fresh"].long() if state["fresh"] is not None else torch.full_like(used, Sq)
    row = torch.arange(Sq, device=dev)
    end = used[:, None] - fresh[:, None] + row                                       # a query's own place
    see = live[:, None].expand(B, Sq, -1)
    if case["causal"]:
        see = see & (j <= end[:, :, None])
    if case["window"] >= 0:
        see = see & (j >= end[:, :, None] - case["window"])
    s = s.masked_fill(~see[:, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    if state["sink"] is not None:
        top = torch.maximum(top, state["sink"].view(1, G, 1, 1))
    top = torch.where(top > -math.inf, top, 0.0)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    if state["sink"] is not None:
        total = total + torch.exp(state["sink"].view(1, G, 1, 1) - top)
    o = (p.view(B, H, -1, p.shape[-1]) @ v).view(B, G, Sq, D) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    there = row < fresh[:, None]                                                     # (B, Sq)
    out = torch.where(there[:, :, None, None], o.permute(0, 2, 1, 3).to(torch.bfloat16), state["out"])
    return {"out": out, "lse": torch.where(there[:, None], lse, state["lse"])}


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def _pairs(case):
    """(row, key) pairs that are seen, and keys that some row sees, over the batch, for one query head."""
    held, fresh = _lengths(case)
    pairs = keys = 0
    for n, rows in zip(held, fresh):
        low = n
        for i in range(rows):
            at = n - rows + i
            hi = min(n, at + 1) if case["causal"] else n
            lo = max(0, at - case["window"]) if case["window"] >= 0 else 0
            pairs += max(0, hi - lo)
            low = min(low, lo)
        keys += n - low
    return pairs, keys


def work(case):
    D, G, H = case["D"], case["Hq"], case["Hkv"]
    held, fresh = _lengths(case)
    if case["op"] == "append":
        tokens = sum(fresh)
        blocks = sum((h + n - 1) // case["block"] - h // case["block"] + 1 for h, n in zip(held, fresh))
        turned = case["rotary"] > 0
        places = max(h + n for h, n in zip(held, fresh)) - min(held)
        return {"bytes": tokens * 2 * H * D * (2 + 1) + blocks * 2 * H * 4 + turned * (tokens * G * D * 4 + min(places, tokens) * case["rotary"] * 4),
                "flops": turned * tokens * (G + H) * case["rotary"] * 3}
    pairs, keys = _pairs(case)
    return {"bytes": keys * 2 * H * D + keys / case["block"] * 2 * H * 4 + sum(fresh) * G * (D * 4 + 4),
            "flops": 4 * D * G * pairs}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _round_e4m3(x):
    """The nearest e4m3 value, ties to the even one: three bits behind the leading one, steps of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6.0)
    step = torch.exp2(exponent - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact(case, seed):
    state = prepare(case, seed)
    held, fresh = _lengths(case)
    B, D, G, H, bt = case["B"], case["D"], case["Hq"], case["Hkv"], case["block"]
    size = state["k"].shape[1]
    table = state["table"].tolist() if state["table"] is not None else [[b] for b in range(B)]
    if case["op"] == "append":
        cos, sin = (state[n].double() if case["rotary"] else None for n in ("cos", "sin"))
        got = {n: state[n].double() for n in ("k", "v", "k_scale", "v_scale")}
        if case["rotary"]:
            got["q"] = state["q"].double().clone()

        def turned(x, start):                                  # (n, heads, D) from place `start` on
            half = case["rotary"] // 2
            c, s = (t[start:start + x.shape[0], None] for t in (cos, sin))
            y = x.clone()
            one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            y[..., one] = x[..., one] * c - x[..., two] * s
            y[..., two] = x[..., one] * s + x[..., two] * c
            return y

        for b in range(B):
            start, n = held[b], fresh[b]
            fed = {"k": state["k_new"][b, :n].double(), "v": state["v_new"][b, :n].double()}
            if case["rotary"]:
                # (rows of padding are turned too: their places follow)
                got["q"][b] = turned(state["q"][b].double(), start)
                fed["k"] = turned(fed["k"], start)
            # a sequence's blocks in one row, filled up to whole ones: what was there, then what is new
            b0, b1 = start // bt, (start + n - 1) // bt + 1
            places = [(table[b][i * bt // size], i * bt % size) for i in range(b0, b1)]
            pg = torch.tensor([p for p, _ in places], device=state["k"].device)
            off = torch.tensor([o for _, o in places], device=state["k"].device)
            slots = off[:, None] + torch.arange(bt, device=off.device)
            where = torch.arange(b0 * bt, b1 * bt, device=off.device).view(-1, bt)
            is_new = (where >= start) & (where < start + n)
            was_there = where < start
            for name in ("k", "v"):
                full = torch.zeros((b1 - b0) * bt, H, D, dtype=torch.float64, device=off.device)
                full[start - b0 * bt:start - b0 * bt + n] = fed[name]
                full = full.view(b1 - b0, bt, H, D)
                top = (full.abs() * is_new[:, :, None, None]).amax(dim=(1, 3))
                need = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(-120, 120))
                before = got[name + "_scale"][pg, off // bt]
                keep = was_there.any(1)[:, None]
                scale = torch.where(keep, torch.maximum(before, need), need)
                was = got[name][pg[:, None], slots]
                moved = torch.where((keep & (scale > before))[:, None, :, None], _round_e4m3(was * (before / scale)[:, None, :, None]), was)
                y = torch.where(is_new[:, :, None, None], _round_e4m3(full / scale[:, None, :, None]),
                                torch.where(was_there[:, :, None, None], moved, was))
                got[name][pg[:, None], slots] = y
                got[name + "_scale"][pg, off // bt] = scale
        return got
    out, lse = state["out"].double(), state["lse"].double()
    for b in range(B):
        n, rows = held[b], fresh[b]
        pg = torch.tensor(table[b][:-(-n // size)], device=out.device)
        kv = []
        for name in ("k", "v"):
            x = state[name][pg].double().view(len(pg), size // bt, bt, H, D) * state[name + "_scale"][pg].double()[:, :, None, :, None]
            kv.append(x.view(-1, H, D)[:n])
        place = n - rows + torch.arange(rows, device=out.device)[:, None]
        j = torch.arange(n, device=out.device)[None]
        hidden = torch.zeros(rows, n, dtype=torch.bool, device=out.device)
        if case["causal"]:
            hidden |= j > place
        if case["window"] >= 0:
            hidden |= j < place - case["window"]
        for g in range(G):
            s = state["q"][b, :rows, g].double() @ kv[0][:, g // (G // H)].T / math.sqrt(D)
            if case["softcap"]:
                s = case["softcap"] * torch.tanh(s / case["softcap"])
            s[hidden] = -math.inf
            if case["sink"]:
                s = torch.cat([s, state["sink"][g].double().expand(rows, 1)], dim=1)
            total = torch.logsumexp(s, dim=1)
            p = torch.exp(s - torch.where(total > -math.inf, total, 0.0)[:, None])
            out[b, :rows, g] = p[:, :n] @ kv[1][:, g // (G // H)]
            lse[b, g, :rows] = total
    return {"out": out, "lse": lse}
