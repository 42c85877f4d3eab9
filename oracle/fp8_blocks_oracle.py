"""Chosen blocks of the 8-bit KV cache on the CPU: the index, the choice and the attention over it, in whole numbers and 64
bits.  Test infrastructure only; plain loops over sequences, heads and blocks."""
import math

import torch


def index(values, k_scale):
    """Bounds (H, 2, D) int8 and their scale (H,) fp32 of a block's keys: values (tokens, H, D) of the bytes, k_scale (H,)."""
    n, H, D = values.shape
    bounds = torch.zeros(H, 2, D, dtype=torch.int8)
    scale = torch.zeros(H)
    for h in range(H):
        x = values[:, h].double()
        if x.isnan().any():
            scale[h] = math.nan
            continue
        top = float(x.abs().max())
        e = math.frexp(top)[1] - 1 if top > 0 else -9
        step = 2.0 ** (e - 6)
        bounds[h, 0] = torch.ceil(x.amax(0) / step).to(torch.int8)
        bounds[h, 1] = torch.floor(x.amin(0) / step).to(torch.int8)
        scale[h] = k_scale[h].float() * step
    return bounds, scale


def seven_bits(q):
    """p and n (D,) of the queries (rows, heads, D) that choose together, as Python integers' tensor."""
    q = q.double()
    q = torch.where(q.isfinite(), q, 0.0)
    top = float(q.abs().max()) if q.numel() else 0.0
    e = max(-100, math.frexp(top)[1] - 1) if top > 0 else -100
    x = torch.round(q * 2.0 ** (14 - e)).long().flatten(0, 1)              # (half to even)
    P, N = x.clamp(min=0).sum(0), (-x).clamp(min=0).sum(0)
    s = max(0, int(max(P.max(), N.max())).bit_length() - 7)
    half = (1 << s) >> 1
    return ((P + half) >> s).clamp(max=127), ((N + half) >> s).clamp(max=127)


def scores(q, bounds, scale):
    """fp32 scores of blocks (n,) for bounds (n, 2, D) and scale (n,) of one kv head; NaN as +inf."""
    p, n = seven_bits(q)
    dot = (bounds[:, 0].long() * p - bounds[:, 1].long() * n).sum(-1)
    assert int(dot.abs().max()) < 2 ** 24 if len(dot) else True
    s = dot.float() * scale
    return torch.where(s.isnan(), math.inf, s)


def select(q, bounds, scale, first, end, block, chosen, front, recent):
    """The list of a query block: q (rows, heads, D), the first row at position `first`, the last one seeing tokens in front of `end`."""
    n = -(-max(end, 0) // block)
    own = max(0, max(first, 0) // block - (recent - 1))
    if n <= chosen:
        got = list(range(n))
    else:
        s = scores(q, bounds[:n], scale[:n]).tolist()
        must = [j for j in range(n) if j < front or j >= own]
        rest = sorted((j for j in range(n) if not (j < front or j >= own)), key=lambda j: (-s[j], j))
        got = sorted(must + rest[:chosen - len(must)])
    return got + [-1] * (chosen - len(got))


def attend(q, k, v, keys, place, softmax_scale=None, sink=None, softcap=0.0):
    """One row of a kv head: q (heads, D) at position `place`, over the tokens `keys` of k, v (tokens, D).  out (heads, D), lse (heads,)."""
    keys = [t for t in keys if t <= place]
    scale = 1 / math.sqrt(q.shape[-1]) if softmax_scale is None else softmax_scale
    s = q.double() @ k[keys].double().T * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if sink is not None:
        s = torch.cat([s, sink.double()[:, None]], dim=1)
    if s.shape[1] == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    total = torch.logsumexp(s, dim=1)
    p = torch.exp(s - torch.where(total > -math.inf, total, 0.0)[:, None])[:, :len(keys)]
    return p @ v[keys].double(), total


def keys_of(entries, block):
    """The tokens of a list, which ends at the first entry that is not above the one in front of it."""
    got, last = [], -1
    for e in entries:
        if e <= last:
            break
        got += range(e * block, (e + 1) * block)
        last = e
    return got
