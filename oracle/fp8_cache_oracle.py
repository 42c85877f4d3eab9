"""The 8-bit KV cache in 64 bits on the CPU: what appending tokens leaves in it and what attention over it gives.  Test
infrastructure only; plain loops over sequences and heads."""
import math

import torch


def round_e4m3(x):
    """The nearest e4m3 value (ties to even, at most 448): three bits behind the leading one, steps of 2^-9 below 2^-6."""
    x = x.double()
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -40))).clamp(min=-6.0)
    step = torch.exp2(e - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def rotate(x, cos, sin, start, interleaved):
    """x (S, heads, D), row i at position start + i; fp32, each step rounded, as the definition says."""
    x = x.float().clone()
    half = cos.shape[1]
    c = cos[start:start + x.shape[0], None].float()
    s = sin[start:start + x.shape[0], None].float()
    if interleaved:
        a, b = x[..., 0:2 * half:2].clone(), x[..., 1:2 * half:2].clone()
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :half].clone(), x[..., half:2 * half].clone()
        x[..., :half], x[..., half:2 * half] = a * c - b * s, b * c + a * s
    return x


def scale_for(top):
    """The smallest power of two, 2^-120 at least, that leaves `top` at most 448."""
    if top == 0:
        return 2.0 ** -120
    return 2.0 ** min(120, max(-120, math.ceil(math.log2(top / 448.0))))


def append(values, scales, new, held, table, block):
    """Tokens `new` (n, heads, D) behind the `held` ones of a sequence whose pages are `table`; values (pages, size, heads, D)
    and scales (pages, size / block, heads), both float64 of what the cache stands for in units of the scale, are changed."""
    n, H, _ = new.shape
    if n == 0:
        return
    size = values.shape[1]
    new = new.double()
    for first in range(held // block * block, held + n, block):
        page, off = table[first // size], first % size
        t0, t1 = max(held, first), min(held + n, first + block)
        for h in range(H):
            x = new[t0 - held:t1 - held, h]
            fine = x.isfinite()
            top = float(torch.where(fine, x.abs(), 0.0).max())
            scale = scale_for(top)
            if held > first:
                old = float(scales[page, off // block, h])
                scale = max(scale, old)
                if scale != old:
                    part = values[page, off:off + held - first, h]
                    values[page, off:off + held - first, h] = torch.where(part.isnan(), part, round_e4m3(part * (old / scale)))
            values[page, off + t0 - first:off + t1 - first, h] = torch.where(fine, round_e4m3(x / scale), math.nan)
            scales[page, off // block, h] = scale


def attend(q, k, v, rows, softmax_scale=None, causal=False, window=(None, None), sink=None, softcap=0.0):
    """q (Sq, Hq, D) of a sequence, of which the first `rows` are there; k, v (n, Hkv, D) what the cache stands for.
    Returns out (rows, Hq, D) and lse (Hq, rows)."""
    n, H, D = k.shape
    G = q.shape[1]
    scale = 1 / math.sqrt(D) if softmax_scale is None else softmax_scale
    left, right = window
    if causal:
        right = 0
    at = n - rows + torch.arange(rows, device=k.device)[:, None]
    j = torch.arange(n, device=k.device)[None]
    hidden = torch.zeros(rows, n, dtype=torch.bool, device=k.device)
    if left is not None:
        hidden |= j < at - left
    if right is not None:
        hidden |= j > at + right
    out = torch.zeros(rows, G, D, dtype=torch.float64, device=k.device)
    lse = torch.zeros(G, rows, dtype=torch.float64, device=k.device)
    for g in range(G):
        s = q[:rows, g].double() @ k[:, g // (G // H)].double().T * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s[hidden] = -math.inf
        if sink is not None:
            s = torch.cat([s, sink[g].double().expand(rows, 1)], dim=1)
        total = torch.logsumexp(s, dim=1) if s.shape[1] else torch.full((rows,), -math.inf, dtype=torch.float64, device=k.device)
        p = torch.exp(s - torch.where(total > -math.inf, total, 0.0)[:, None])[:, :n]
        # (a key that a row does not see adds nothing to it, whatever its value is)
        out[:, g] = p @ v[:, g // (G // H)].double()
        lse[g] = total
    return out, lse
