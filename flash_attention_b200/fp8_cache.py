"""A KV cache in 8 bits: filled token by token, read by bf16 queries.

The NVFP4 operands of :func:`flash_attn_fp4_func` are made from whole tensors; a serving loop gets its keys and values a
token (or a prompt) at a time.  Here the cache holds e4m3 values and one fp32 scale for each block of tokens and kv
head: :func:`append_kv_fp8` writes new tokens into its pages, rotating keys and queries on the way, and
:func:`flash_attn_fp8_cache_func` attends to it.  The reference's call of this kind is ``flash_attn_with_kvcache``
(hopper/flash_attn_interface.py), which does both in one for fp16 / bf16 caches.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib


@dataclass
class FP8KVCache:
    """Keys and values of a pool of pages, or (without a page table) of one page for each sequence.

    k, v              (num_pages, page_size, heads, head_dim) float8_e4m3fn (or its bytes as uint8); head_dim 64 or 128, contiguous;
                      the other strides are multiples of 16 bytes, so a pool stored as (page, head, token) is passed transposed
    k_scale, v_scale  (num_pages, page_size / block, heads) fp32, contiguous: value = byte * scale, no scale below 0.  ``block`` tokens
                      (16, 32, 64 or 128) share a scale
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    @classmethod
    def empty(cls, num_pages: int, page_size: int, num_heads_kv: int, head_dim: int, block: Optional[int] = None,
              device=None) -> "FP8KVCache":
        """A cache that holds nothing (its memory is not cleared: what no sequence's length covers is never used).
        ``block``: tokens of a scale, the largest of 128, 64, 32, 16 that divides the page by default."""
        if block is None:
            block = next((n for n in (128, 64, 32, 16) if page_size % n == 0), 0)
        if block not in (16, 32, 64, 128) or page_size % block != 0:
            raise ValueError(f"page_size {page_size} is no multiple of a block of 16, 32, 64 or 128 tokens (block {block})")
        device = torch.device("cuda") if device is None else torch.device(device)
        values = lambda: torch.empty(num_pages, page_size, num_heads_kv, head_dim, dtype=torch.float8_e4m3fn, device=device)
        scales = lambda: torch.empty(num_pages, page_size // block, num_heads_kv, dtype=torch.float32, device=device)
        return cls(values(), values(), scales(), scales())

    @property
    def block(self) -> int:
        return self.k.shape[1] // self.k_scale.shape[1]

    def dequantize(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """fp32 keys and values in the layout of the pool."""
        def whole(x, scale):
            x = x.view(torch.float8_e4m3fn) if x.dtype == torch.uint8 else x
            return x.float() * scale.repeat_interleave(self.block, dim=1)[..., None]
        return whole(self.k, self.k_scale), whole(self.v, self.v_scale)


def append_kv_fp8(
    cache: FP8KVCache, k: torch.Tensor, v: torch.Tensor,
    cache_seqlens: torch.Tensor,
    page_table: Optional[torch.Tensor] = None,
    seqused_new: Optional[torch.Tensor] = None,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    rotary_interleaved: bool = False,
    q: Optional[torch.Tensor] = None,
) -> Optional[torch.Tensor]:
    """Keys and values of new tokens into ``cache``; returns the rotated ``q`` (or ``None``).

    k, v (B, S, heads, head_dim) bf16: token i of sequence b goes to position ``cache_seqlens[b] + i``.  ``cache_seqlens`` (B,)
    int32 is what each sequence holds already; it is not changed.  ``seqused_new`` (B,) int32: how many of the S tokens are
    there (a batch padded to its longest); the rest is not read.  ``page_table`` (B, pages_per_seq) int32: page of every ``page_size``
    positions; ``None``: page b of the cache is sequence b's.

    ``rotary_cos``, ``rotary_sin`` (positions, rotary_dim / 2), fp32 or bf16: the first ``rotary_dim`` elements of keys (and
    of ``q`` (B, S, q heads, head_dim), if given) are rotated by their position, in pairs of halves or, with
    ``rotary_interleaved``, of neighbours -- the reference's arguments of these names.  rotary_dim is a multiple of 16.  All
    S rows of q come back, those of padding too.

    The scale of a block is the smallest power of two that leaves its values at most 448; it grows with the tokens, and those
    in the block are then rounded to the new one (exact but for values 2^15 below the largest).  A value that is not finite is
    stored as NaN.  Nothing here is differentiable.  One launch, no synchronisation; can be captured in a graph.  Positions behind the cache's or the
    tables' end and page numbers outside the pool cannot be refused here (they are on the device): such
    tokens are left out, or turned by the tables' last row, and :func:`check_status` raises.  No block may belong to two sequences that append to it in one call.
    """
    return _lib.host().append_fp8(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, k, v, cache_seqlens, seqused_new,
                                  rotary_cos, rotary_sin, rotary_interleaved, q)


def flash_attn_fp8_cache_func(
    q: torch.Tensor, cache: FP8KVCache,
    seqused_k: torch.Tensor,
    page_table: Optional[torch.Tensor] = None,
    seqused_q: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = False,
    window_size: Tuple[Optional[int], Optional[int]] = (None, None),
    learnable_sink: Optional[torch.Tensor] = None,
    softcap: float = 0.0,
    num_splits: int = 0,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of q (B, Sq, heads, head_dim) bf16 over an 8-bit cache; returns ``(out, lse fp32 (B, heads, Sq) | None)``.

    ``seqused_k`` (B,) int32: sequence b attends to its first ``seqused_k[b]`` tokens (those that :func:`append_kv_fp8` has just
    written among them).  ``seqused_q`` (B,) int32: how many of the Sq rows are there; the others are not written (in a new ``out`` and
    ``lse`` they are zeros).  Row i stands at position ``seqused_k[b] - seqused_q[b] + i``, which ``causal`` and
    ``window_size`` refer to.  ``learnable_sink``, ``softcap``, ``num_splits`` (0: chosen), ``out`` and ``lse`` as in
    :func:`flash_attn_fp4_func` (a soft cap lies in 1e-37 .. 1e37, and so does softmax_scale / softcap); a row that sees nothing gets zeros and an
    lse of -inf, or its head's sink.

    Not differentiable.  Scores take a query's elements as they are down to 2^-10 of the row's largest, smaller ones to 2^-18 of it.  A row's softmax weights, times their value scales, keep eight bits down to 2^-14 of the largest among 128 keys and are
    right to 2^-22 of it below (more than 32 rows per kv head: eleven bits down to 2^-20 of the largest so far, right to 2^-31 of that below).  So an
    output element that is made by less than that (the values of the keys that weigh are zero there) is right to that much of the others, not to
    bf16.  Value scales that a row sees lie within a factor of 2^90 of each other.

    A length beyond the cache's or the table's end counts as that end, a negative one as 0 (they are on the device and cannot be
    refused).  The cache behind a sequence's last token may hold anything, NaN included.  A NaN in a value that some row of a sequence sees may
    reach the other rows of that sequence too.  Page numbers outside the pool stand for keys and values of zero, and
    :func:`check_status` raises.
    """
    win_left, win_right = window_size
    return _lib.host().fwd_fp8(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, q, seqused_k, seqused_q, softmax_scale,
                               causal, win_left, win_right, learnable_sink, softcap, num_splits, return_lse, out, lse)
