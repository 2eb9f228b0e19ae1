"""
Paged KV cache in 16 or 8 bits: rotation and append, and attention to it.

A serving loop keeps every sequence's keys and values in pages of a shared pool, and a page
table that names them in order.  One step of one layer:

    q = paged_kvcache_append(k, v, k_cache, v_cache, page_table, lens, k_scale=k_scale,
                             v_scale=v_scale, q=q, rotary_cos=cos, rotary_sin=sin)
    o = flash_attn_with_paged_kvcache(q, k_cache, v_cache, page_table, lens + q.shape[1],
                                      k_scale=k_scale, v_scale=v_scale)

The same two calls take a whole prompt, a chunk of one behind cached rows, a few proposed
tokens, or the single token of a decode step.  For inference: no gradients flow through them.
The reference has neither a paged nor an 8-bit cache (its decode step is eager PyTorch,
integrations.py:77-98).
"""

import math
from typing import Optional, Tuple, Union

import torch

from . import hip_ext as _ext
from .flash_attn import _DTYPES, _HEAD_DIMS


def rotary_cos_sin(positions: int, rotary_dim: int, base: float = 10000.0,
                   device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cosines and sines [positions, rotary_dim / 2] float32 of the angles p * base^(-2j / rotary_dim),
    computed in 64 bits (in 32 the angle of position 100000 is off by 0.004)."""
    assert rotary_dim % 2 == 0, f"rotary_dim must be even, got {rotary_dim}"
    freq = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _check(name, x, cu_seqlens, max_seqlen):
    assert x.dtype in _DTYPES, f"{name} must be float16 or bfloat16, got {x.dtype}"
    d = x.shape[-1]
    assert d in _HEAD_DIMS, f"head_dim must be 32, 64, 96, 128, or 256, got {d}"
    assert (cu_seqlens is None) == (max_seqlen is None), "cu_seqlens and the longest sequence's length go together"


def _lengths(cache_seqlens, page_table):
    if isinstance(cache_seqlens, int):
        return torch.full((page_table.shape[0],), cache_seqlens, dtype=torch.int32, device=page_table.device)
    return cache_seqlens


def paged_kvcache_append(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_seqlens: Union[torch.Tensor, int],
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    q: Optional[torch.Tensor] = None,
    cu_seqlens: Optional[torch.Tensor] = None,
    max_seqlen: Optional[int] = None,
    rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None,
    rotary_interleaved: bool = False,
    cache_layout: str = "bshd",
) -> Optional[torch.Tensor]:
    """
    Append new keys and values to a paged cache, in place, rotating keys (and queries) by
    their positions on the way; one launch.

    Token i of sequence b becomes row ``cache_seqlens[b] + i``, that is row
    ``(cache_seqlens[b] + i) % page_size`` of page ``page_table[b, (cache_seqlens[b] + i) // page_size]``.
    Rows past the page table's last page and rows of pages outside the pool are dropped.  A page
    that is written must belong to one sequence only, and keys and values have a cache and scales
    each (they may be views of one pool).

    Caches of k's type hold the rows rounded once.  float8_e4m3fn caches hold codes, and
    ``code * scale[page, head]`` is the value.  The scale of a page that the call writes becomes
    the smallest power of two in which every finite value it puts there is at most 448; if the
    page held rows of the sequence before, it only grows, and their codes are rounded to the
    new scale.  Infinities become the largest code, NaN stays NaN.

    Args:
        k, v: [B, n, H_kv, d] float16 or bfloat16, or packed [total, H_kv, d] with ``cu_seqlens``
        k_cache, v_cache: [num_pages, page_size, H_kv, d] (``cache_layout="bshd"``) or
            [num_pages, H_kv, page_size, d] (``"bhsd"``), k's dtype or float8_e4m3fn; page_size
            a multiple of 16; may be strided (contiguous in d, other strides multiples of 16 bytes)
        page_table: int32 [B, max_pages]
        cache_seqlens: int32 [B], rows before the append (or an int for all sequences)
        k_scale, v_scale: float32 [num_pages, H_kv], for float8 caches; updated in place
        q: queries of the same tokens, [B, n, H_q, d] or [total, H_q, d], to be rotated
        cu_seqlens, max_seqlen: int32 [B + 1] offsets of packed tokens and the longest
            sequence's length (only speed depends on it)
        rotary_cos, rotary_sin: float32 [positions, rotary_dim / 2], row p for position p, at
            least as many as the page table holds (see ``rotary_cos_sin``); rotary_dim a
            multiple of 16, at most d: the elements past it are left as they are.  None: no rotation
        rotary_interleaved: rotate the pairs (2j, 2j + 1), not (j, j + rotary_dim / 2)

    Returns:
        The rotated queries (a new tensor; zeros in rows outside every sequence), or None without ``q``.
    """
    _check("k", k, cu_seqlens, max_seqlen)
    return _ext.paged_append(k, v, k_cache, v_cache, page_table, _lengths(cache_seqlens, page_table), k_scale, v_scale,
                             q, cu_seqlens, max_seqlen or 0, rotary_cos, rotary_sin, rotary_interleaved, cache_layout)


def flash_attn_with_paged_kvcache(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    page_table: torch.Tensor,
    cache_seqlens: Union[torch.Tensor, int],
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    max_seqlen_q: Optional[int] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = True,
    return_softmax_lse: bool = False,
    cache_layout: str = "bshd",
):
    """
    Attention of the last tokens of each sequence to its paged cache, which holds their own
    keys and values too (``paged_kvcache_append`` puts them there).

    One token per sequence is a decode step (the causal mask then hides nothing), a few are a
    speculative decoding's proposal, many a prompt or a chunk of one.

    Args:
        q: [B, n, H_q, d] float16 or bfloat16, [B, H_q, d] for one token each, or packed
            [total, H_q, d] with ``cu_seqlens_q``; H_q a multiple of H_kv
        k_cache, v_cache, k_scale, v_scale, page_table, cache_layout: as in
            ``paged_kvcache_append``; pages outside the pool are skipped
        cache_seqlens: int32 [B], rows of the cache, those of the tokens included (or an int for
            all sequences)
        cu_seqlens_q, max_seqlen_q: int32 [B + 1] offsets of packed tokens and the longest
            sequence's length (only speed depends on it)
        softmax_scale: default 1/sqrt(d)
        causal: token i of a sequence's n sees the rows j <= cache_seqlens[b] - n + i
            (bottom-right aligned: the last token sees all); False: every token sees all rows
        return_softmax_lse: also return the natural-log LSE, float32 of q's shape without d

    Returns:
        A tensor of q's shape and dtype, and the LSE if requested.  Tokens that see no row, and
        packed rows outside every sequence, get zeros (LSE -inf).
    """
    _check("q", q, cu_seqlens_q, max_seqlen_q)
    one = cu_seqlens_q is None and q.dim() == 3
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(q.shape[-1])
    res = _ext.paged_attention(q.unsqueeze(1) if one else q, k_cache, v_cache, page_table,
                               _lengths(cache_seqlens, page_table), softmax_scale, k_scale, v_scale, cu_seqlens_q,
                               max_seqlen_q or 0, causal, cache_layout, return_softmax_lse)
    if not one:
        return res
    return tuple(t.squeeze(1) for t in res) if return_softmax_lse else res.squeeze(1)
