"""Exact attention for serving: one new token over a paged cache, and packed prompts.

Next to the eviction kernels, which drop tiles, these attend to every visible
key: x = scale * q.k; x = softcap * tanh(x / softcap) where asked for; a bias
of -slope * distance per head; a mask; softmax; the sum over values.  A key
that the mask hides has no effect, whatever its slot holds (infinities and
NaN included), and a query that sees nothing gives 0 and a log-sum of -inf;
one whose visible scores are all -inf gives NaN, as 0 / 0 does.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib


def paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                           seq_lens: torch.Tensor, *, scale: Optional[float] = None, softcap: float = 0.0,
                           alibi_slopes: Optional[torch.Tensor] = None, window: int = 0, k_scale: float = 1.0,
                           v_scale: float = 1.0, return_lse: bool = False):
    """Attention of the newest token of each sequence over its pages.

    q (num_seqs, heads, head_dim) at position seq_lens - 1, its key already in the cache; caches
    (num_blocks, kv_heads, block_size, head_dim) in q's dtype or float8_e4m3fn (values times k_scale /
    v_scale), heads a multiple of kv_heads, head_dim up to 256; block_tables (num_seqs, max_blocks),
    seq_lens (num_seqs,) any length from 0.  ``scale`` defaults to head_dim ** -0.5; ``window`` > 0 keeps
    the last ``window`` keys; ``alibi_slopes`` (heads,) float32.  Returns out like q, or (out, lse) with
    lse (num_seqs, heads) float32, the natural logarithm of the softmax sum.

    Splits the work over the cache's length where there are few sequences; nothing synchronises with the
    host.  A length or a page outside its tables sets the device's status word (:func:`check_status`); the
    length is clamped, and the page's keys and values count as zeros.  float32, and caches that are not aligned
    to 16 bytes or broadcast over heads, are not split and take many times as long for long sequences.
    """
    return _lib.require_binding().decode(q, k_cache, v_cache, block_tables, seq_lens, scale, softcap, alibi_slopes,
                                         window, k_scale, v_scale, return_lse)


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, *,
                     cu_seqlens_k: Optional[torch.Tensor] = None, causal: bool = True,
                     prefix_lens: Optional[torch.Tensor] = None, window: int = 0, scale: Optional[float] = None,
                     softcap: float = 0.0, alibi_slopes: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of packed prompts over themselves.

    q (tokens, heads, head_dim), k and v (tokens, kv_heads, head_dim); document d holds rows
    [cu_seqlens[d], cu_seqlens[d + 1]) and sees nothing of the others (None: one document).  With
    ``cu_seqlens_k`` a document's keys have a length of their own and its queries are the last of its
    positions.  A query at position p sees key j if j <= p (or not ``causal``) and, with ``window`` > 0,
    j > p - window; and every key below ``prefix_lens[d]``.  The bias is -alibi_slopes[h] * |p - j|.
    float16 and bfloat16 with head_dim a multiple of 8 up to 128; float32 up to 256.  Returns out like q,
    or (out, lse) with lse (tokens, heads) float32.

    float32, and 16-bit inputs that are not aligned to 16 bytes or broadcast over heads, go row by row, which
    takes hundreds of times as long for long prompts: make such k and v contiguous first.
    """
    return _lib.require_binding().prompt(q, k, v, cu_seqlens, cu_seqlens_k, causal, prefix_lens, window, scale, softcap,
                                         alibi_slopes, return_lse)
