"""Exact attention of sequences that share a long prefix (hokv_packed_attention
with a prefix).

Samples of one prompt, or requests behind one system prompt, see the same
leading keys and values and some tokens of their own.  The prefix is held
once, without a batch dim, and is attended once for the queries of all
sequences together (their rows fill the tensor-core tiles); each sequence's
own keys sit in its slot of a store (CDC03Store.k[layer], [B, H_kv, capacity,
D]) and the parts are joined by their softmax statistics.  The reference has
no counterpart: its caches hold one sequence per batch row
(compressed_cache.py:72-105).
"""

from __future__ import annotations

from typing import Optional

import torch

from .prefill import _packed


def shared_prefix_attention(query: torch.Tensor, prefix_key: torch.Tensor, prefix_value: torch.Tensor,
                            key: torch.Tensor, value: torch.Tensor, kv_len: Optional[torch.Tensor] = None,
                            cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                            scaling: Optional[float] = None, is_causal: bool = True,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(query [prefix_key; key_b]^T * scaling) [prefix_value; value_b] for every sequence b.

    prefix_key/prefix_value [H_kv, P, D], seen whole by every query; the other arguments are packed_attention's:
    query [T, H_q, D] with cu_seqlens_q (without it one token per sequence), each sequence's own key/value in slots
    [B, H_kv, capacity, D] with kv_len [B], or packed [S, H_kv, D] with cu_seqlens_k, causal among its own keys (query i
    of m sits at own position n - m + i).  -> [T, H_q, D].  Scratch grows with T (about 8 H_q D bytes per token), so
    this form is for decoding and drafted tokens, not for long prompts behind a prefix."""
    if (prefix_key is None) != (prefix_value is None):
        raise ValueError("Expected prefix_key and prefix_value, got one of them")
    return _packed("shared_prefix_attention", query, key, value, cu_seqlens_q, cu_seqlens_k, kv_len, scaling, is_causal,
                   out, prefix_key, prefix_value)
