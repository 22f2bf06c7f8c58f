"""Norm, rotary position and append of a packed batch's new tokens
(hokv_norm_rotate_append).

Between a layer's projections and its attention, the new tokens of every
sequence get their queries and keys normed per head and rotated, and their
keys and values written behind the rows that their sequences' slots already
hold (a CDC-03 store's tiers, [B, H_kv, capacity, D]).  One launch reads the
projections once and writes queries, keys and values once.  The reference's
cache receives rotated keys from the model and stores them token by token
(layer_state.py:68-133).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib as L
from .prefill import _lengths, _rows_apart

_DTYPES = {torch.float16: L.F16, torch.bfloat16: L.BF16, torch.float32: L.F32}


def _check(query, key, value, key_slots, value_slots, cu_seqlens, kv_len, inv_freq, q_weight, k_weight, eps,
           interleaved, positions, out):
    """hokv_norm_rotate_args of these arguments without their addresses."""
    if query.dtype not in _DTYPES or not query.is_cuda or query.dim() != 3:
        raise ValueError(f"Expected f16/bf16/f32 CUDA queries [T, H_q, D], got {tuple(query.shape)} {query.dtype} on "
                         f"{query.device}")
    T, Hq, D = query.shape
    dev, dt = query.device, query.dtype
    if D % 2 or not 2 <= D <= 256:
        raise ValueError(f"Expected an even head_dim up to 256, got {D}")
    Hkv = key.shape[1] if key.dim() == 3 else 0
    if Hq == 0 or Hkv == 0:
        raise ValueError(f"Expected key [{T}, H_kv, {D}], got {tuple(key.shape)} (and {Hq} query heads)")
    slots = tuple(key_slots.shape)
    if key_slots.dim() != 4 or slots[1] != Hkv or slots[3] != D:
        raise ValueError(f"Expected key_slots [B, {Hkv}, capacity, {D}], got {slots}")
    for name, t, shape in (("query", query, (T, Hq, D)), ("key", key, (T, Hkv, D)), ("value", value, (T, Hkv, D)),
                           ("key_slots", key_slots, slots), ("value_slots", value_slots, slots), ("out", out, (T, Hq, D)),
                           ("q_weight", q_weight, (D,)), ("k_weight", k_weight, (D,))):
        if t is None:
            continue
        if t.shape != shape or t.dtype != dt or t.device != dev or (t.numel() and t.stride(-1) != 1):
            raise ValueError(f"Expected {name} {list(shape)} {dt} on {dev} with contiguous head dims, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}, strides {t.stride()}")
    for name, t in (("key_slots", key_slots), ("value_slots", value_slots), ("out", out)):
        if t is not None and not _rows_apart(t):
            raise ValueError(f"Expected {name} with rows that do not overlap, got {tuple(t.shape)}, strides {t.stride()}")
    B = slots[0]
    _lengths(kv_len, B, "kv_len", dev)
    if cu_seqlens is not None:
        _lengths(cu_seqlens, B + 1, "cu_seqlens", dev)
    elif T != B:
        raise ValueError(f"without cu_seqlens every sequence has one token: got {T} tokens for {B} sequences")
    if positions is not None:
        _lengths(positions, T, "positions", dev)
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or inv_freq.device != dev or not inv_freq.is_contiguous() \
            or 2 * inv_freq.shape[0] > D:
        raise ValueError(f"Expected inv_freq as a contiguous float32 vector of up to {D // 2} entries on {dev}, got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype} on {inv_freq.device}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"Expected a finite eps >= 0, got {eps}")
    a = L.NormRotateArgs()
    a.dtype, a.n_seqs, a.q_heads, a.kv_heads, a.head_dim = _DTYPES[dt], B, Hq, Hkv, D
    a.n_freq, a.interleaved, a.zero_tail, a.eps, a.n_tokens = inv_freq.shape[0], interleaved, out is None, eps, T
    a.q_stride_t, a.q_stride_h = query.stride()[:2]
    a.k_stride_t, a.k_stride_h = key.stride()[:2]
    a.v_stride_t, a.v_stride_h = value.stride()[:2]
    a.out_stride_t, a.out_stride_h = (Hq * D, D) if out is None else out.stride()[:2]
    a.ks_stride_b, a.ks_stride_h, a.ks_stride_t = key_slots.stride()[:3]
    a.vs_stride_b, a.vs_stride_h, a.vs_stride_t = value_slots.stride()[:3]
    a.capacity = slots[2]
    return a


_checked = L.Checked()


def norm_rotate_append(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, key_slots: torch.Tensor,
                       value_slots: torch.Tensor, cu_seqlens: Optional[torch.Tensor], kv_len: torch.Tensor,
                       inv_freq: torch.Tensor, q_weight: Optional[torch.Tensor] = None,
                       k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                       positions: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotated queries [T, H_q, D]; keys and values appended to their slots.

    query [T, H_q, D], key/value [T, H_kv, D] (contiguous head dims, any other strides: parts of one projection are
    fine); sequence b owns tokens [cu_seqlens[b], cu_seqlens[b + 1]) (cu_seqlens None: token b).  Token i of b sits at
    position kv_len[b] + i, or positions[t] when given (sequences behind a shared prefix), and its key and value go to
    row kv_len[b] + i of key_slots/value_slots [B, H_kv, capacity, D].  kv_len (the rows held before the call) is
    not changed.  With q_weight / k_weight [D] the head is first multiplied by weight / sqrt(mean(x^2) + eps).
    inv_freq [F] float32, 2F <= D, turns dims (f, f + F), or (2f, 2f + 1) when ``interleaved``, by position *
    inv_freq[f]; the dims behind 2F keep their values.  f16, bf16 or f32, the same for all but lengths and inv_freq;
    even head dims up to 256.  ``out`` may be the query itself; rows of no sequence (ahead of the first,
    behind the last) are zeros, or left as they were in a given ``out``.  A row that does not fit its slot is reported by the device status."""
    eps, interleaved = float(eps), bool(interleaved)   # values, not objects: a tensor may change behind its identity
    sig = L.signature
    geometry = (sig(query), sig(key), sig(value), sig(key_slots), sig(value_slots), sig(kv_len), sig(inv_freq), eps,
                interleaved, cu_seqlens is not None and sig(cu_seqlens), q_weight is not None and sig(q_weight),
                k_weight is not None and sig(k_weight), positions is not None and sig(positions),
                out is not None and sig(out))
    known = _checked.get(geometry)
    if known is None:
        known = _checked.keep(geometry, _check(query, key, value, key_slots, value_slots, cu_seqlens, kv_len, inv_freq,
                                               q_weight, k_weight, eps, interleaved, positions, out))
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if not known.n_tokens:
        return out
    a = L.NormRotateArgs.from_buffer_copy(known)
    a.q, a.k, a.v, a.out, a.k_slots, a.v_slots, a.kv_len, a.inv_freq = (
        query.data_ptr(), key.data_ptr(), value.data_ptr(), out.data_ptr(), key_slots.data_ptr(), value_slots.data_ptr(),
        kv_len.data_ptr(), inv_freq.data_ptr())
    if cu_seqlens is not None:
        a.cu_seqlens = cu_seqlens.data_ptr()
    if positions is not None:
        a.positions = positions.data_ptr()
    if q_weight is not None:
        a.q_weight = q_weight.data_ptr()
    if k_weight is not None:
        a.k_weight = k_weight.data_ptr()
    L.check_call(L.call_on(geometry[0][3], L.lib().hokv_norm_rotate_append, a), "norm_rotate_append")
    return out
