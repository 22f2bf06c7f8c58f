"""Exact multi-token attention on the tensor cores (hokv_prefill_attention).

The reference's cache hands exact K/V to the model's own attention for every
prefill and for the layers it keeps exact (compressed_cache.py:72-105).  This
module is that attention as one CUDA launch per layer: causal (query i at
position kv_len - q_len + i) or full, grouped-query heads read from their
shared KV head, f16/bf16, head_dim 64 or 128, (batch, head, token) strides that
nest (any permutation of a packed layout, or a slice of one: the CDC-03 store's
views and the transposed projections a model passes need no copy), contiguous
head dims, key and value with the same strides.

``packed_attention`` is the same attention for a batch of sequences of
different lengths in one launch (hokv_packed_attention): whole prompts, chunks
of prompts behind their histories and single tokens side by side, with the keys
and values packed like the queries or in slots (a CDC-03 store's tiers).
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib as L

_DTYPES = {torch.float16: L.F16, torch.bfloat16: L.BF16}


def supported(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> bool:
    """True when hokv_prefill_attention takes these tensors as they are."""
    if query.dtype not in _DTYPES or key.dtype != query.dtype or value.dtype != query.dtype:
        return False
    if query.dim() != 4 or key.dim() != 4 or value.dim() != 4 or query.shape[-1] not in (64, 128):
        return False
    if key.shape != value.shape or key.shape[-1] != query.shape[-1] or query.shape[0] != key.shape[0]:
        return False
    if query.shape[1] % key.shape[1] != 0:
        return False
    for t in (query, key, value):
        if not t.is_cuda or t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:3]):
            return False
        if not _nests(t):
            return False
    return key.stride() == value.stride()


def _nests(t: torch.Tensor) -> bool:
    """The (token, head, batch) dims, in ascending stride order, each cover the
    dims inside them (the tensor maps the kernel loads through need this;
    dims of extent 1 always fit)."""
    dims = sorted(((t.stride(i), t.shape[i]) for i in (2, 1, 0) if t.shape[i] > 1))
    need = t.shape[3]
    for stride, extent in dims:
        if stride < need:
            return False
        need = stride * extent
    return True


def prefill_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scaling: Optional[float] = None,
                      is_causal: bool = True, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(query key^T * scaling [causal]) value.

    query [B, H_q, q_len, D], key/value [B, H_kv, kv_len, D] (H_q a multiple of
    H_kv) -> [B, q_len, H_q, D] (the layout a Hugging Face attention function
    returns), in the query's dtype."""
    if not supported(query, key, value):
        raise ValueError(f"Expected f16/bf16 CUDA tensors [B, H, S, 64|128] with contiguous head dims and "
                         f"strides in multiples of 8 elements, got {tuple(query.shape)} {query.dtype}, "
                         f"{tuple(key.shape)} {key.dtype}")
    B, Hq, Sq, D = query.shape
    Hkv, Skv = key.shape[1], key.shape[2]
    if is_causal and Skv < Sq:
        raise ValueError(f"causal attention needs kv_len >= q_len, got {Skv} < {Sq}")
    scale = float(scaling) if scaling is not None else D ** -0.5
    if out is None:
        out = torch.empty((B, Sq, Hq, D), dtype=query.dtype, device=query.device)
    elif out.shape != (B, Sq, Hq, D) or out.dtype != query.dtype or out.stride(-1) != 1:
        raise ValueError(f"Expected out [{B}, {Sq}, {Hq}, {D}] {query.dtype}, got {tuple(out.shape)} {out.dtype}")
    lib = L.lib()
    L.check(lib.hokv_prefill_attention(
        L.ptr(query), L.ptr(key), L.ptr(value), L.ptr(out), _DTYPES[query.dtype], B, Hq, Hkv, Sq, Skv, D,
        query.stride(0), query.stride(1), query.stride(2), key.stride(0), key.stride(1), key.stride(2),
        value.stride(0), value.stride(1), value.stride(2), out.stride(0), out.stride(2), out.stride(1),
        scale, 1 if is_causal else 0, L.stream()), "prefill_attention")
    return out


def _rows_apart(t: torch.Tensor) -> bool:
    """No two rows (last dim) of t share memory: in ascending stride order every dim covers the dims inside it."""
    if t.numel() == 0:
        return True
    need = t.shape[-1]
    for stride, extent in sorted((t.stride(i), t.shape[i]) for i in range(t.dim() - 1) if t.shape[i] > 1):
        if stride < need:
            return False
        need = stride * extent
    return True


def _lengths(t, n: Optional[int], name: str, device) -> None:
    """A contiguous int32 CUDA vector (of n entries, when given) on `device`."""
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != device or not t.is_cuda:
        raise ValueError(f"Expected {name} as a contiguous int32 vector on {device}, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device}")
    if n is not None and t.shape[0] != n:
        raise ValueError(f"Expected {name} of {n} entries, got {t.shape[0]}")


def _packed_check(query, key, value, cu_seqlens_q, cu_seqlens_k, kv_len, scaling, is_causal, out, prefix_key,
                  prefix_value):
    """hokv_packed_args of these arguments without their addresses, and its workspace bytes."""
    if query.dtype not in _DTYPES or not query.is_cuda or query.dim() != 3:
        raise ValueError(f"Expected f16/bf16 CUDA queries [T, H_q, D], got {tuple(query.shape)} {query.dtype} on "
                         f"{query.device}")
    T, Hq, D = query.shape
    dev = query.device
    slots = key.dim() == 4
    for name, t in (("key", key), ("value", value)):
        if t.dtype != query.dtype or t.device != dev or t.dim() not in (3, 4) or t.shape != key.shape or t.shape[-1] != D:
            raise ValueError(f"Expected {name} [S, H_kv, {D}] or [B, H_kv, capacity, {D}] like the key, {query.dtype} on "
                             f"{dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    Hkv = key.shape[1]
    if Hkv == 0 or Hq == 0 or Hq % Hkv or Hq // Hkv > 128:
        raise ValueError(f"Expected query heads a multiple (up to 128) of the KV heads, got {Hq} and {Hkv}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"Expected a head_dim in multiples of 8 up to 128, got {D}")
    a = L.PackedArgs()
    if slots:
        if kv_len is None or cu_seqlens_k is not None:
            raise ValueError("keys in slots [B, H_kv, capacity, D] need kv_len [B] (and no cu_seqlens_k)")
        B = key.shape[0]
        _lengths(kv_len, B, "kv_len", dev)
        a.kv_in_slots, a.kv_rows = 1, key.shape[2]
    else:
        if kv_len is not None:
            raise ValueError("packed keys [S, H_kv, D] take cu_seqlens_k, not kv_len")
        if cu_seqlens_k is None:
            raise ValueError("packed keys [S, H_kv, D] need cu_seqlens_k or cu_seqlens_q")
        _lengths(cu_seqlens_k, None, "cu_seqlens_k", dev)
        B = cu_seqlens_k.shape[0] - 1
        a.kv_rows = key.shape[0]
    if B < 0:
        raise ValueError("cu_seqlens_k needs at least one entry")
    if cu_seqlens_q is not None:
        _lengths(cu_seqlens_q, B + 1, "cu_seqlens_q", dev)
    elif T != B:
        raise ValueError(f"without cu_seqlens_q every sequence has one query: got {T} queries for {B} sequences")
    scale = scaling if scaling is not None else D ** -0.5
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"Expected a positive finite scaling, got {scaling}")
    prefix = (("prefix_key", prefix_key), ("prefix_value", prefix_value)) if prefix_key is not None else ()
    for name, t in prefix:
        if t.dim() != 3 or t.shape[0] != Hkv or t.shape[2] != D or t.shape != prefix_key.shape or t.dtype != query.dtype \
                or t.device != dev:
            raise ValueError(f"Expected {name} [{Hkv}, P, {D}] {query.dtype} on {dev}, got {tuple(t.shape)} {t.dtype} on "
                             f"{t.device}")
    for name, t in (("query", query), ("key", key), ("value", value), *prefix):
        if t.numel() and (t.stride(-1) != 1 or any(s % 8 for s in t.stride()[:-1])):
            raise ValueError(f"Expected {name} with contiguous head dims and strides in multiples of 8 elements, got "
                             f"strides {t.stride()}")
    if T > 1 and query.stride(0) < (Hq * query.stride(1) if Hq > 1 else D):
        raise ValueError(f"Expected queries [T, H_q, D] whose token stride covers the heads, got strides {query.stride()}")
    if out is not None and (out.shape != query.shape or out.dtype != query.dtype or out.device != dev
                            or (out.numel() and (out.stride(2) != 1 or out.stride(0) % 8 or out.stride(1) % 8))):
        raise ValueError(f"Expected out [{T}, {Hq}, {D}] {query.dtype} on {dev} with contiguous rows and strides in "
                         f"multiples of 8 elements, got {tuple(out.shape)} {out.dtype} on {out.device}")
    if out is not None and not _rows_apart(out):
        raise ValueError(f"Expected out with rows that do not overlap, got {tuple(out.shape)}, strides {out.stride()}")
    a.dtype, a.n_seqs, a.q_heads, a.kv_heads, a.head_dim, a.causal = _DTYPES[query.dtype], B, Hq, Hkv, D, is_causal
    a.scale, a.n_tokens, a.zero_tail = scale, T, out is None
    a.q_stride_t, a.q_stride_h = query.stride(0), query.stride(1)
    a.out_stride_t, a.out_stride_h = (Hq * D, D) if out is None else out.stride()[:2]
    if slots:
        a.k_stride_b, a.k_stride_h, a.k_stride_t = key.stride()[:3]
        a.v_stride_b, a.v_stride_h, a.v_stride_t = value.stride()[:3]
    else:
        a.k_stride_t, a.k_stride_h = key.stride()[:2]
        a.v_stride_t, a.v_stride_h = value.stride()[:2]
    if prefix:
        a.pk_stride_h, a.pk_stride_t = prefix_key.stride()[:2]
        a.pv_stride_h, a.pv_stride_t = prefix_value.stride()[:2]
        a.prefix_len = prefix_key.shape[1]
    need = ctypes.c_size_t(0)
    with torch.cuda.device(dev):
        L.check_call(L.lib().hokv_packed_attention_workspace_size(ctypes.byref(a), ctypes.byref(need)), "packed_attention")
    return a, need.value


_checked = L.Checked()


def _packed(what, query, key, value, cu_seqlens_q, cu_seqlens_k, kv_len, scaling, is_causal, out, prefix_key=None,
            prefix_value=None):
    """Check, take the output and this call's workspace from the allocator, launch on the current stream."""
    if cu_seqlens_k is None and kv_len is None:
        cu_seqlens_k = cu_seqlens_q
    # values, not objects: a tensor would be found again by its identity after it has changed
    scaling, is_causal = None if scaling is None else float(scaling), bool(is_causal)
    sig = L.signature
    geometry = (sig(query), sig(key), sig(value), cu_seqlens_q is not None and sig(cu_seqlens_q),
                cu_seqlens_k is not None and sig(cu_seqlens_k), kv_len is not None and sig(kv_len), scaling, is_causal,
                out is not None and sig(out), prefix_key is not None and (sig(prefix_key), sig(prefix_value)))
    known = _checked.get(geometry)
    if known is None:
        known = _checked.keep(geometry, _packed_check(query, key, value, cu_seqlens_q, cu_seqlens_k, kv_len, scaling,
                                                      is_causal, out, prefix_key, prefix_value))
    args, need = known
    if out is None:
        out = torch.empty_like(query, memory_format=torch.contiguous_format)
    if not args.n_tokens:
        return out
    a = L.PackedArgs.from_buffer_copy(args)
    ws = torch.empty(need, dtype=torch.uint8, device=query.device)
    a.q, a.k, a.v, a.out, a.workspace, a.workspace_bytes = (query.data_ptr(), key.data_ptr(), value.data_ptr(),
                                                            out.data_ptr(), ws.data_ptr(), need)
    if prefix_key is not None:
        a.prefix_k, a.prefix_v = prefix_key.data_ptr(), prefix_value.data_ptr()
    if cu_seqlens_q is not None:
        a.cu_seqlens_q = cu_seqlens_q.data_ptr()
    if kv_len is not None:
        a.kv_len = kv_len.data_ptr()
    else:
        a.cu_seqlens_k = cu_seqlens_k.data_ptr()
    status = L.call_on(geometry[0][3], L.lib().hokv_packed_attention, a)
    if status:
        L.check_call(status, what)   # strides that do not nest; addresses, which the signatures do not show
    return out


def packed_attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                     cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_k: Optional[torch.Tensor] = None,
                     kv_len: Optional[torch.Tensor] = None, scaling: Optional[float] = None, is_causal: bool = True,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(query key^T * scaling [causal]) value for every sequence of a packed batch.

    query [T, H_q, D]: sequence b owns tokens [cu_seqlens_q[b], cu_seqlens_q[b + 1]) (without cu_seqlens_q, token
    b).  key/value either packed [S, H_kv, D] with cu_seqlens_k [B + 1] (default: cu_seqlens_q) or in slots [B,
    H_kv, capacity, D] with kv_len [B], the keys each sequence holds, its new tokens included (a slot's rows behind
    kv_len are not used).  Lengths are int32 CUDA vectors and stay on the device.  Causal: query i of a sequence
    with n keys and m queries sits at position n - m + i; a query that sees no key gives zeros.  f16/bf16, head
    dims in multiples of 8 up to 128, contiguous head dims, strides in multiples of 8 elements, H_q a multiple of
    H_kv.  -> [T, H_q, D] in the query's dtype; rows of no sequence (ahead of the first, behind the last) are zeros,
    or left as they were in a given ``out`` (whose rows overlap neither each other nor the inputs)."""
    return _packed("packed_attention", query, key, value, cu_seqlens_q, cu_seqlens_k, kv_len, scaling, is_causal, out)
