"""Refusals of the packed-batch entry points that need no GPU: the Python checks
on CPU tensors, and the C ABI's argument checks, made before any device call."""

import ctypes

import pytest
import torch

from helix_online_kv import _lib as L


def _args(**kw):
    a = L.PackedArgs()
    a.dtype, a.n_seqs, a.q_heads, a.kv_heads, a.head_dim, a.causal, a.scale = L.BF16, 2, 8, 2, 64, 1, 0.125
    a.n_tokens, a.kv_rows, a.kv_in_slots = 2, 16, 1
    a.q = a.out = a.k = a.v = a.kv_len = 1 << 20   # never dereferenced: the checks fail first
    a.q_stride_t = a.out_stride_t = 512
    a.q_stride_h = a.out_stride_h = 64
    for n in "kv":
        setattr(a, n + "_stride_b", 2048)
        setattr(a, n + "_stride_h", 1024)
        setattr(a, n + "_stride_t", 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=L.F32), L.ERR_UNSUPPORTED, "dtype"),
    (dict(head_dim=132), L.ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=60), L.ERR_UNSUPPORTED, "head_dim"),
    (dict(q_heads=7), L.ERR_INVALID, "q_heads"),
    (dict(q_heads=258), L.ERR_UNSUPPORTED, "query heads per KV head"),
    (dict(scale=0.0), L.ERR_INVALID, "scale"),
    (dict(scale=float("nan")), L.ERR_INVALID, "scale"),
    (dict(n_tokens=-1), L.ERR_INVALID, "n_tokens"),
    (dict(n_tokens=3), L.ERR_INVALID, "one token"),
    (dict(q=None), L.ERR_INVALID, "null"),
    (dict(kv_len=None), L.ERR_INVALID, "key lengths"),
    (dict(k=None), L.ERR_INVALID, "null"),
    (dict(prefix_len=5), L.ERR_INVALID, "prefix"),
    (dict(k_stride_t=63), L.ERR_INVALID, "stride"),
    (dict(out=(1 << 20) + 8), L.ERR_INVALID, "aligned"),
    (dict(kv_in_slots=0), L.ERR_INVALID, "key lengths"),
])
def test_packed_attention_host_checks(kw, status, text):
    a = _args(**kw)
    assert L.lib().hokv_packed_attention(ctypes.byref(a), None) == status
    assert text in L.lib().hokv_last_error().decode()


def test_packed_attention_null_and_empty():
    assert L.lib().hokv_packed_attention(None, None) == L.ERR_INVALID
    assert L.lib().hokv_packed_attention_workspace_size(None, None) == L.ERR_INVALID
    a = _args(n_tokens=0, q=None)
    assert L.lib().hokv_packed_attention(ctypes.byref(a), None) == L.OK


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=L.U8), L.ERR_INVALID, "dtype"),
    (dict(head_dim=65), L.ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=258), L.ERR_UNSUPPORTED, "head_dim"),
    (dict(n_freq=33), L.ERR_INVALID, "frequencies"),
    (dict(eps=-1.0), L.ERR_INVALID, "eps"),
    (dict(kv_heads=0), L.ERR_INVALID, "kv_heads"),
    (dict(inv_freq=None), L.ERR_INVALID, "null"),
    (dict(k_slots=None), L.ERR_INVALID, "slots"),
    (dict(cu_seqlens=None, n_tokens=5), L.ERR_INVALID, "one token"),
])
def test_norm_rotate_host_checks(kw, status, text):
    a = L.NormRotateArgs()
    a.dtype, a.n_seqs, a.q_heads, a.kv_heads, a.head_dim, a.n_freq, a.eps, a.n_tokens = L.F16, 2, 8, 2, 64, 32, 1e-6, 4
    a.capacity = 8
    for n in ("q", "k", "v", "out", "k_slots", "v_slots", "kv_len", "inv_freq", "cu_seqlens"):
        setattr(a, n, 1 << 20)
    for k, v in kw.items():
        setattr(a, k, v)
    assert L.lib().hokv_norm_rotate_append(ctypes.byref(a), None) == status
    assert text in L.lib().hokv_last_error().decode()
    assert L.lib().hokv_norm_rotate_append(None, None) == L.ERR_INVALID


def test_python_refuses_cpu_tensors():
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    q, k = torch.zeros(4, 8, 64, dtype=torch.float16), torch.zeros(4, 2, 64, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        packed_attention(q, k, k, cu)
    with pytest.raises(ValueError, match="CUDA"):
        shared_prefix_attention(q, k.transpose(0, 1), k.transpose(0, 1), k, k, cu_seqlens_q=cu)
    with pytest.raises(ValueError, match="CUDA"):
        norm_rotate_append(q, k, k, k[None], k[None], cu, cu[1:], torch.ones(32))


@pytest.mark.gpu
def test_python_refusals():
    """Shapes, dtypes, strides and lengths that the entry points do not take; nothing is launched."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")   # noqa: E731
    q, k, cu = z(4, 8, 64), z(4, 2, 64), torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    slots, n1 = z(1, 2, 16, 64), cu[1:]
    bad = [
        (dict(query=q.float()), "queries"),
        (dict(query=q[0]), "queries"),
        (dict(key=k.bfloat16()), "key"),
        (dict(value=k[:3]), "value"),
        (dict(query=z(4, 7, 64)), "multiple"),
        (dict(query=z(4, 8, 60), key=z(4, 2, 60), value=z(4, 2, 60)), "head_dim"),
        (dict(query=z(4, 8, 136), key=z(4, 2, 136), value=z(4, 2, 136)), "head_dim"),
        (dict(cu_seqlens_q=cu.long()), "int32"),
        (dict(cu_seqlens_q=cu.cpu()), "int32"),
        (dict(cu_seqlens_q=None), "cu_seqlens"),
        (dict(cu_seqlens_q=torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), cu_seqlens_k=cu), "entries"),
        (dict(kv_len=n1), "kv_len"),
        (dict(key=slots, value=slots), "kv_len"),
        (dict(scaling=-1.0), "scaling"),
        (dict(scaling=float("nan")), "scaling"),
        (dict(query=z(4, 8, 128)[:, :, ::2]), "strides"),
        (dict(query=z(4, 8, 65)[:, :, :64]), "strides"),
        (dict(query=z(8, 4, 64).transpose(0, 1)), "token stride"),
        (dict(out=z(4, 8, 64, dtype=torch.bfloat16)), "out"),
        (dict(out=z(3, 8, 64)), "out"),
    ]
    for kw, text in bad:
        args = dict(query=q, key=k, value=k, cu_seqlens_q=cu)
        args.update(kw)
        with pytest.raises(ValueError, match=text):
            packed_attention(**args)
    off = z(4 * 8 * 64 + 8)[1:-7].view(4, 8, 64)   # rows that start between 16-byte boundaries
    with pytest.raises(ValueError, match="aligned"):
        packed_attention(off, k, k, cu)
    with pytest.raises(ValueError, match="one query"):
        packed_attention(q, slots, slots, kv_len=n1)
    for pk in (z(2, 9, 32), z(3, 9, 64), z(2, 9, 64, dtype=torch.bfloat16), z(9, 64), z(2, 9, 65)[:, :, :64]):
        with pytest.raises(ValueError, match="prefix_key"):
            shared_prefix_attention(q, pk, z(2, 9, 64), slots, slots, n1, cu)
    with pytest.raises(ValueError, match="prefix_value"):
        shared_prefix_attention(q, z(2, 9, 64), z(2, 8, 64), slots, slots, n1, cu)
    f = torch.ones(32, device="cuda")
    nra = dict(query=q, key=k, value=k, key_slots=slots, value_slots=slots, cu_seqlens=cu, kv_len=n1, inv_freq=f)
    for kw, text in [(dict(query=q.double()), "queries"), (dict(key=k[:3]), "key"), (dict(value=k.float()), "value"),
                     (dict(key_slots=slots[0]), "key_slots"), (dict(value_slots=slots[:, :, :8]), "value_slots"),
                     (dict(kv_len=cu), "kv_len"), (dict(cu_seqlens=n1), "cu_seqlens"), (dict(cu_seqlens=None), "one token"),
                     (dict(inv_freq=f.double()), "inv_freq"), (dict(inv_freq=torch.ones(33, device="cuda")), "inv_freq"),
                     (dict(q_weight=f), "q_weight"), (dict(k_weight=z(32)), "k_weight"), (dict(eps=float("inf")), "eps"),
                     (dict(positions=cu), "positions"), (dict(out=z(4, 8, 32)), "out"),
                     (dict(query=z(4, 8, 128)[:, :, ::2]), "contiguous")]:
        args = dict(nra)
        args.update(kw)
        with pytest.raises(ValueError, match=text):
            norm_rotate_append(**args)
    # nothing to do
    assert packed_attention(q[:0], k[:0], k[:0], cu[:1]).shape == (0, 8, 64)
    assert norm_rotate_append(q[:0], k[:0], k[:0], slots, slots, torch.zeros(2, dtype=torch.int32, device="cuda"), n1,
                              f).shape == (0, 8, 64)
