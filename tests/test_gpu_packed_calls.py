"""Calls of the packed-batch operators that the documentation allows, at the ends
of their ranges: head dims and groups, offsets above 2^31, views, another
stream's load, the first call of a process inside a capture."""

import os
import subprocess
import sys

import pytest
import torch

from packed_reference import lens_tensor, reference

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
HERE = os.path.dirname(os.path.abspath(__file__))


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _check(out, ref, tol):
    from helix_online_kv import _lib as L
    torch.cuda.synchronize()
    L.device_status()
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err.max()), float((err / tol).max()), bad.nonzero()[:3].tolist())


@pytest.mark.parametrize("D,Hq,Hkv", [(8, 4, 2), (16, 32, 1), (24, 6, 2), (56, 8, 8), (72, 4, 1), (104, 10, 2), (120, 8, 2),
                                      (64, 128, 1), (128, 64, 1), (128, 127, 1)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_head_dims_and_groups(D, Hq, Hkv, dtype):
    """Prompts, chunks and single tokens; outputs in a wider buffer whose other columns and heads stay."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(D + Hq)
    q, kv = [1, 70, 3, 0, 130], [1500, 70, 300, 9, 401]
    query = _randn(g, sum(q), Hq, D, dtype=dtype)
    k, v = _randn(g, sum(kv), Hkv, D, dtype=dtype), _randn(g, sum(kv), Hkv, D, dtype=dtype)
    buf = torch.full((sum(q) + 2, Hq + 1, D + 16), 7.0, dtype=dtype, device="cuda")
    out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv), out=buf[1:-1, :Hq, 8:D + 8])
    _check(out, *reference(query, q, k.split(kv), v.split(kv), D ** -0.5))
    out.fill_(7.0)
    assert (buf == 7).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_full_attention_behind_a_prefix(dtype):
    """is_causal=False: every query sees its sequence's own keys whole, too."""
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(2)
    q, kv, Hq, Hkv, D = [5, 1, 40], [300, 0, 129], 8, 2, 64
    query, pk, pv = _randn(g, sum(q), Hq, D, dtype=dtype), _randn(g, Hkv, 500, D, dtype=dtype), _randn(g, Hkv, 500, D, dtype=dtype)
    k, v = _randn(g, sum(kv), Hkv, D, dtype=dtype), _randn(g, sum(kv), Hkv, D, dtype=dtype)
    out = shared_prefix_attention(query, pk, pv, k, v, cu_seqlens_q=lens_tensor(q), cu_seqlens_k=lens_tensor(kv), is_causal=False)
    _check(out, *reference(query, q, k.split(kv), v.split(kv), D ** -0.5, False, (pk, pv)))


def test_slots_beyond_2_31_elements():
    """The last sequence's rows lie 2^31 elements into the slots: appended there, attended there, alone and behind a
    prefix; the rows around them stay."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(3)
    Hq, Hkv, D, cap, B = 8, 8, 128, 1 << 20, 3
    ks, vs = (torch.empty(B, Hkv, cap, D, dtype=BF16, device="cuda") for _ in range(2))
    assert ks.stride(0) * 2 >= 2 ** 31
    held, q = [300, 0, cap - 40], [1, 2, 30]
    kl = torch.tensor([300, 0, cap - 40], dtype=torch.int32, device="cuda")
    for s in (ks, vs):
        for b, n in enumerate(held):
            s[b, :, max(n - 500, 0):n + q[b]] = 3.0
            s[b, :, n + q[b]:n + q[b] + 5] = 5.0
    query, key, value = (_randn(g, sum(q), h, D, dtype=BF16) for h in (Hq, Hkv, Hkv))
    # no rotation, no norm: the rows are the projections themselves
    out = norm_rotate_append(query, key, value, ks, vs, lens_tensor(q), kl, torch.zeros(0, device="cuda"))
    assert torch.equal(out, query)
    at = 0
    for b, (n, m) in enumerate(zip(held, q)):
        assert torch.equal(ks[b, :, n:n + m].transpose(0, 1), key[at:at + m])
        assert torch.equal(vs[b, :, n:n + m].transpose(0, 1), value[at:at + m])
        assert (ks[b, :, n + m:n + m + 5] == 5).all() and (ks[b, :, max(n - 500, 0):n] == 3).all()
        at += m
    # attend the last thousand rows of the last slot, as slots of a view whose own offset is far
    tail_k, tail_v = ks[:, :, cap - 1010:cap - 10], vs[:, :, cap - 1010:cap - 10]
    tail_k[1:] = _randn(g, 2, Hkv, 1000, D, dtype=BF16)
    tail_v[1:] = _randn(g, 2, Hkv, 1000, D, dtype=BF16)
    lens = torch.tensor([0, 7, 1000], dtype=torch.int32, device="cuda")
    one = query[:3].contiguous()
    keys = [tail_k[b, :, :n].transpose(0, 1) for b, n in enumerate(lens.tolist())]
    values = [tail_v[b, :, :n].transpose(0, 1) for b, n in enumerate(lens.tolist())]
    _check(packed_attention(one, tail_k, tail_v, kv_len=lens), *reference(one, [1, 1, 1], keys, values, D ** -0.5))
    pk, pv = tail_k[2, :, 100:400], tail_v[2, :, 100:400]
    _check(shared_prefix_attention(one, pk, pv, tail_k, tail_v, lens),
           *reference(one, [1, 1, 1], keys, values, D ** -0.5, True, (pk, pv)))


def test_a_long_history_in_one_slot():
    """Key rows whose offset inside one head passes 2^31 elements."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(4)
    n, D = (1 << 24) + 777, 128
    k, v = torch.zeros(1, 1, n, D, dtype=F16, device="cuda"), torch.zeros(1, 1, n, D, dtype=F16, device="cuda")
    # all but the last rows score far below: the result is theirs
    k[..., 0] = -60.0
    k[0, 0, -300:] = _randn(g, 300, D, dtype=F16) * 0.25
    v[0, 0, -300:] = _randn(g, 300, D, dtype=F16)
    query = _randn(g, 3, 4, D, dtype=F16) * 0.25
    query[..., 0] = 4.0
    out = packed_attention(query, k, v, lens_tensor([3]), kv_len=torch.tensor([n], dtype=torch.int32, device="cuda"), scaling=1.0)
    ref, tol = reference(query, [3], [k[0, 0, -300:, None]], [v[0, 0, -300:, None]], 1.0)
    # a weight of e^-180 at most is left out of the reference; fp32 sums hold 300 keys that count
    _check(out, ref, tol)


def test_a_long_tail_of_unused_rows():
    """Rows behind the last sequence beyond 2^31 elements of the output: zeros, or left as they were."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(5)
    T, Hq, D = (1 << 19) + 5, 32, 128
    query = torch.ones(T, Hq, D, dtype=F16, device="cuda")
    query[:4] = _randn(g, 4, Hq, D, dtype=F16)
    k, v = _randn(g, 4, 8, D, dtype=F16), _randn(g, 4, 8, D, dtype=F16)
    q, cu = [3, 1], lens_tensor([3, 1])
    out = packed_attention(query, k, v, cu)
    _check(out[:4], *reference(query[:4], q, k.split(q), v.split(q), D ** -0.5))
    assert not out[4:].any()
    out.fill_(2.0)
    packed_attention(query, k, v, cu, out=out)
    assert (out[4:] == 2).all()
    key, ks = torch.ones(T, 1, D, dtype=F16, device="cuda"), torch.zeros(2, 1, 8, D, dtype=F16, device="cuda")
    f = torch.zeros(0, device="cuda")
    out = norm_rotate_append(query, key, key, ks, ks.clone(), cu, lens_tensor([0])[:2], f)
    assert torch.equal(out[:4], query[:4]) and not out[4:].any()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_from_and_to_views_off_16_byte_boundaries(dtype, interleaved):
    """The scalar form (views that start one element in) against the vector form: the same values but for the order of
    fp32 sums; negative positions among them."""
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(6)
    q, Hq, Hkv, D = [5, 0, 9], 4, 2, 64
    T = sum(q)
    wide = lambda *s: torch.full((*s[:-1], s[-1] + 2), 9.0, dtype=dtype, device="cuda")   # noqa: E731
    query, key, value = (_randn(g, T, h, D, dtype=dtype) for h in (Hq, Hkv, Hkv))
    w, f = 1 + 0.1 * _randn(g, D, dtype=dtype), 10000.0 ** (-torch.arange(32, device="cuda") / 32)
    pos = torch.randint(-3000, 3000, (T,), generator=g, device="cuda", dtype=torch.int32)
    kl = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    res = []
    for odd in (False, True):
        ts = []
        for t in (query, key, value):
            b = wide(*t.shape)
            x = b[..., 1:-1] if odd else t
            x.copy_(t)
            ts.append(x)
        kb, vb, ob = wide(3, Hkv, 12, D), wide(3, Hkv, 12, D), wide(T, Hq, D)
        ks, vs, out = ((b[..., 1:-1] if odd else b[..., 1:-1].contiguous()) for b in (kb, vb, ob))
        norm_rotate_append(*ts, ks, vs, lens_tensor(q), kl, f, w, w, 1e-5, interleaved, pos, out=out)
        if odd:
            for b in (kb, vb, ob):
                assert (b[..., 0] == 9).all() and (b[..., -1] == 9).all()
        res.append((out, ks, vs))
    assert torch.equal(res[0][2], res[1][2])
    for a, b in zip(res[0][:2], res[1][:2]):
        # half a step each, and some fp32 roundings (sum of 64 squares, products) of the pair's size
        size = a.double().abs() + a.double().abs().amax(-1, keepdim=True)
        assert ((a.double() - b.double()).abs() <= size * (torch.finfo(dtype).eps + 2.0 ** -18)).all()


def test_the_same_bits_beside_another_streams_work():
    """Cut items, joins and a prefix, ten times each while matrix products of another stream take SMs away."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(7)
    Hq, Hkv, D = 32, 8, 128
    a = _randn(g, 4096, 4096, dtype=BF16)
    side = torch.cuda.Stream()
    q, kv = [512, 1, 1, 700, 1], [4000, 5000, 77, 700, 12345]
    query = _randn(g, sum(q), Hq, D, dtype=BF16)
    k, v = _randn(g, sum(kv), Hkv, D, dtype=BF16), _randn(g, sum(kv), Hkv, D, dtype=BF16)
    pk, pv = _randn(g, Hkv, 9000, D, dtype=BF16), _randn(g, Hkv, 9000, D, dtype=BF16)
    cu_q, cu_k = lens_tensor(q), lens_tensor(kv)
    calls = (lambda: packed_attention(query, k, v, cu_q, cu_k),
             lambda: shared_prefix_attention(query[:64], pk, pv, k[:6400], v[:6400], cu_seqlens_q=lens_tensor([1] * 64),
                                             cu_seqlens_k=lens_tensor([100] * 64)))
    for call in calls:
        want = call()
        torch.cuda.synchronize()
        outs = []
        for _ in range(10):
            with torch.cuda.stream(side):
                b = a @ a
            outs.append(call())
        torch.cuda.synchronize()
        assert b.numel() and all(torch.equal(o, want) for o in outs)


def first_call_in_a_capture():
    """No call before the capture: kernels are loaded and configured inside it."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(8)
    x, k = _randn(g, 2, 4, 64, dtype=F16), _randn(g, 2, 2, 3000, 64, dtype=F16)
    kl, key, f = torch.tensor([2999, 40], dtype=torch.int32, device="cuda"), _randn(g, 2, 2, 64, dtype=F16), torch.ones(32, device="cuda")
    ks = torch.zeros(2, 2, 3001, 64, dtype=F16, device="cuda")
    call = lambda: (packed_attention(x, k, k, kv_len=kl), shared_prefix_attention(x, k[0], k[0], k, k, kl),   # noqa: E731
                    norm_rotate_append(x, key, key, ks, ks.clone(), None, kl, f))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, call()))


def test_the_first_call_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


if __name__ == "__main__":
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "helix-online-kv_b200"))
    first_call_in_a_capture()
