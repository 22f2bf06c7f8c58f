"""norm_rotate_append against the formula in 64 bits, and a ragged batch's steps
through a CDC-03 store: append, attention, codes of the aged tokens, decoding
behind a shared prefix."""

import pytest
import torch

from packed_reference import lens_tensor, reference

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _freqs(n, base=10000.0):
    return (base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().cuda()


def _turned(x, weight, place, inv_freq, eps, interleaved):
    """The formula in 64 bits and its tolerance: half a step of the output, and for the fp32 arithmetic before it
    (sum of D squares: D / 2 roundings in the root, twelve more in products, cosine and sine; the angle in turns is
    rounded to fp32, 2^-24 pi) (D / 2 + 24) 2^-24 of the pair's size."""
    D, F = x.shape[-1], inv_freq.shape[0]
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    ang = place.double()[:, None, None] * inv_freq.double()
    c, s = ang.cos(), ang.sin()
    ia = torch.arange(F, device="cuda") * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else F)
    out, size = y.clone(), y.abs()
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = a.abs() + b.abs()
    fi = torch.finfo(x.dtype)
    return out, out.abs() * fi.eps / 2 + size * (D / 2 + 24) * 2.0 ** -24 + fi.smallest_normal * fi.eps


def _close(got, ref, tol):
    err = (got.double() - ref).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


CASES = [
    # q_lens, kv_lens, Hq, Hkv, D, F, dtype, norm, interleaved
    ([1], [0], 1, 1, 64, 32, F16, True, False),
    ([5, 0, 130, 1], [7, 3, 0, 1000], 32, 8, 128, 64, BF16, True, False),
    ([5, 0, 130, 1], [7, 3, 0, 1000], 4, 4, 64, 16, F16, False, True),
    ([40, 3], [0, 9], 6, 2, 96, 48, BF16, True, False),
    ([40, 3], [0, 9], 6, 2, 80, 24, F16, True, False),     # 5 of 8 lanes, 32 dims pass through
    ([40, 3], [0, 9], 5, 1, 256, 128, F16, True, True),
    ([17], [300], 8, 2, 64, 20, F16, True, False),         # halves of 20 dims: scalar form
    ([17], [300], 8, 2, 64, 20, BF16, True, True),
    ([17], [300], 3, 1, 40, 20, F32, True, False),         # scalar form
    ([17, 2], [300, 0], 3, 1, 64, 32, F32, True, False),
    ([9], [0], 2, 2, 128, 0, F16, True, False),            # no rotation
    ([9], [4], 2, 2, 250, 125, F32, False, True),
    ([1] * 50, list(range(50)), 8, 2, 128, 64, BF16, True, False),
    ([3000], [0], 32, 8, 128, 64, BF16, True, False),      # several heads a group
]


@pytest.mark.parametrize("q,kv,Hq,Hkv,D,F,dtype,norm,interleaved", CASES)
def test_matches_formula(q, kv, Hq, Hkv, D, F, dtype, norm, interleaved):
    from helix_online_kv import _lib as L
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(sum(q) + D + F)
    T, B, cap = sum(q), len(q), max(a + b for a, b in zip(q, kv)) + 3
    qkv = _randn(g, T, Hq + 2 * Hkv, D, dtype=dtype)
    query, key, value = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    ks, vs = torch.full((B, Hkv, cap, D), 3.0, dtype=dtype, device="cuda"), torch.full((B, Hkv, cap, D), 3.0, dtype=dtype, device="cuda")
    qw, kw = (1 + 0.3 * _randn(g, D, dtype=dtype), 1 + 0.3 * _randn(g, D, dtype=dtype)) if norm else (None, None)
    kl, f = torch.tensor(kv, dtype=torch.int32, device="cuda"), _freqs(F)
    out = norm_rotate_append(query, key, value, ks, vs, lens_tensor(q), kl, f, qw, kw, 1e-5, interleaved)
    torch.cuda.synchronize()
    L.device_status()
    place = torch.cat([torch.arange(n, n + m) for n, m in zip(kv, q)]).cuda()
    _close(out, *_turned(query, qw, place, f, 1e-5, interleaved))
    want, tol = _turned(key, kw, place, f, 1e-5, interleaved)
    t = 0
    for b, (n, m) in enumerate(zip(kv, q)):
        _close(ks[b, :, n:n + m].transpose(0, 1), want[t:t + m], tol[t:t + m])
        assert torch.equal(vs[b, :, n:n + m].transpose(0, 1), value[t:t + m])
        for s in (ks, vs):   # the rows before and behind stay
            assert (s[b, :, :n] == 3).all() and (s[b, :, n + m:] == 3).all()
        t += m


def test_far_positions():
    """Positions of a million: an fp32 angle would be off by hundredths of a radian."""
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(3)
    query, key = _randn(g, 4, 2, 64, dtype=F32), _randn(g, 4, 1, 64, dtype=F32)
    pos = torch.tensor([1 << 20, 999983, 2 ** 31 - 1, 0], dtype=torch.int32, device="cuda")
    ks, vs, f = torch.zeros(1, 1, 8, 64, device="cuda"), torch.zeros(1, 1, 8, 64, device="cuda"), _freqs(32, 500000.0)
    out = norm_rotate_append(query, key, key, ks, vs, lens_tensor([4]), lens_tensor([]), f, positions=pos)
    _close(out, *_turned(query, None, pos, f, 0.0, False))
    _close(ks[0, :, :4].transpose(0, 1), *_turned(key, None, pos, f, 0.0, False))


@pytest.mark.parametrize("D", [64, 36])
def test_in_place_tail_and_one_token_each(D):
    """out = the query itself; rows behind the last sequence; no cu_seqlens."""
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(4)
    query, key = _randn(g, 7, 4, D, dtype=F16), _randn(g, 7, 2, D, dtype=F16)
    w, f = 1 + _randn(g, D, dtype=F16) * 0.1, _freqs(D // 2)
    kl = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    new = lambda: torch.zeros(2, 2, 12, D, dtype=F16, device="cuda")   # noqa: E731
    ks, vs = new(), new()
    out = norm_rotate_append(query, key, key, ks, vs, lens_tensor([2, 3]), kl, f, w, w)
    assert (out[5:] == 0).all()
    mine, ks2, vs2 = query.clone(), new(), new()
    assert norm_rotate_append(mine, key, key, ks2, vs2, lens_tensor([2, 3]), kl, f, w, w, out=mine) is mine
    assert torch.equal(mine[:5], out[:5]) and torch.equal(mine[5:], query[5:])
    assert torch.equal(ks, ks2) and torch.equal(vs, vs2)
    one = norm_rotate_append(query[:2], key[:2], key[:2], new(), new(), None, kl, f, w, w)
    two = norm_rotate_append(query[:2], key[:2], key[:2], new(), new(), lens_tensor([1, 1]), kl, f, w, w)
    assert torch.equal(one, two)


def test_rows_that_do_not_fit_are_reported():
    from helix_online_kv import _lib as L
    from helix_online_kv.rotary import norm_rotate_append
    g = _gen(5)
    x = _randn(g, 6, 1, 64, dtype=F16)
    big = torch.full((3, 1, 8, 64), 3.0, dtype=F16, device="cuda")
    ks, vs = big[:2, :, :4], big.clone()[:2, :, :4]
    norm_rotate_append(x, x, x, ks, vs, lens_tensor([3, 3]), torch.tensor([2, 1], dtype=torch.int32, device="cuda"),
                       _freqs(32))
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_DEVICE_INPUT
    assert torch.equal(vs[0, :, 2:4].transpose(0, 1), x[:2]) and torch.equal(vs[1, :, 1:4].transpose(0, 1), x[3:])
    assert (big[:, :, 4:] == 3).all() and (big[2] == 3).all() and (big[0, :, :2] == 3).all()


def test_steps_of_a_ragged_batch_through_a_store():
    """Prompts of three lengths, a mixed step, then a decode step behind a shared prefix: each step's attention
    against the 64-bit reference on the rows the store holds, the codes against one assignment of the whole."""
    from helix_online_kv.cdc03 import CDC03Store
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(6)
    Hq, H, D, hot = 8, 2, 64, 64
    st = CDC03Store(3, 1, H, D, 800, n_subspaces=8, dtype=F16)
    f, w = _freqs(32), (1 + 0.1 * _randn(g, D, dtype=F16))
    held, keys, scale = [0, 0, 0], [torch.zeros(0, H, D, device="cuda")] * 3, D ** -0.5
    for step, q in enumerate(([400, 150, 257], [1, 300, 1], [1, 1, 1])):
        cu = lens_tensor(q)
        qkv = _randn(g, sum(q), Hq + 2 * H, D, dtype=F16)
        query = st.append_packed(0, qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], cu, f, w, w)
        lens = st.lengths_after(cu)
        held = [a + b for a, b in zip(held, q)]
        own_k = [st.k[0, b, :, :n].transpose(0, 1) for b, n in enumerate(held)]
        own_v = [st.v[0, b, :, :n].transpose(0, 1) for b, n in enumerate(held)]
        out = st.attend_packed(0, query, cu, lens, scale)
        ref, tol = reference(query, q, own_k, own_v, scale)
        assert ((out.double() - ref).abs() <= tol).all()
        if step == 2:
            pk, pv = _randn(g, H, 1000, D, dtype=F16), _randn(g, H, 1000, D, dtype=F16)
            out = shared_prefix_attention(query, pk, pv, st.k[0], st.v[0], lens, cu, scaling=scale)
            ref, tol = reference(query, q, own_k, own_v, scale, True, (pk, pv))
            assert ((out.double() - ref).abs() <= tol).all()
        t = 0
        place = torch.cat([torch.arange(n - m, n) for n, m in zip(held, q)]).cuda()
        want, tol = _turned(qkv[:, Hq:Hq + H], w, place, f, 1e-6, False)
        for b, (n, m) in enumerate(zip(held, q)):
            _close(own_k[b][n - m:], want[t:t + m], tol[t:t + m])
            t += m
        if step == 0:
            st.calibrate(0, 128)
        st.advance(cu, hot)
        assert st.seq_len.tolist() == held
    codes = st.codes.clone()
    st.codes.zero_()
    st.age(0, torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([n - hot for n in held], device="cuda"))
    assert torch.equal(codes, st.codes) and codes.any()


def test_model_step_in_one_graph():
    """Append, attention and advance captured once, replayed as lengths grow."""
    from helix_online_kv.cdc03 import CDC03Store
    g = _gen(7)
    Hq, H, D = 8, 2, 64
    st = CDC03Store(2, 1, H, D, 400, n_subspaces=8, dtype=F16)
    st.k[0, :, :, :300] = _randn(g, 2, H, 300, D, dtype=F16)
    st.v[0, :, :, :300] = _randn(g, 2, H, 300, D, dtype=F16)
    st.seq_len.copy_(torch.tensor([300, 40], dtype=torch.int32))
    st.calibrate(0, 40)
    f, cu, qkv = _freqs(32), lens_tensor([1, 1]), _randn(g, 2, Hq + 2 * H, D, dtype=F16)

    def step():
        query = st.append_packed(0, qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], cu, f)
        out = st.attend_packed(0, query, cu, st.lengths_after(cu), D ** -0.5)
        st.advance(cu)
        return query, out

    state = {k: v.clone() for k, v in st.state_dict().items() if k != "geometry"}
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        query, out = step()
    for k, v in state.items():
        getattr(st, k).copy_(v)
    held = [300, 40]
    for _ in range(3):
        qkv.copy_(_randn(g, 2, Hq + 2 * H, D, dtype=F16))
        graph.replay()
        held = [n + 1 for n in held]
        assert st.seq_len.tolist() == held
        ref, tol = reference(query, [1, 1], [st.k[0, b, :, :n].transpose(0, 1) for b, n in enumerate(held)],
                             [st.v[0, b, :, :n].transpose(0, 1) for b, n in enumerate(held)], D ** -0.5)
        assert ((out.double() - ref).abs() <= tol).all()


def test_no_sequences():
    from helix_online_kv.rotary import norm_rotate_append
    x = torch.ones(3, 2, 64, dtype=F16, device="cuda")
    ks = torch.zeros(0, 2, 8, 64, dtype=F16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert (norm_rotate_append(x, x, x, ks, ks, lens_tensor([]), none, _freqs(32)) == 0).all()
