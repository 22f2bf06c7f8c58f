"""packed_attention and shared_prefix_attention against the plain 64-bit
reference: ragged prompts, chunks, single tokens, empty sequences, rows that see
nothing, odd groups and head dims, strided views, pieces of cut items, and what
may stand in masked places."""

import pytest
import torch

from packed_reference import lens_tensor, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _verify(out, ref, tol):
    from helix_online_kv import _lib as L
    torch.cuda.synchronize()
    L.device_status()
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err.max()), float((err / tol).max()), bad.nonzero()[:3].tolist())


def _slots(g, kv, Hkv, D, dtype, cap=None, stale=float("nan")):
    """Slots [B, H_kv, cap, D]; everything behind a sequence's keys is `stale`."""
    cap = cap or max(kv) + 5
    k = torch.full((len(kv), Hkv, cap, D), stale, dtype=dtype, device="cuda")
    v = k.clone()
    for b, n in enumerate(kv):
        k[b, :, :n] = _randn(g, Hkv, n, D, dtype=dtype)
        v[b, :, :n] = _randn(g, Hkv, n, D, dtype=dtype)
    return k, v, torch.tensor(kv, dtype=torch.int32, device="cuda")


CASES = [
    # q_lens, kv_lens, Hq, Hkv, D, dtype, causal
    ([1], [1], 1, 1, 64, F16, True),
    ([1], [130], 8, 2, 128, BF16, True),
    ([5, 1, 300, 0, 129], [5, 77, 300, 40, 513], 8, 2, 128, BF16, True),
    ([128, 256, 127, 129], [128, 256, 127, 129], 4, 4, 64, F16, True),
    ([700], [700], 32, 4, 64, F16, True),              # 8 heads a group
    ([33, 2], [1000, 2], 14, 2, 128, F16, True),       # 7 heads a group: 18 tokens, 126 rows of a tile
    ([9, 200], [9, 200], 6, 2, 96, BF16, True),        # head dim 96, groups of 3
    ([3, 50], [300, 50], 5, 1, 40, F16, True),         # head dim 40
    ([4, 1], [260, 3], 96, 1, 64, F16, True),          # one KV head, 96 query heads: one token a tile
    ([64, 7], [300, 1000], 8, 8, 128, BF16, False),    # full attention
    ([10, 300], [4, 290], 4, 2, 64, F16, True),        # more queries than keys: the first rows see nothing
    ([3, 0, 2], [0, 5, 0], 4, 2, 64, BF16, True),      # sequences without keys, one without queries
    ([1] * 40, [1 + 29 * i % 701 for i in range(40)], 8, 2, 64, F16, True),
]


@pytest.mark.parametrize("layout", ["packed", "slots"])
@pytest.mark.parametrize("q,kv,Hq,Hkv,D,dtype,causal", CASES)
def test_matches_reference(q, kv, Hq, Hkv, D, dtype, causal, layout):
    from helix_online_kv.prefill import packed_attention
    g = _gen(sum(q) * 7 + sum(kv) + D)
    query = _randn(g, sum(q), Hq, D, dtype=dtype)
    if layout == "slots":
        k, v, kl = _slots(g, kv, Hkv, D, dtype)
        keys, values = [k[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], [v[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)]
        out = packed_attention(query, k, v, lens_tensor(q), kv_len=kl, is_causal=causal)
    else:
        k, v = (_randn(g, sum(kv), Hkv, D, dtype=dtype) for _ in range(2))
        keys, values = k.split(kv), v.split(kv)
        out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv), is_causal=causal)
    _verify(out, *reference(query, q, keys, values, D ** -0.5, causal))


@pytest.mark.parametrize("q,kv,Hq,Hkv,D,dtype", [
    ([1], [9000], 8, 2, 128, BF16),             # one token over every CTA
    ([1, 1, 1], [5000, 1, 12345], 32, 4, 64, F16),
    ([2048, 1], [2048, 3000], 8, 2, 128, BF16),  # causal items cut between CTAs
    ([50, 3], [7000, 6001], 8, 1, 128, F16),     # two-tile items with long histories
])
def test_cut_items(q, kv, Hq, Hkv, D, dtype):
    from helix_online_kv.prefill import packed_attention
    g = _gen(sum(kv))
    query = _randn(g, sum(q), Hq, D, dtype=dtype)
    k, v, kl = _slots(g, kv, Hkv, D, dtype, stale=float("inf"))
    out = packed_attention(query, k, v, lens_tensor(q), kv_len=kl)
    again = packed_attention(query, k, v, lens_tensor(q), kv_len=kl)
    assert torch.equal(out, again)
    keys, values = [k[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], [v[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)]
    _verify(out, *reference(query, q, keys, values, D ** -0.5))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_growing_and_large_scores(dtype):
    """Each row's maximum rises from tile to tile past the lazy-rescaling step; scores of a few hundred."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(11)
    q, Hq, Hkv, D = [1500, 1], 4, 2, 64
    kv = [1500, 2000]
    query = _randn(g, sum(q), Hq, D, dtype=dtype, scale=2.0)
    ramp = torch.cat([torch.linspace(0.1, 6.0, n, device="cuda") for n in kv])[:, None, None]
    k = (torch.randn((sum(kv), Hkv, D), generator=g, device="cuda") * ramp).to(dtype)
    v = _randn(g, sum(kv), Hkv, D, dtype=dtype)
    out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv))
    _verify(out, *reference(query, q, k.split(kv), v.split(kv), D ** -0.5))


def test_neighbours_stay_out():
    """Queries, keys and values of other sequences, NaN and infinities among them, share tiles but not results."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(5)
    q, Hq, Hkv, D = [70, 30, 90], 4, 2, 128
    query = _randn(g, 190, Hq, D, dtype=BF16)
    k, v = _randn(g, 190, Hkv, D, dtype=BF16), _randn(g, 190, Hkv, D, dtype=BF16)
    clean = packed_attention(query, k, v, lens_tensor(q))
    query[70:100], k[70:100], v[70:100] = float("nan"), float("inf"), float("nan")
    dirty = packed_attention(query, k, v, lens_tensor(q))
    assert torch.equal(clean[:70], dirty[:70]) and torch.equal(clean[100:], dirty[100:])
    assert dirty[70:100].isnan().all()
    ref, tol = reference(torch.cat((query[:70], query[100:])), [70, 90], [k[:70], k[100:]], [v[:70], v[100:]], D ** -0.5)
    _verify(torch.cat((dirty[:70], dirty[100:])), ref, tol)


def test_strided_views_and_given_out():
    """Queries, keys and values as parts of one projection; out a view whose rows behind the last sequence stay."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(6)
    q, Hq, Hkv, D = [40, 100], 8, 2, 64
    qkv = _randn(g, 150, Hq + 2 * Hkv, D, dtype=F16)
    buf = torch.full((150, Hq + 3, D + 8), 7.0, dtype=F16, device="cuda")
    out = buf[:, :Hq, :D]
    query, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    got = packed_attention(query, k, v, lens_tensor(q), out=out)
    assert got is out
    ref, tol = reference(query[:140], q, k[:140].split(q), v[:140].split(q), D ** -0.5)
    _verify(out[:140], ref, tol)
    assert (out[140:] == 7).all() and (buf[:, Hq:] == 7).all() and (buf[:, :, D:] == 7).all()
    fresh = packed_attention(query, k, v, lens_tensor(q))
    assert torch.equal(fresh[:140], out[:140]) and (fresh[140:] == 0).all()


def test_store_tiers_without_starts():
    """One query each against a CDC-03 store's layer (slots), no cu_seqlens_q."""
    from helix_online_kv.cdc03 import CDC03Store
    from helix_online_kv.prefill import packed_attention
    g = _gen(8)
    st = CDC03Store(3, 2, 2, 64, 640, n_subspaces=8, dtype=F16)
    kv = [640, 17, 0]
    for b, n in enumerate(kv):
        st.k[1, b, :, :n] = _randn(g, 2, n, 64, dtype=F16)
        st.v[1, b, :, :n] = _randn(g, 2, n, 64, dtype=F16)
    st.seq_len.copy_(torch.tensor(kv, dtype=torch.int32))
    query = _randn(g, 3, 8, 64, dtype=F16)
    out = packed_attention(query, st.k[1], st.v[1], kv_len=st.seq_len)
    _verify(out, *reference(query, [1, 1, 1], [st.k[1, b, :, :n].transpose(0, 1) for b, n in enumerate(kv)],
                            [st.v[1, b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], 64 ** -0.5))


def test_graph_replay_with_new_lengths():
    """A captured call follows the lengths and data its tensors hold at replay."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(9)
    Hq, Hkv, D, cap = 8, 2, 64, 3000
    k, v, kl = _slots(g, [100, 200], Hkv, D, F16, cap, stale=0.5)
    query = _randn(g, 20, Hq, D, dtype=F16)
    cu = lens_tensor([10, 10])
    packed_attention(query, k, v, cu, kv_len=kl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = packed_attention(query, k, v, cu, kv_len=kl)
    for q, kv in (([10, 10], [100, 200]), ([1, 19], [2900, 1900]), ([20, 0], [20, 0])):
        cu.copy_(lens_tensor(q))
        kl.copy_(torch.tensor(kv, dtype=torch.int32))
        query.copy_(_randn(g, 20, Hq, D, dtype=F16))
        graph.replay()
        _verify(out, *reference(query, q, [k[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)],
                                [v[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], D ** -0.5))


def test_two_streams_at_once():
    """Calls on two streams have workspaces of their own."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(10)
    query = _randn(g, 2, 8, 128, dtype=BF16)
    k, v, kl = _slots(g, [9000, 7000], 2, 128, BF16)
    alone = packed_attention(query, k, v, kv_len=kl)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(packed_attention(query, k, v, kv_len=kl))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone) for o in outs)


def test_lengths_that_do_not_fit_are_reported():
    """The device status names them; the other sequences and the memory around stay right."""
    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    g = _gen(12)
    query = _randn(g, 6, 4, 64, dtype=F16)
    k, v, kl = _slots(g, [50, 60, 70], 2, 64, F16, cap=80)
    good = packed_attention(query, k, v, lens_tensor([2, 2, 2]), kv_len=kl)
    kl[1] = 81
    out = packed_attention(query, k, v, lens_tensor([2, 2, 2]), kv_len=kl)
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_DEVICE_INPUT
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])


SHARED = [
    # prefix, q_lens, kv_lens, Hq, Hkv, D, dtype
    (200, [3, 3], [90, 11], 32, 8, 128, BF16),
    (1, [1], [1], 2, 1, 64, F16),
    (128, [1, 1, 1], [1, 128, 129], 8, 2, 64, F16),
    (9000, [1, 1], [40, 300], 32, 4, 64, F16),                   # the prefix cut over the CTAs
    (5000, [1] * 70, [1 + 37 * i % 509 for i in range(70)], 8, 2, 128, BF16),   # more rows than one pair of tiles
    (300, [2, 1, 0, 5], [2, 0, 9, 3], 6, 2, 96, BF16),           # no own keys; more queries than own keys
    (1000, [4, 2], [3000, 70], 14, 2, 128, F16),                 # own parts cut too
]


@pytest.mark.parametrize("layout", ["slots", "packed"])
@pytest.mark.parametrize("P,q,kv,Hq,Hkv,D,dtype", SHARED)
def test_shared_prefix_matches_reference(P, q, kv, Hq, Hkv, D, dtype, layout):
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(P + sum(kv))
    query = _randn(g, sum(q), Hq, D, dtype=dtype)
    pk, pv = _randn(g, Hkv, P, D, dtype=dtype), _randn(g, Hkv, P, D, dtype=dtype)
    if layout == "slots":
        k, v, kl = _slots(g, kv, Hkv, D, dtype)
        keys, values = [k[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], [v[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)]
        out = shared_prefix_attention(query, pk, pv, k, v, kl, lens_tensor(q))
    else:
        k, v = (_randn(g, sum(kv), Hkv, D, dtype=dtype) for _ in range(2))
        keys, values = k.split(kv), v.split(kv)
        out = shared_prefix_attention(query, pk, pv, k, v, cu_seqlens_q=lens_tensor(q), cu_seqlens_k=lens_tensor(kv))
    _verify(out, *reference(query, q, keys, values, D ** -0.5, True, (pk, pv)))


def test_shared_prefix_of_another_store_and_no_prefix():
    """The prefix as a view of a store's slot (strided); an empty prefix is packed_attention."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(21)
    big = _randn(g, 2, 1, 2, 700, 64, dtype=F16)
    k, v, kl = _slots(g, [30, 600], 2, 64, F16)
    query = _randn(g, 2, 8, 64, dtype=F16)
    keys, values = [k[b, :, :n].transpose(0, 1) for b, n in enumerate([30, 600])], [v[b, :, :n].transpose(0, 1) for b, n in enumerate([30, 600])]
    pk, pv = big[0, 0, :, :333], big[1, 0, :, :333]
    out = shared_prefix_attention(query, pk, pv, k, v, kl)
    _verify(out, *reference(query, [1, 1], keys, values, 64 ** -0.5, True, (pk, pv)))
    none = shared_prefix_attention(query, pk[:, :0], pv[:, :0], k, v, kl)
    assert torch.equal(none, packed_attention(query, k, v, kv_len=kl))


def test_no_sequences_and_no_keys():
    """A batch of no sequences, tensors without rows: nothing to attend, zeros behind the last sequence."""
    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.shared_prefix import shared_prefix_attention
    z = lambda *s: torch.zeros(s, dtype=F16, device="cuda")   # noqa: E731
    query = torch.ones(3, 4, 64, dtype=F16, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert (packed_attention(query, z(0, 2, 64), z(0, 2, 64), lens_tensor([]), lens_tensor([])) == 0).all()
    assert (packed_attention(query, z(0, 2, 8, 64), z(0, 2, 8, 64), lens_tensor([]), kv_len=none) == 0).all()
    assert (packed_attention(query, z(0, 2, 64), z(0, 2, 64), lens_tensor([1, 2]), lens_tensor([0, 0])) == 0).all()
    assert (packed_attention(query, z(2, 2, 0, 64), z(2, 2, 0, 64), lens_tensor([1, 2]), kv_len=lens_tensor([0])) == 0).all()
    # only the prefix to see
    g = _gen(31)
    pk, pv = _randn(g, 2, 200, 64, dtype=F16), _randn(g, 2, 200, 64, dtype=F16)
    query = _randn(g, 3, 4, 64, dtype=F16)
    out = shared_prefix_attention(query, pk, pv, z(0, 2, 64), z(0, 2, 64), cu_seqlens_q=lens_tensor([1, 2]),
                                  cu_seqlens_k=lens_tensor([0, 0]))
    empty = [torch.zeros(0, 2, 64, dtype=F16, device="cuda")] * 2
    _verify(out, *reference(query, [1, 2], empty, empty, 64 ** -0.5, True, (pk, pv)))
    torch.cuda.synchronize()
    L.device_status()


@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (6, 2)])
def test_outputs_in_any_layout(Hq, Hkv):
    """out as a transposed view (heads outside tokens) and with rows off 32-byte boundaries."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(32)
    q, D = [300, 5], 64
    query, k, v = _randn(g, 305, Hq, D, dtype=BF16), _randn(g, 305, Hkv, D, dtype=BF16), _randn(g, 305, Hkv, D, dtype=BF16)
    want = packed_attention(query, k, v, lens_tensor(q))
    out = torch.full((Hq, 305, D), 3.0, dtype=BF16, device="cuda").transpose(0, 1)
    assert torch.equal(packed_attention(query, k, v, lens_tensor(q), out=out), want)
    wide = torch.full((305, Hq, D + 8), 3.0, dtype=BF16, device="cuda")
    assert torch.equal(packed_attention(query, k, v, lens_tensor(q), out=wide[:, :, 8:]), want)
    assert (wide[:, :, :8] == 3).all()
    # values with strides of their own, and slots whose heads lie outside the batch
    k4 = torch.empty(Hkv, 2, 320, D, dtype=BF16, device="cuda").fill_(float("nan")).transpose(0, 1)
    v4 = torch.empty(2, 320, Hkv, D, dtype=BF16, device="cuda").fill_(float("nan")).transpose(1, 2)
    for b, (a, n) in enumerate(((0, 300), (300, 5))):
        k4[b, :, :n], v4[b, :, :n] = k[a:a + n].transpose(0, 1), v[a:a + n].transpose(0, 1)
    assert torch.equal(packed_attention(query, k4, v4, lens_tensor(q), kv_len=torch.tensor(q, dtype=torch.int32, device="cuda")), want)


def test_many_short_sequences_and_long_tables():
    """More sequences than the schedule's lanes hold one each; items of one key tile share the slots in turn."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(33)
    kv = [1 + (i * 37) % 190 for i in range(700)]
    q = [0 if i % 13 == 5 else 1 + (i % 7 == 3) for i in range(700)]
    q = [min(a, b) for a, b in zip(q, kv)]
    query = _randn(g, sum(q), 4, 128, dtype=BF16)
    k, v = _randn(g, sum(kv), 1, 128, dtype=BF16), _randn(g, sum(kv), 1, 128, dtype=BF16)
    out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv))
    _verify(out, *reference(query, q, k.split(kv), v.split(kv), 128 ** -0.5))


def test_one_and_two_tile_items_in_turn():
    """Single tokens, prompts and short chunks one after the other: each CTA changes between the item forms."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(34)
    q = [1, 65, 1, 1, 33, 200, 1, 32, 3, 64, 1, 97] * 12
    kv = [n + (i * 113) % 700 for i, n in enumerate(q)]
    for D, dtype in ((128, F16), (64, BF16)):
        query = _randn(g, sum(q), 8, D, dtype=dtype)
        k, v = _randn(g, sum(kv), 2, D, dtype=dtype), _randn(g, sum(kv), 2, D, dtype=dtype)
        out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv))
        _verify(out, *reference(query, q, k.split(kv), v.split(kv), D ** -0.5))


def test_non_finite_scores_propagate():
    """A NaN or infinite score of a key that a row sees makes that row NaN, as the formula does, also where the running
    maximum was taken before; other rows of the tile stay right."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(35)
    for D in (64, 128):
        query = _randn(g, 300, 2, D, dtype=BF16)
        k, v = _randn(g, 300, 2, D, dtype=BF16), _randn(g, 300, 2, D, dtype=BF16)
        clean = packed_attention(query, k, v, lens_tensor([300]))
        k2 = k.clone()
        k2[250, 0, 3] = float("nan")
        k2[270, 1] = float("inf")
        out = packed_attention(query, k2, v, lens_tensor([300]))
        assert torch.equal(out[:250, 0], clean[:250, 0]) and out[250:, 0].isnan().all()
        assert torch.equal(out[:270, 1], clean[:270, 1]) and out[270:, 1].isnan().all()


def test_shared_prefix_in_a_graph_and_on_two_streams():
    """Both launches captured and replayed with other lengths; eager calls on two streams at once."""
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(41)
    Hq, Hkv, D, P = 8, 2, 128, 3000
    k, v, kl = _slots(g, [700, 90, 1], Hkv, D, BF16, 2100, stale=0.25)
    pk, pv = _randn(g, Hkv, P, D, dtype=BF16), _randn(g, Hkv, P, D, dtype=BF16)
    query, cu = _randn(g, 6, Hq, D, dtype=BF16), lens_tensor([2, 3, 1])
    call = lambda: shared_prefix_attention(query, pk, pv, k, v, kl, cu)   # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for q, kv in (([2, 3, 1], [700, 90, 1]), ([1, 1, 4], [5, 2000, 130]), ([6, 0, 0], [6, 0, 40])):
        cu.copy_(lens_tensor(q))
        kl.copy_(torch.tensor(kv, dtype=torch.int32))
        query.copy_(_randn(g, 6, Hq, D, dtype=BF16))
        graph.replay()
        _verify(out, *reference(query, q, [k[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)],
                                [v[b, :, :n].transpose(0, 1) for b, n in enumerate(kv)], D ** -0.5, True, (pk, pv)))
    alone = call()
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone) for o in outs)


def test_two_graphs_and_replays_of_cut_items():
    """Two captured calls whose items are cut between CTAs, replayed in turn many times: every replay starts from
    clean marks of its own workspace."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(42)
    k, v, kl = _slots(g, [9000, 12000], 2, 64, F16)
    q1, q2 = _randn(g, 2, 8, 64, dtype=F16), _randn(g, 2, 8, 64, dtype=F16)
    w1, w2 = packed_attention(q1, k, v, kv_len=kl), packed_attention(q2, k, v, kv_len=kl)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in (q1, q2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(packed_attention(q, k, v, kv_len=kl))
    for _ in range(20):
        for graph, o in zip(graphs, outs):
            o.zero_()
            graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], w1) and torch.equal(outs[1], w2)


def test_workspace_contents_do_not_matter():
    """The C entry point on a workspace full of ones, NaN patterns, and what the call before left there."""
    import ctypes

    from helix_online_kv import _lib as L
    from helix_online_kv import prefill as F
    g = _gen(43)
    k, v, kl = _slots(g, [9000, 40, 3000], 2, 128, BF16)
    query = _randn(g, 3, 8, 128, dtype=BF16)
    want = F.packed_attention(query, k, v, kv_len=kl)
    args, need = F._packed_check(query, k, v, None, None, kl, None, True, None, None, None)
    a = L.PackedArgs.from_buffer_copy(args)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.empty_like(query)
    a.q, a.k, a.v, a.out, a.kv_len = query.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), kl.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    for fill in (1, 255, None, None):
        if fill is not None:
            ws.fill_(fill)
        out.zero_()
        L.check(L.lib().hokv_packed_attention(ctypes.byref(a), L.stream()))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    a.workspace_bytes = need - 1
    assert L.lib().hokv_packed_attention(ctypes.byref(a), L.stream()) == L.ERR_WORKSPACE


def test_bad_lengths_behind_a_prefix():
    """A slot longer than its capacity, starts outside the batch: reported, without waiting; later calls are unharmed."""
    import time

    from helix_online_kv import _lib as L
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(44)
    k, v, kl = _slots(g, [50, 60, 70], 2, 64, F16, cap=80)
    pk, pv = _randn(g, 2, 300, 64, dtype=F16), _randn(g, 2, 300, 64, dtype=F16)
    query, cu = _randn(g, 6, 4, 64, dtype=F16), lens_tensor([2, 2, 2])
    good = shared_prefix_attention(query, pk, pv, k, v, kl, cu)
    torch.cuda.synchronize()
    kl[1] = 81
    out = shared_prefix_attention(query, pk, pv, k, v, kl, cu)
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_DEVICE_INPUT
    assert torch.equal(out[:2], good[:2]) and torch.equal(out[4:], good[4:])
    kl[1] = 60
    cu[1] = 9
    t = time.time()
    shared_prefix_attention(query, pk, pv, k, v, kl, cu)
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_DEVICE_INPUT and time.time() - t < 1
    cu.copy_(lens_tensor([2, 2, 2]))
    assert torch.equal(shared_prefix_attention(query, pk, pv, k, v, kl, cu), good)


def test_many_pairs_behind_a_prefix():
    """Many whole and cut prefix items a CTA: 300 sequences of up to three tokens behind prefixes of 40 and 2,000."""
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(45)
    q = [1 + i % 3 for i in range(300)]
    kv = [max(n, (i * 61) % 400) for i, n in enumerate(q)]
    kv[7], q[7] = 9000, 3   # one own part cut over CTAs
    query = _randn(g, sum(q), 8, 64, dtype=F16)
    k, v = _randn(g, sum(kv), 2, 64, dtype=F16), _randn(g, sum(kv), 2, 64, dtype=F16)
    for P in (40, 2000):
        pk, pv = _randn(g, 2, P, 64, dtype=F16), _randn(g, 2, P, 64, dtype=F16)
        out = shared_prefix_attention(query, pk, pv, k, v, cu_seqlens_q=lens_tensor(q), cu_seqlens_k=lens_tensor(kv))
        _verify(out, *reference(query, q, k.split(kv), v.split(kv), 64 ** -0.5, True, (pk, pv)))
