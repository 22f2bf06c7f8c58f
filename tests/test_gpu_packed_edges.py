"""packed_attention and shared_prefix_attention where a mistake hides from random
data: keys far below a row's largest score, scores of any finite size, starts, hidden
rows, and results that show the loss of a single key."""

import math

import pytest
import torch

from packed_reference import lens_tensor, reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _check(out, ref, tol):
    from helix_online_kv import _lib as L
    torch.cuda.synchronize()
    L.device_status()
    err = (out.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), float(err.max()), float((err / tol).max()), bad.nonzero()[:3].tolist())


def _far_tail(g, n, Hkv, D, gap, sinks, dtype):
    """Keys [n, H_kv, D] whose dim 0 holds the score in log2 units for a query with 1 there and scaling ln 2: `gap` for
    the keys in `sinks`, 0 for the others, whose weights then all round the same way; values 0 for the sinks, 0.5 to 1.5
    for the others."""
    k = torch.zeros(n, Hkv, D, device="cuda")
    v = torch.rand((n, Hkv, D), generator=g, device="cuda") + 0.5
    k[sinks, :, 0], v[sinks] = gap, 0.0
    return k.to(dtype), v.to(dtype)


def _tail_tolerance(tol, dtype, values):
    """Weights that the type holds below its normal range are off by up to half its smallest step, 2^-25 in f16, where a
    row's largest weight is stored as 2^11 at least: 2^-36 sum |V| of the result (bf16 has the range of fp32)."""
    if dtype == BF16:
        return tol
    return tol + 2.0 ** -36 * float(sum(v.double().abs().sum(0).max() for v in values))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q,kv,gap,sink", [
    ([1], [131072], 25.125, 0),      # one token over every CTA: a tail of 2^-25 each holds a thousandth of the mass
    ([1], [131072], 25.125, 131071),
    ([1], [16384], 17.5, 9000),
    ([1, 2], [1000, 900], 20.25, 5),  # whole items of one tile
    ([300], [300], 19.25, 0),        # two-tile items; rows that see few keys and many
    ([2048], [2048], 22.25, 0),
])
def test_keys_far_below_the_largest_score(q, kv, gap, sink, dtype):
    """A key that dominates its row (an attention sink) takes none of the others' values away."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(sum(kv))
    Hq, Hkv, D = 8, 2, 64
    sinks, at = [], 0
    for n in kv:
        sinks.append(at + min(sink, n - 1))
        at += n
    k, v = _far_tail(g, sum(kv), Hkv, D, gap, sinks, dtype)
    query = torch.zeros(sum(q), Hq, D, dtype=dtype, device="cuda")
    query[..., 0] = 1
    out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv), scaling=math.log(2.0))
    keys, values = k.split(kv), v.split(kv)
    ref, tol = reference(query, q, keys, values, math.log(2.0))
    _check(out, ref, _tail_tolerance(tol, dtype, values))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("P,sink", [(20000, 0), (20000, None), (700, 0)])
def test_keys_far_below_the_largest_score_behind_a_prefix(P, sink, dtype):
    """The same over the join of a prefix with own keys: the dominating key in the prefix, or among the own keys."""
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(P)
    Hq, Hkv, D, kv, q = 8, 2, 64, [3000, 40], [1, 3]
    pk, pv = _far_tail(g, P, Hkv, D, 21.25, [] if sink is None else [sink], dtype)
    k, v = _far_tail(g, sum(kv), Hkv, D, 21.25, [7, 3001] if sink is None else [], dtype)
    query = torch.zeros(sum(q), Hq, D, dtype=dtype, device="cuda")
    query[..., 0] = 1
    pk, pv = pk.transpose(0, 1), pv.transpose(0, 1)
    out = shared_prefix_attention(query, pk, pv, k, v, cu_seqlens_q=lens_tensor(q), cu_seqlens_k=lens_tensor(kv),
                                  scaling=math.log(2.0))
    keys, values = k.split(kv), v.split(kv)
    ref, tol = reference(query, q, keys, values, math.log(2.0), True, (pk, pv))
    _check(out, ref, _tail_tolerance(tol, dtype, [pv.transpose(0, 1), *values]))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rising", [False, True])
def test_scores_of_any_finite_size(dtype, rising):
    """Scores of 2^28, whose differences are far above the rounding of an fp32 score: each row is the value of its
    largest key, but for the rounding of that key's weight and of the output (half a step each), and of a few fp32
    products."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(9)
    n, D = 900, 64
    query = torch.zeros(n, 4, D, dtype=dtype, device="cuda")
    query[..., 0] = 8192.0
    rank = torch.arange(n, device="cuda") if rising else torch.randperm(n, generator=g, device="cuda")
    k = torch.zeros(n, 2, D, dtype=dtype, device="cuda")
    # 8 significant bits: 128 keys of one binade each; 8192 times the least step is 2^13
    k[..., 0] = torch.ldexp(1 + (rank % 128) / 128, (rank // 128) + 8)[:, None].to(dtype)
    v = torch.randn((n, 2, D), generator=g, device="cuda").to(dtype)
    top = torch.stack([rank[:i + 1].argmax() for i in range(n)])
    out = packed_attention(query, k, v, lens_tensor([n]), scaling=1.0)
    ref = v[top].repeat_interleave(2, 1).double()
    fi = torch.finfo(dtype)
    _check(out, ref, ref.abs() * (fi.eps + 2.0 ** -20) + fi.smallest_normal * fi.eps)


@pytest.mark.parametrize("kind", ["packed", "prefix", "append"])
def test_tokens_ahead_of_the_first_sequence(kind):
    """Starts that do not begin at 0: the sequences' rows are those of the batch without the tokens ahead, which get
    zeros, or keep a given out, and append nothing; a negative start is reported."""
    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(3)
    x = lambda *s: torch.randn(s, generator=g, device="cuda").to(F16)   # noqa: E731
    T, ahead, q, kv = 400, 150, [130, 0, 70], [1000, 20, 300]
    query, key = x(T, 4, 64), x(T, 2, 64)
    k, v, pk, pv = x(3, 2, 1100, 64), x(3, 2, 1100, 64), x(2, 3000, 64), x(2, 3000, 64)
    kl, f = torch.tensor(kv, dtype=torch.int32, device="cuda"), torch.rand(32, generator=g, device="cuda")

    def call(query, key, cu, out=None):
        if kind == "packed":
            return packed_attention(query, k, v, cu, kv_len=kl, out=out), ()
        if kind == "prefix":
            return shared_prefix_attention(query, pk, pv, k, v, kl, cu, out=out), ()
        slots = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
        return norm_rotate_append(query, key, key, *slots, cu, kl - torch.tensor(q, device="cuda", dtype=torch.int32), f, out=out), slots

    want, kept = call(query[ahead:], key[ahead:], lens_tensor(q))
    cu = lens_tensor(q) + ahead
    out, slots = call(query, key, cu)
    end = ahead + sum(q)
    assert torch.equal(out[ahead:end], want[:sum(q)]) and not out[:ahead].any() and not out[end:].any()
    assert all(torch.equal(a, b) for a, b in zip(slots, kept))
    out, slots = call(query, key, cu, torch.full_like(query, 5.0))
    assert torch.equal(out[ahead:end], want[:sum(q)]) and (out[:ahead] == 5).all() and (out[end:] == 5).all()
    assert all(torch.equal(a, b) for a, b in zip(slots, kept))
    L.device_status()
    cu[0] = -1
    call(query, key, cu)
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_DEVICE_INPUT


def test_keys_may_start_behind_the_first_row():
    """Packed keys have starts of their own: rows ahead of cu_seqlens_k[0] belong to no sequence."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(4)
    query, k, v = (torch.randn((n, h, 64), generator=g, device="cuda").to(F16) for n, h in ((9, 4), (40, 2), (40, 2)))
    k[:7], v[:7] = float("nan"), float("inf")
    cu_k = torch.tensor([7, 20, 40], dtype=torch.int32, device="cuda")
    out = packed_attention(query, k, v, lens_tensor([4, 5]), cu_k)
    _check(out, *reference(query, [4, 5], [k[7:20], k[20:]], [v[7:20], v[20:]], 64 ** -0.5))


def test_refusals_of_the_library_are_value_errors():
    """Strides that do not nest, numbers that fp32 does not hold: refused before anything is launched."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    from helix_online_kv.shared_prefix import shared_prefix_attention
    z = lambda *s: torch.zeros(s, dtype=F16, device="cuda")   # noqa: E731
    q, k, cu = z(4, 8, 64), z(4, 2, 64), lens_tensor([4])
    for kw in (dict(key=z(1, 2, 64).expand(4, 2, 64)), dict(value=z(4, 1, 64).expand(4, 2, 64)), dict(scaling=1e-60),
               dict(scaling=1e39)):
        with pytest.raises(ValueError):
            packed_attention(**{**dict(query=q, key=k, value=k, cu_seqlens_q=cu), **kw})
    with pytest.raises(ValueError):
        shared_prefix_attention(q, z(1, 9, 64).expand(2, 9, 64), z(2, 9, 64), k, k, cu_seqlens_q=cu)
    slots, n = z(1, 2, 16, 64), lens_tensor([])
    with pytest.raises(ValueError):
        norm_rotate_append(q, k, k, slots, slots.clone(), cu, n, torch.ones(32, device="cuda"), eps=1e39)


@pytest.mark.parametrize("Hq,Hkv,D", [(2, 2, 64), (8, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_rows_that_the_mask_hides(Hq, Hkv, D, bad):
    """A hidden key reaches no query; a hidden value reaches at most the queries W + 126 tokens ahead of it, W = 2
    floor(128 / group), as the documentation says; whole items, two tiles each, and items cut over CTAs."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(D + Hq)
    n, W = 1500, 2 * (128 * Hkv // Hq)
    query, k, v = (torch.randn((n, h, D), generator=g, device="cuda").to(BF16) for h in (Hq, Hkv, Hkv))
    clean = packed_attention(query, k, v, lens_tensor([n]))
    for j in (200, 777, 1499):
        k2, v2 = k.clone(), v.clone()
        k2[j], v2[j] = bad, bad
        out = packed_attention(query, k2, v, lens_tensor([n]))
        assert torch.equal(out[:j], clean[:j])
        out = packed_attention(query, k, v2, lens_tensor([n]))
        free = max(j - (W + 126), 0)
        assert torch.equal(out[:free], clean[:free])
        assert not out[j:].isfinite().any()


# ---- every key counts: results that show the loss of a single one ------------------


def _counted(q, kv, ahead, step, D, Hq):
    """Rows of equal scores: the share of each channel's keys among those a query sees, [T, H_q, D]; key j of a row
    (`ahead` prefix keys, then the own ones) is marked in channel j // step."""
    rows = []
    for m, n in zip(q, kv):
        marks = torch.nn.functional.one_hot(torch.arange(ahead + n, device="cuda") // step, D).double().cumsum(0)
        seen = torch.arange(ahead + n - m, ahead + n, device="cuda") + 1
        rows.append(torch.where((seen > 0)[:, None], marks[seen - 1] / seen[:, None], 0.0))
    return torch.cat(rows)[:, None].expand(-1, Hq, -1)


def _share_tolerance(ref, dtype):
    """Equal scores give equal weights, exact sums of whole numbers and one quotient: half a step of the output, and
    2^-20 for the weights' common factor and the quotient.  One key of a channel's 128 is 2^-7."""
    return ref * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q,kv,step", [
    ([1], [9000], 128), ([1], [12345], 128), ([1, 1, 1], [5000, 1, 16384], 128),   # one token over many CTAs
    ([1, 3], [1030, 2047], 16),
    ([2048], [2048], 16), ([300, 1], [2000, 2041], 16),                           # causal prompts, cut and whole
    ([40, 3], [7000, 6001], 128),
])
def test_equal_scores_count_every_key(q, kv, step, dtype):
    from helix_online_kv.prefill import packed_attention
    g = _gen(sum(kv))
    Hq, Hkv, D = 8, 2, 128
    query = torch.zeros(sum(q), Hq, D, dtype=dtype, device="cuda")
    k = torch.randn((sum(kv), Hkv, D), generator=g, device="cuda").to(dtype)
    v = torch.cat([torch.nn.functional.one_hot(torch.arange(n, device="cuda") // step, D) for n in kv])
    v = v[:, None].expand(-1, Hkv, -1).to(dtype).contiguous()
    out = packed_attention(query, k, v, lens_tensor(q), lens_tensor(kv))
    ref = _counted(q, kv, 0, step, D, Hq)
    _check(out, ref, _share_tolerance(ref, dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("P,q,kv", [(8000, [1, 2, 1], [40, 300, 1]), (129, [1, 3], [900, 5]),
                                    (5001, [1] * 40, [7 * i + 1 for i in range(40)])])
def test_equal_scores_count_every_key_behind_a_prefix(P, q, kv, dtype):
    from helix_online_kv.shared_prefix import shared_prefix_attention
    g = _gen(P)
    Hq, Hkv, D = 8, 2, 128
    query = torch.zeros(sum(q), Hq, D, dtype=dtype, device="cuda")
    k, pk = (torch.randn(s, generator=g, device="cuda").to(dtype) for s in ((sum(kv), Hkv, D), (Hkv, P, D)))
    one_hot = lambda j: torch.nn.functional.one_hot(j // 128, D).to(dtype)   # noqa: E731
    pv = one_hot(torch.arange(P, device="cuda"))[None].expand(Hkv, -1, -1).contiguous()
    v = torch.cat([one_hot(P + torch.arange(n, device="cuda")) for n in kv])[:, None].expand(-1, Hkv, -1).contiguous()
    out = shared_prefix_attention(query, pk, pv, k, v, cu_seqlens_q=lens_tensor(q), cu_seqlens_k=lens_tensor(kv))
    ref = _counted(q, kv, P, 128, D, Hq)
    _check(out, ref, _share_tolerance(ref, dtype))


def _codes(n, D, dtype):
    """Keys [n, D] of +-1: the 14 bits of the key's number, nine times over; two keys whose numbers differ in d bits have
    the product 126 - 18 d."""
    bits = (torch.arange(n, device="cuda")[:, None] >> torch.arange(14, device="cuda")) & 1
    k = torch.zeros(n, D, device="cuda")
    k[:, :126] = (2 * bits - 1).float().repeat(1, 9)
    return k.to(dtype)


def _one_key_tolerance(ref, dtype):
    """With a scaling of 4 the key that a query names outweighs each other one by e^72: half a step each for its weight
    and the output, 2^-20 for fp32 products."""
    fi = torch.finfo(dtype)
    return ref.abs() * (fi.eps + 2.0 ** -20) + fi.smallest_normal * fi.eps


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("n", [700, 3000, 9000, 12345])
def test_single_keys_are_found(n, dtype):
    """Queries that name one key each: the first, the last, both sides of every tile's edge; as one sequence of many
    queries, and eight heads of one token at a time (items cut over CTAs)."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(n)
    D = 128
    k, v = _codes(n, D, dtype)[:, None], torch.randn((n, 1, D), generator=g, device="cuda").to(dtype)
    names = sorted({x for e in range(0, n + 128, 128) for x in (e - 1, e, e + 1) if 0 <= x < n} | {n - 1})
    names += names[:-len(names) % 8]
    query = k[names]
    out = packed_attention(query, k, v, lens_tensor([len(names)]), lens_tensor([n]), scaling=4.0, is_causal=False)
    ref = v[names].double()
    _check(out, ref, _one_key_tolerance(ref, dtype))
    for at in range(0, len(names), 8):
        out = packed_attention(query[at:at + 8].transpose(0, 1).contiguous(), k, v, lens_tensor([1]), lens_tensor([n]), scaling=4.0)
        _check(out[0], ref[at:at + 8, 0], _one_key_tolerance(ref[at:at + 8, 0], dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_prompt_whose_queries_name_themselves(dtype):
    """The diagonal: query i names key i, the last one it sees."""
    from helix_online_kv.prefill import packed_attention
    g = _gen(1)
    n, D = 3001, 128
    k, v = _codes(n, D, dtype)[:, None], torch.randn((n, 1, D), generator=g, device="cuda").to(dtype)
    out = packed_attention(k.expand(-1, 4, -1).contiguous(), k, v, lens_tensor([n]), scaling=4.0)
    ref = v.double().expand(-1, 4, -1)
    _check(out, ref, _one_key_tolerance(ref, dtype))


def test_outputs_whose_rows_overlap_are_refused():
    """An expanded out, or slots that several sequences share: rows would be written over one another."""
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.rotary import norm_rotate_append
    z = lambda *s: torch.zeros(s, dtype=F16, device="cuda")   # noqa: E731
    q, k, cu = z(4, 8, 64), z(4, 2, 64), lens_tensor([4])
    for out in (z(1, 8, 64).expand(4, 8, 64), z(4, 1, 64).expand(4, 8, 64)):
        with pytest.raises(ValueError, match="overlap"):
            packed_attention(q, k, k, cu, out=out)
        with pytest.raises(ValueError, match="overlap"):
            norm_rotate_append(q, k, k, z(1, 2, 16, 64), z(1, 2, 16, 64), cu, lens_tensor([]), torch.ones(32, device="cuda"), out=out)
    shared, own = z(1, 2, 16, 64).expand(2, 2, 16, 64), z(2, 2, 16, 64)
    for ks, vs in ((shared, own), (own, shared)):
        with pytest.raises(ValueError, match="overlap"):
            norm_rotate_append(q, k, k, ks, vs, lens_tensor([2, 2]), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda"))
