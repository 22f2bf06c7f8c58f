"""prefill_attention where one key dominates a row: thousands of keys far below it
hold mass that f16 weights must not lose."""

import math

import pytest
import torch

from packed_reference import reference

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Skv,gap,sink,causal", [
    (300, 300, 19.25, 0, True), (2048, 2048, 22.25, 0, True), (40, 3000, 20.25, 2000, True),
    (5, 16384, 24.75, 0, False), (130, 1000, 17.25, 999, False),
])
def test_keys_far_below_the_largest_score(Sq, Skv, gap, sink, causal, D, dtype):
    """Scores in log2 units: `gap` for the sink, whose value is 0, and 0 for the others.  f16 weights are stored times 2^7,
    so one below the normal range is off by up to 2^-25 of 2^7: 2^-32 sum |V| of the result."""
    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import prefill_attention
    g = torch.Generator(device="cuda")
    g.manual_seed(Skv)
    Hq, Hkv = 4, 2
    k = torch.zeros(1, Hkv, Skv, D, dtype=dtype, device="cuda")
    v = (torch.rand((1, Hkv, Skv, D), generator=g, device="cuda") + 0.5).to(dtype)
    k[:, :, sink, 0], v[:, :, sink] = gap, 0.0
    q = torch.zeros(1, Hq, Sq, D, dtype=dtype, device="cuda")
    q[..., 0] = 1
    out = prefill_attention(q, k, v, math.log(2.0), is_causal=causal)[0]
    torch.cuda.synchronize()
    L.device_status()
    ref, tol = reference(q[0].transpose(0, 1), [Sq], [k[0].transpose(0, 1)], [v[0].transpose(0, 1)], math.log(2.0), causal)
    if dtype == F16:
        tol = tol + 2.0 ** -32 * float(v[0].double().abs().sum(1).max())
    err = (out.double() - ref).abs()
    assert (err <= tol).all(), (float(err.max()), float((err / tol).max()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_very_different_sizes(D, dtype):
    """A row's scores rise from -2^22 to 2^22 and fall again, across the sizes from which weights are stored as they
    are: each row is the value of its largest key (half a step each for weight and output, 2^-20 for fp32 products)."""
    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import prefill_attention
    g = torch.Generator(device="cuda")
    g.manual_seed(D)
    n = 1400
    k = torch.zeros(1, 1, n, D, dtype=dtype, device="cuda")
    level = torch.cat((torch.linspace(-8, 8, n // 2), torch.linspace(8, -8, n - n // 2))) + 0.001 * torch.arange(n)
    # two dims sum to a score that fp32 keeps and the type represents: 2^11 * (whole part, fraction in 1/64)
    whole = level.round()
    k[0, 0, :, 0], k[0, 0, :, 1] = (whole * 16).cuda().to(dtype), ((level - whole) * 64).round().cuda().to(dtype)
    v = torch.randn((1, 1, n, D), generator=g, device="cuda").to(dtype)
    q = torch.zeros(1, 2, n, D, dtype=dtype, device="cuda")
    q[..., 0], q[..., 1] = 32768.0, 8192.0
    score = (k[0, 0].double() * q[0, 0, 0].double()).sum(-1)
    out = prefill_attention(q, k, v, 1.0, is_causal=True)[0]
    torch.cuda.synchronize()
    L.device_status()
    best, top = torch.cummax(score, 0)
    alone = (score[None, :] > best[:, None] - 60).tril().sum(1) == 1   # rows with one key in reach of the largest
    assert alone.sum() >= n // 2
    ref = v[0, 0, top].double()[:, None].expand(-1, 2, -1)[alone]
    fi = torch.finfo(dtype)
    err = (out[alone].double() - ref).abs()
    assert (err <= ref.abs() * (fi.eps + 2.0 ** -20) + fi.smallest_normal * fi.eps).all(), float(err.max())
