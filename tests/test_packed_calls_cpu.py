"""What the packed-batch entry points keep between calls and refuse, without a
GPU: the argument checks are stubbed, nothing is launched."""

import pytest
import torch

from helix_online_kv import _lib as L
from helix_online_kv import prefill as F
from helix_online_kv import rotary as R
from helix_online_kv.shared_prefix import shared_prefix_attention


class _Nothing:
    """A checked call that has no tokens: the entry point returns before any launch."""

    n_tokens = 0


@pytest.mark.parametrize("kind", ["packed", "prefix"])
def test_a_scaling_changed_in_place_is_read_again(monkeypatch, kind):
    seen = []
    monkeypatch.setattr(F, "_checked", L.Checked())
    monkeypatch.setattr(F, "_packed_check", lambda *a: seen.append(a[6]) or (_Nothing, 0))
    q, cu, scale = torch.zeros(2, 2, 64), torch.zeros(3, dtype=torch.int32), torch.tensor(0.5)

    def call(s):
        if kind == "packed":
            return F.packed_attention(q, q, q, cu, scaling=s)
        return shared_prefix_attention(q, q, q, q, q, cu_seqlens_q=cu, scaling=s)

    call(scale)
    scale.fill_(2.0)
    call(scale)
    assert seen == [0.5, 2.0] and all(type(s) is float for s in seen)
    call(2.0)
    call(torch.tensor(2.0))
    assert len(seen) == 2   # the same value is the same geometry
    with pytest.raises((TypeError, ValueError)):
        call("much")
    with pytest.raises((TypeError, ValueError, RuntimeError)):
        call(torch.ones(2))
    assert all(not isinstance(x, torch.Tensor) for key in F._checked for x in key)


def test_an_eps_changed_in_place_is_read_again(monkeypatch):
    seen = []
    monkeypatch.setattr(R, "_checked", L.Checked())
    monkeypatch.setattr(R, "_check", lambda *a: seen.append(a[10]) or _Nothing)
    q, n, eps = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), torch.tensor(0.5)
    call = lambda e: R.norm_rotate_append(q, q, q, q, q, None, n, q, eps=e)   # noqa: E731
    call(eps)
    eps.fill_(2.0)
    call(eps)
    assert seen == [0.5, 2.0] and all(type(e) is float for e in seen)
    assert all(not isinstance(x, torch.Tensor) for key in R._checked for x in key)


@pytest.mark.parametrize("status,error", [(L.ERR_INVALID, ValueError), (L.ERR_UNSUPPORTED, ValueError),
                                          (L.ERR_CUDA, L.HokvError), (L.ERR_WORKSPACE, L.HokvError)])
@pytest.mark.parametrize("stage", ["workspace", "call"])
def test_arguments_that_the_library_refuses_are_value_errors(monkeypatch, status, error, stage):
    """Refusals of the C entry points (strides that do not nest, a scaling that is 0 in fp32) are as Python's own."""
    class Args:
        n_tokens = 2

    monkeypatch.setattr(L, "call_on", lambda *a: status)
    q, cu = torch.zeros(2, 2, 64), torch.zeros(3, dtype=torch.int32)
    if stage == "call":
        with pytest.raises(error):
            L.check_call(L.call_on(), "packed_attention")
        from_buffer = type("A", (), {"from_buffer_copy": staticmethod(lambda a: a)})
        monkeypatch.setattr(L, "PackedArgs", from_buffer)
        monkeypatch.setattr(L, "NormRotateArgs", from_buffer)
        monkeypatch.setattr(F, "_checked", L.Checked())
        monkeypatch.setattr(R, "_checked", L.Checked())
        monkeypatch.setattr(F, "_packed_check", lambda *a: (Args(), 16))
        monkeypatch.setattr(R, "_check", lambda *a: Args())
        with pytest.raises(error):
            F.packed_attention(q, q, q, cu)
        with pytest.raises(error):
            R.norm_rotate_append(q, q, q, q, q, None, cu[:2], q)
    else:
        assert L.check_call(L.OK, "x") is None
        with pytest.raises(error, match="packed"):
            L.check_call(status, "packed")


def test_half_a_prefix_is_refused():
    q, cu = torch.zeros(2, 2, 64), torch.zeros(3, dtype=torch.int32)
    for pk, pv in ((q, None), (None, q)):
        with pytest.raises(ValueError, match="prefix_key and prefix_value"):
            shared_prefix_attention(q, pk, pv, q, q, cu_seqlens_q=cu)


@pytest.mark.parametrize("shape,stride,ok", [
    ((4, 8, 64), (512, 64, 1), True), ((4, 8, 64), (64, 256, 1), True),         # heads inside tokens, and outside
    ((4, 8, 64), (640, 72, 1), True), ((1, 8, 64), (0, 64, 1), True),           # padded; one token
    ((4, 8, 64), (0, 64, 1), False), ((4, 8, 64), (512, 0, 1), False),          # expanded
    ((4, 8, 64), (64, 64, 1), False), ((4, 8, 64), (512, 32, 1), False),
    ((2, 2, 16, 64), (2048, 1024, 64, 1), True), ((2, 2, 16, 64), (0, 1024, 64, 1), False),
    ((0, 8, 64), (0, 0, 1), True),
])
def test_rows_that_overlap(shape, stride, ok):
    assert F._rows_apart(torch.zeros(1 << 13).as_strided(shape, stride)) is ok
