"""Waits of the packed attention that run out: signals that they need are kept
back in the instrumented build (include/hokv.h, hokv_hold), each for a few
hundredths of a second, in a process of its own.  The call reports
HOKV_ERR_TIMEOUT, the context stays usable, later calls are right.

Run as a program, this file is that process."""

import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
MARKS, WEIGHTS, END = 1, 2, 4


def _times_out(L, call):
    import torch
    torch.cuda.synchronize()
    call()
    with pytest.raises(L.HokvError) as e:
        L.device_status()
    assert e.value.status == L.ERR_TIMEOUT


def _held(L, what, call):
    """`call` while the signals `what` are kept back."""
    L.check(L.lib().hokv_hold(what))
    try:
        _times_out(L, call)
    finally:
        L.check(L.lib().hokv_hold(0))


def _batch(torch, kv, Hq=8, Hkv=2, D=128, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()   # noqa: E731
    return (r(len(kv), Hq, D), r(len(kv), Hkv, max(kv), D), r(len(kv), Hkv, max(kv), D),
            torch.tensor(kv, dtype=torch.int32, device="cuda"))


def run_out():
    """Marks, weights and the end of the stream, one by one and together; items cut over dozens of CTAs, and a prefix."""
    import torch

    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    from helix_online_kv.shared_prefix import shared_prefix_attention
    query, k, v, kl = _batch(torch, [9000, 40, 7000])
    alone = lambda: packed_attention(query, k, v, kv_len=kl)   # noqa: E731
    behind = lambda: shared_prefix_attention(query, k[0], v[0], k, v, kl)   # noqa: E731
    for call, signals in ((alone, (MARKS, WEIGHTS, END, MARKS | WEIGHTS | END)), (behind, (WEIGHTS, END))):
        want = call()
        L.device_status()
        for what in signals:
            _held(L, what, call)
            for _ in range(3):
                assert torch.equal(call(), want)
            L.device_status()


def _child(name):
    env = dict(os.environ, HOKV_LIB_VARIANT="stamps")
    r = subprocess.run([sys.executable, os.path.abspath(__file__), name], env=env, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.gpu
def test_waits_that_run_out_are_reported_and_the_next_call_is_right():
    _child("run_out")


def test_the_product_keeps_nothing_back():
    from helix_online_kv import _lib as L
    if os.environ.get("HOKV_LIB_VARIANT"):
        pytest.skip("an instrumented build is loaded")
    assert L.lib().hokv_hold(1) == L.ERR_UNSUPPORTED


if __name__ == "__main__":
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "helix-online-kv_b200"))
    {f.__name__: f for f in (run_out,)}[sys.argv[1]]()
