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


def run_out_in_long_items():
    """Hundreds of key tiles an item: a CTA that gave up does not wait for each of them again."""
    import time

    import torch

    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    query, k, v, kl = _batch(torch, [6 << 20], 4, 1)
    call = lambda: packed_attention(query, k, v, kv_len=kl)   # noqa: E731
    want = call()
    torch.cuda.synchronize()
    for what in (WEIGHTS, END):
        t = time.time()
        _held(L, what, call)
        assert time.time() - t < 5
        assert torch.equal(call(), want)
    L.device_status()


def replay():
    """A captured call whose waits run out, marks of some pieces left behind; its replays on new data, at once and after
    more failures, and a graph captured before in the same pool are right."""
    import torch

    from helix_online_kv import _lib as L
    from helix_online_kv.prefill import packed_attention
    query, k, v, kl = _batch(torch, [9000, 7000, 12000], D=64)
    other, *_ = _batch(torch, [1, 1, 1], D=64, seed=2)
    first = packed_attention(query, k, v, kv_len=kl)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=pool):
            outs.append(packed_attention(query, k, v, kv_len=kl))
        pool = graphs[0].pool()
    for graph, out in zip(graphs, outs):
        graph.replay()
        assert torch.equal(out, first)
    for round_ in range(4):
        graph, out = graphs[round_ % 2], outs[round_ % 2]
        _held(L, MARKS, graph.replay)
        if round_ == 3:
            _held(L, WEIGHTS, graph.replay)
        # other data: a piece taken from the failed replay would show
        query.copy_(other if round_ % 2 == 0 else query.flip(1))
        want = packed_attention(query, k, v, kv_len=kl)
        for graph, out in zip(graphs, outs):
            for _ in range(3):
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want)
        L.device_status()


def _child(name):
    env = dict(os.environ, HOKV_LIB_VARIANT="stamps")
    r = subprocess.run([sys.executable, os.path.abspath(__file__), name], env=env, capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.gpu
def test_waits_that_run_out_are_reported_and_the_next_call_is_right():
    _child("run_out")


@pytest.mark.gpu
def test_waits_that_run_out_in_long_items():
    _child("run_out_in_long_items")


@pytest.mark.gpu
def test_replays_after_a_failed_one_do_not_take_its_marks():
    _child("replay")


def test_the_product_keeps_nothing_back():
    from helix_online_kv import _lib as L
    if os.environ.get("HOKV_LIB_VARIANT"):
        pytest.skip("an instrumented build is loaded")
    assert L.lib().hokv_hold(1) == L.ERR_UNSUPPORTED


if __name__ == "__main__":
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "helix-online-kv_b200"))
    {f.__name__: f for f in (run_out, run_out_in_long_items, replay)}[sys.argv[1]]()
