"""The packed attention's schedule (packed_schedule.cuh) built for the host: tokens
ahead of the first sequence, and the search for the sequence and pair in which
a CTA's share begins, the kernel's own code over 32 emulated lanes.  CPU only."""

import bisect
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

from test_packed_schedule import CSRC, HERE, ITEM, lib  # noqa: F401  (lib: the fixture that builds the host library)


def _items(lib, starts, kv, T, prefix=0):   # noqa: F811
    cq, kl = np.asarray(starts, np.int32), np.asarray(kv, np.int32)
    out, units = np.zeros((4096, 16), np.int32), ctypes.c_int64(0)
    n = lib.host_schedule(cq.ctypes.data, None, kl.ctypes.data, len(kv), T, 2, 32, max(kv, default=0), prefix, 1, 5,
                          out.ctypes.data, len(out), ctypes.addressof(units))
    assert n >= 0
    return {(int(r[5]), int(r[3])): int(r[4]) for r in out[:n]}   # (source, first token): tokens


@pytest.mark.parametrize("prefix", [0, 300])
def test_tokens_ahead_of_the_first_sequence_have_no_work(lib, prefix):   # noqa: F811
    """They belong to no sequence, and are no queries of a prefix."""
    ahead = lambda n, m: {(1, n): m} if prefix else {}   # noqa: E731
    assert _items(lib, [0, 4, 9], [8, 8], 9, prefix) == {**ahead(0, 9), (0, 0): 4, (0, 4): 5}
    assert _items(lib, [3, 4, 9], [8, 8], 9, prefix) == {**ahead(3, 6), (0, 3): 1, (0, 4): 5}
    assert _items(lib, [9, 9, 9], [8, 8], 9, prefix) == {}
    assert _items(lib, [5], [], 9, prefix) == {}
    # a start that no tensor has, or behind the end of the batch: no work for that sequence, none outside the tokens
    assert _items(lib, [-1, 4, 9], [8, 8], 9, prefix) == {**ahead(0, 9), (0, 4): 5}
    assert _items(lib, [20, 4, 9], [8, 8], 9, prefix) == {(0, 4): 5}


# ---- the warp's search for where a share begins ------------------------------------


@pytest.fixture(scope="module")
def starts_lib():
    src, out = os.path.join(HERE, "native", "hokv_start_host.cpp"), os.path.join(HERE, "native", "_build", "libhokv_start_host.so")
    os.makedirs(os.path.dirname(out), exist_ok=True)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", out, src])
    L = ctypes.CDLL(out)
    L.host_starts.restype = ctypes.c_int64
    vp, i, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    L.host_starts.argtypes = [vp, vp, i, i, i, i, i64, i, i, vp, i, vp]
    return L


def _pairs(q, kv, hkv, tt, prefix, causal):
    """(first unit, sequence, pair, first unit of the sequence) of every pair, and the total, by walking all of them."""
    W, at, out = 2 * tt, 0, []
    seqs = [(sum(q), prefix, False)] if prefix else []
    seqs += [(m, n, causal) for m, n in zip(q, kv)]
    for s, (m, n, c) in enumerate(seqs):
        first = at
        for pr in range(-(-m // W)):
            out.append((at, s, pr, first))
            rows = min(W, m - pr * W)
            keys = max(0, n - m + pr * W + rows) if c else n
            at += hkv * (ITEM + (2 if rows > tt else 1) * keys)
    return out, at


def _check_starts(lib, q, kv, hkv, tt, prefix, causal, rng, most=400):
    pairs, total = _pairs(q, kv, hkv, tt, prefix, causal)
    if not total:
        return
    firsts = [p[0] for p in pairs]
    some = firsts if len(firsts) < most else rng.sample(firsts, most) + firsts[-3:]
    begin = sorted({x for a in some for x in (a - 1, a, a + 1) if 0 <= x < total} | {0, total - 1} |
                   {rng.randrange(total) for _ in range(100)})
    cq, kl = np.concatenate([[0], np.cumsum(q)]).astype(np.int32), np.asarray(kv, np.int32)
    b, out = np.asarray(begin, np.int64), np.zeros((len(begin), 3), np.int64)
    assert lib.host_starts(cq.ctypes.data, kl.ctypes.data, len(q), int(cq[-1]), hkv, tt, max(kv, default=0), prefix,
                           int(causal), b.ctypes.data, len(b), out.ctypes.data) == total
    want = [pairs[bisect.bisect_right(firsts, x) - 1] for x in begin]
    assert out.tolist() == [[s, pr, first] for _, s, pr, first in want]


@pytest.mark.parametrize("n", [1, 3, 31, 32, 33, 64, 65, 700])
def test_the_search_finds_the_pair_that_holds_a_unit(starts_lib, n):
    """Borders on, before and behind a pair; up to 32 sequences and several a lane; empty ones first, last and between."""
    rng = random.Random(n)
    for _ in range(12):
        kv = [rng.choice([0, 1, 127, 128, 129, rng.randint(0, 3000)]) for _ in range(n)]
        q = [rng.choice([0, 0, 1, rng.randint(0, 500), k]) for k in kv]
        if rng.random() < 0.5:
            q[0] = q[-1] = 0
        _check_starts(starts_lib, q, kv, rng.choice([1, 2, 8]), rng.choice([128, 32, 18, 1]),
                      rng.choice([0, 0, 1, 300, 9000]), rng.random() < 0.7, rng)


def test_the_search_in_thousands_of_pairs(starts_lib):
    rng = random.Random(5)
    for q, kv, tt in (([100000], [100000], 1), ([70000, 0, 33], [200000, 9, 40], 4), ([40000], [100], 1),
                      ([1, 262144, 1], [5, 262144, 70], 128)):
        for causal in (True, False):
            _check_starts(starts_lib, q, kv, 2, tt, 0, causal, rng)
        _check_starts(starts_lib, q, kv, 8, tt, 1000, True, rng)
