"""The packed attention's schedule (packed_schedule.cuh), built for the host with
g++: every key tile that a (token pair, KV head) item sees is attended once,
pieces of cut items chain in CTA order through distinct workspace slots, the
shares are even, and lengths that do not fit their tensors give no work.  CPU
only."""

import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "helix-online-kv_b200", "csrc")
OUT = os.path.join(HERE, "native", "_build", "libhokv_schedule_host.so")
DIRECT, PIECE, ROWWISE = 0, 1, 2
ITEM, MIN_SHARE, WHOLE = 512, 768, 1536


@pytest.fixture(scope="module")
def lib():
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    src = os.path.join(HERE, "native", "hokv_schedule_host.cpp")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, "-o", OUT, src])
    L = ctypes.CDLL(OUT)
    L.host_schedule.restype = ctypes.c_int64
    vp, i, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    L.host_schedule.argtypes = [vp, vp, vp, i, i, i, i, i64, i, i, i, vp, i64, vp]
    return L


def _schedule(lib, q, kv, hkv, tt, prefix, causal, ctas, layout, T=None, rows=None, cu_q=True):
    cq = np.concatenate([[0], np.cumsum(q)]).astype(np.int32)
    ck = np.concatenate([[0], np.cumsum(kv)]).astype(np.int32)
    kl = np.asarray(kv, np.int32)
    T = int(cq[-1]) if T is None else T
    rows = (int(ck[-1]) if layout == "packed" else max(kv, default=0)) if rows is None else rows
    cap = 1 << 18
    out = np.zeros((cap, 16), np.int32)
    units = ctypes.c_int64(0)
    n = lib.host_schedule(cq.ctypes.data if cu_q else None, ck.ctypes.data if layout == "packed" else None, kl.ctypes.data,
                          len(q), T, hkv, tt, rows, prefix, int(causal), ctas, out.ctypes.data, cap,
                          ctypes.addressof(units))
    assert n >= 0
    return out[:n], units.value


def _expected(q, kv, hkv, tt, prefix, causal):
    """{(src, first token, KV head): (tokens, keys)} of every item."""
    W, items, starts = 2 * tt, {}, np.concatenate([[0], np.cumsum(q)]).astype(int)
    seqs = [(1, 0, int(starts[-1]), prefix, False)] if prefix else []
    seqs += [(0, int(s), n, k, causal) for s, n, k in zip(starts, q, kv)]
    for src, s, n, k, c in seqs:
        for p in range(-(-n // W)):
            m = min(W, n - p * W)
            end = max(0, k - n + p * W + m) if c else k
            for h in range(hkv):
                items[src, s + p * W, h] = (m, end)
    return items


def _check(lib, q, kv, hkv, tt, prefix, causal, ctas, layout="slots"):
    rows, units = _schedule(lib, q, kv, hkv, tt, prefix, causal, ctas, layout)
    want = _expected(q, kv, hkv, tt, prefix, causal)
    assert units == sum(ITEM + (2 if m > tt else 1) * e for m, e in want.values())
    share = max(units // ctas + 1, MIN_SHARE)
    pieces, slots, load = {}, set(), {}
    for r in rows.tolist():
        cta, begins, ends, tok0, n_tok, src, row0, slot, hk, j0, j1, kv_len, pos0, mode, at, chain = r
        pieces.setdefault((src, tok0, hk), []).append((cta, begins, ends, n_tok, j0, j1, mode, at, chain))
        if mode == PIECE:
            assert at // 2 == cta and at not in slots
            slots.add(at)
        load[cta] = load.get(cta, 0) + (2 if n_tok > tt else 1) * (128 * (j1 - j0))
    assert set(pieces) == set(want)
    for key, (m, keys) in want.items():
        tiles = -(-keys // 128)
        ps = sorted(pieces[key])
        assert [p[4] for p in ps][0] == 0 and ps[-1][5] == tiles
        assert all(a[5] == b[4] for a, b in zip(ps, ps[1:]))
        assert all(p[3] == m and (p[4] < p[5] or tiles == 0) for p in ps)
        assert [bool(p[1]) for p in ps] == [True] + [False] * (len(ps) - 1)
        assert [bool(p[2]) for p in ps] == [False] * (len(ps) - 1) + [True]
        if len(ps) == 1:
            assert ps[0][6] == (ROWWISE if prefix else DIRECT)
        else:
            # the chain that the joins follow: slot 1 of the first CTA, slot 0 of those behind it up to the last
            first, last = ps[0][0], ps[-1][0]
            assert [p[7] for p in ps] == [first * 2 + 1] + [c * 2 for c in range(first + 1, last + 1)]
            assert all(p[6] == PIECE for p in ps)
        units_of = ITEM + (2 if m > tt else 1) * keys
        assert len(ps) == 1 or units_of > WHOLE
        if tiles and units_of > WHOLE:
            assert all(p[8] == ps[0][0] * 1000 + ps[-1][0] for p in ps)   # pa_first_cta, pa_last_cta
    # a share's keys, padded to whole tiles item by item
    n_items = {c: sum(1 for ps in pieces.values() for p in ps if p[0] == c) for c in load}
    assert all(v <= share + WHOLE + 256 * (n_items[c] + 1) for c, v in load.items())


@pytest.mark.parametrize("ctas", [1, 7, 148])
def test_random_batches(lib, ctas):
    rng = random.Random(ctas)
    for _ in range(150):
        n = rng.randint(1, 40)
        kv = [rng.choice([0, 1, 127, 128, 129, rng.randint(0, 5000)]) for _ in range(n)]
        q = [rng.choice([0, 1, rng.randint(0, 700), k]) for k in kv]
        tt = rng.choice([128, 64, 42, 32, 18, 16, 1])
        if tt == 1:
            q = [min(x, 40) for x in q]
        _check(lib, q, kv, rng.choice([1, 2, 3, 8]), tt, rng.choice([0, 0, 1, 300, 9000]), rng.random() < 0.7, ctas,
               rng.choice(["slots", "packed"]))


def test_one_long_sequence_is_spread_over_every_cta(lib):
    rows, units = _schedule(lib, [1], [16384], 8, 32, 0, True, 148, "slots")
    assert set(rows[:, 0].tolist()) == set(range(148))
    _check(lib, [1], [16384], 8, 32, 0, True, 148)
    _check(lib, [16384], [16384], 8, 32, 0, True, 148)
    _check(lib, [200000], [1000000], 2, 128, 0, True, 148)


def test_bad_lengths_give_no_work(lib):
    # more tokens than T, a slot longer than its capacity, a negative length
    rows, _ = _schedule(lib, [4, 4], [8, 8], 2, 32, 0, True, 5, "slots", T=4)
    assert set(rows[:, 3].tolist()) == {0}
    rows, _ = _schedule(lib, [4, 4], [8, 9], 2, 32, 0, True, 5, "slots", rows=8)
    assert set(rows[:, 3].tolist()) == {0}
    rows, _ = _schedule(lib, [4, 4], [-1, 8], 2, 32, 0, True, 5, "slots", rows=8)
    assert set(rows[:, 3].tolist()) == {4}
    rows, _ = _schedule(lib, [4, 4], [8, 8], 2, 32, 0, True, 5, "packed", rows=12)
    assert set(rows[:, 3].tolist()) == {0}


def test_one_token_each_without_starts(lib):
    rows, _ = _schedule(lib, [1, 1, 1], [5, 0, 300], 2, 32, 0, True, 9, "slots", cu_q=False)
    assert sorted(set(rows[:, 3].tolist())) == [0, 1, 2]
