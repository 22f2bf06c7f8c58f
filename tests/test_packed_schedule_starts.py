"""The packed attention's schedule (packed_schedule.cuh) built for the host: where
the first sequence must start.  CPU only."""

import ctypes

import numpy as np
import pytest

from test_packed_schedule import lib  # noqa: F401  (the fixture that builds the host library)


def _items(lib, starts, kv, T, prefix=0):   # noqa: F811
    cq, kl = np.asarray(starts, np.int32), np.asarray(kv, np.int32)
    out, units = np.zeros((4096, 16), np.int32), ctypes.c_int64(0)
    n = lib.host_schedule(cq.ctypes.data, None, kl.ctypes.data, len(kv), T, 2, 32, max(kv, default=0), prefix, 1, 5,
                          out.ctypes.data, len(out), ctypes.addressof(units))
    assert n >= 0
    return {(int(r[5]), int(r[3])): int(r[4]) for r in out[:n]}   # (source, first token): tokens


@pytest.mark.parametrize("first", [1, 3, -1])
def test_a_batch_that_does_not_start_at_its_first_token(lib, first):   # noqa: F811
    """Its first sequence gets no work, like any other whose lengths do not fit; the others get theirs."""
    assert _items(lib, [0, 4, 9], [8, 8], 9) == {(0, 0): 4, (0, 4): 5}
    assert _items(lib, [first, 4, 9], [8, 8], 9) == {(0, 4): 5}


def test_no_sequence_owns_no_token(lib):   # noqa: F811
    """A single start that is not 0 gives the prefix no rows."""
    assert _items(lib, [0], [], 9, prefix=300) == {}
    assert _items(lib, [5], [], 9, prefix=300) == {}
