"""Attention's bookkeeping of TMA copies in flight when a wait expires, against a model of the barriers."""
import ctypes

import pytest

from spinn_b200 import lib


class Barrier:
    """An mbarrier of one arrival: a phase is open from its arming until the copy's bytes are there."""

    def __init__(self):
        self.phase, self.open = 0, False

    def arm(self):
        assert not self.open, "armed while a copy is in flight"
        self.open = True

    def land(self):
        assert self.open
        self.open, self.phase = False, self.phase ^ 1

    def would_wait_for(self, parity):
        """Whether a wait for the phase of this parity waits for the copy in flight."""
        return self.open and self.phase == parity


def ring(ops):
    a, out = (ctypes.c_int32 * max(len(ops), 1))(*ops), (ctypes.c_int32 * (3 * len(ops) + 3))()
    assert lib.lib().spinn_cuda_diag_attention_ring(a, len(ops), out) == 0
    return out[3 * len(ops) - 3:3 * len(ops)] if ops else [0, 0, 0]


@pytest.mark.parametrize("stages", [2, 3, 6])
def test_after_an_expired_wait_nothing_is_armed_and_what_flies_is_waited_for(stages):
    tiles = 3 * stages + 1
    for late, again in [(i, j) for i in range(tiles + 1) for j in (False, True)]:
        # the wait for tile `late` expires (tiles: none does), and with it those behind it whose copies are
        # still in flight; again: those copies land before they are waited for, the late one never does
        bars, ops, expired = [Barrier() for _ in range(stages)], [], False

        def issue(i):
            ops.append(i % stages)
            if ring(ops)[0]:
                bars[i % stages].arm()

        for i in range(min(stages - 1, tiles)):
            issue(i)
        for i in range(tiles):
            if i + stages - 1 < tiles:
                issue(i + stages - 1)
            s = i % stages
            parity = ring(ops)[1] >> s & 1
            assert bars[s].would_wait_for(parity) or expired
            lands = bars[s].would_wait_for(parity) and (not expired or again) and not (i - late >= 0 and (i - late) % stages == 0)
            expired |= i == late
            if lands:
                bars[s].land()
            assert lands or expired
            ops.append(s + (16 if lands else 32))
        _, parity, flight = ring(ops)
        for s, b in enumerate(bars):
            assert (flight >> s & 1) == b.open
            if b.open:
                assert b.would_wait_for(parity >> s & 1)
        assert (flight != 0) == (late < tiles)


def test_ring_diagnostic_refuses_other_operations():
    out = (ctypes.c_int32 * 3)()
    for bad in (48, -1):
        assert lib.lib().spinn_cuda_diag_attention_ring((ctypes.c_int32 * 1)(bad), 1, out) == lib.EINVAL
    assert lib.lib().spinn_cuda_diag_attention_ring(None, 1, out) == lib.EINVAL
