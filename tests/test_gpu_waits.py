"""Bounded waits of the decoder-serving kernels that run out: every warp of a group takes the same
way, nothing hangs, and the context keeps working."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EINVAL = -1


def test_a_group_gives_up_together(cuda_lib):
    """A warp that gives up a millisecond before the barrier completes takes its neighbours with it: they
    would wait for it at the next barrier of the four."""
    from spinn_b200 import runtime as rt
    call = cuda_lib.spinn_cuda_selftest_group_wait
    assert call(0, 1_000_000_000) == 15
    assert call(1_000_000, 1_000_000_000) == 15
    assert call(20_000_000, 1_000_000) == 0      # the first warp's limit is 1 ms, the others see the arrival
    assert call(0, 1_000_000_000) == 15
    assert call(0, 0) == EINVAL and call(200_000_000, 1) == EINVAL and call(0, 2_000_000_000) == EINVAL
    x, w = torch.ones(700, 128, device="cuda").half(), torch.ones(300, 128, device="cuda").half()
    y = torch.empty(700, 300, device="cuda").half()
    rt.linear(x, w, y)
    rt.stream_sync()
    assert bool((y == 128).all())
