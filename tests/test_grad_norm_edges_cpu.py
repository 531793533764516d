"""What the native call for the gradients' norm asks of the device, without one."""
import numpy as np
import pytest
import torch

from powersgd_b200.ops import grad_norm as module
from powersgd_b200.ops import native


def items(*sizes):
    """A list as the native call takes it; its addresses are never read."""
    listed = np.zeros(len(sizes), dtype=module.ITEM)
    listed["g"], listed["n"] = 1 << 40, sizes
    return listed.tobytes(), len(sizes)


@pytest.mark.skipif(not native.available(), reason="the native library is not built")
@pytest.mark.skipif(torch.cuda.is_available(), reason="there is a GPU")
def test_short_lists_ask_for_scratch_where_no_device_runs_their_cluster():
    """One launch of a cluster of 16 blocks is for devices that run it; elsewhere a short list takes two launches, and scratch."""
    long = native.lib().psgd_grad_norm_parts(*items(1 << 30))
    assert long > 0
    for sizes in ([5], [100] * 50, [10] * 400, [0] * 2000 + [1]):
        words = native.lib().psgd_grad_norm_parts(*items(*sizes))
        assert words >= long
    for sizes in ([0], [0] * 50, [0] * 2000):
        assert native.lib().psgd_grad_norm_parts(*items(*sizes)) == 0     # (nothing to add up)
