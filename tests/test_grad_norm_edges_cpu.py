"""Gradients whose squares leave the range of float64; what the native call for the gradients' norm asks of the device, without one."""
import math

import numpy as np
import pytest
import torch

from powersgd_b200 import clip_grad_norm, grad_norm
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


def check_range_of_float64(device):
    """As the library has it: beyond 1.3e154 the norm is infinite and clipping leaves zeros; below 1e-162 it is zero. Float32 gradients in the same list count by
    their own size, and the largest magnitude has the range of its type."""
    for value, norm, left in ((1e200, math.inf, 0.0), (1e-200, 0.0, 1e-200), (1e153, 1e153 * 10, 1.0 / 10)):
        params = []
        for _ in range(2):
            p = torch.nn.Parameter(torch.zeros(50, dtype=torch.float64, device=device))
            p.grad = torch.full((50,), value, dtype=torch.float64, device=device)
            params.append(p)
        theirs = [torch.nn.Parameter(p.detach().clone()) for p in params]
        for p, t in zip(params, theirs):
            t.grad = p.grad.clone()
        got, want = clip_grad_norm(params, 1.0), torch.nn.utils.clip_grad_norm_(theirs, 1.0)
        assert got.dtype == torch.float64
        if math.isinf(norm):
            assert got == norm and want == norm
        else:
            assert abs(got.item() - norm) <= norm * 2.0**-50
        for p, t in zip(params, theirs):
            assert ((p.grad - left).abs() <= left * 2.0**-49).all() and torch.allclose(p.grad, t.grad, rtol=2.0**-40, atol=0.0)
        for p in params:
            p.grad.fill_(value)
        assert grad_norm(params, math.inf).item() == value
    with pytest.raises(RuntimeError, match="nothing was scaled"):
        params[0].grad.fill_(1e200)
        clip_grad_norm(params, 1.0, error_if_nonfinite=True)
    assert (params[0].grad == 1e200).all()


def test_range_of_float64():
    check_range_of_float64("cpu")


def check_small_factors(numel, dtype, device):
    """Gradients near the end of float32's range: what they are multiplied with is far below its normal numbers, and what comes of it is not. Bounds: the factor's
    rounding to 32 bits, the product's, and half a step of the type."""
    p, q = (torch.nn.Parameter(torch.zeros(n, dtype=t, device=device)) for n, t in ((numel, dtype), (77, torch.float32)))
    for t, seed in ((p, 0), (q, 1)):
        t.grad = ((1 + torch.rand(t.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)) * 2.0**126).to(t.dtype).to(device)
    before = [t.grad.double() for t in (p, q)]
    norm = math.sqrt(sum(b.square().sum().item() for b in before))
    clip_grad_norm([p, q], 2.0**-10)
    for t, b in zip((p, q), before):
        want = b * (2.0**-10 / norm)
        own = 2.0**-22.9 + (torch.finfo(t.dtype).eps / 2 if t.dtype.itemsize == 2 else 0)
        assert ((t.grad.double() - want).abs() <= want * own).all(), ((t.grad.double() - want).abs() / want).max().item()


@pytest.mark.parametrize("numel", [3, 30000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_the_normal_numbers(numel, dtype):
    check_small_factors(numel, dtype, "cpu")


@pytest.mark.parametrize("default", [torch.float16, torch.float64])
def test_other_default_types(default):
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        check_small_factors(300, torch.float32, "cpu")
        p = torch.nn.Parameter(torch.zeros(100, dtype=torch.float32))
        p.grad = torch.ones(100, dtype=torch.float32)
        assert abs(clip_grad_norm([p], 5.0).item() - 10) <= 10 * 2.0**-23
        assert ((p.grad - 0.5).abs() <= 2.0**-22).all()
    finally:
        torch.set_default_dtype(before)
