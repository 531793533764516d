"""Gradients whose memory is another tensor's until they are written, short lists on devices that do not run their cluster."""
import math

import numpy as np
import pytest
import torch
from test_grad_norm_cpu import TYPES, check, make
from test_grad_norm_edges_cpu import check_range_of_float64, check_small_factors

from powersgd_b200 import clip_grad_norm, grad_norm
from powersgd_b200.ops import grad_norm as module
from powersgd_b200.ops import host, native

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(module, "operators", None)
    else:
        assert host.operators is not None
    return request.param


@pytest.mark.parametrize("numel", [1000, 3_000_000])
@pytest.mark.parametrize("clones", [1, 2])
def test_gradients_that_are_copied_when_written(form, clones, numel):
    """The tensor that a gradient was cloned from keeps what it holds; each clone is scaled."""
    source = torch.randn(numel, device="cuda")
    before = source.clone()
    params = [torch.nn.Parameter(torch.zeros(numel, device="cuda")) for _ in range(clones)]
    for p in params:
        p.grad = torch._lazy_clone(source)
    norm = clip_grad_norm(params, 1.0)
    want = math.sqrt(clones * before.double().square().sum().item())
    assert abs(norm.item() - want) <= want * 2.0**-23
    assert torch.equal(source, before)
    for p in params:
        off = (p.grad.double() - before.double() / (want + 1e-6)).abs()
        assert (off <= before.double().abs() / want * 2.0**-22).all()
    assert abs(grad_norm(params).item() - 1) <= 2.0**-20


@pytest.mark.parametrize("largest", [2, math.inf])
@pytest.mark.parametrize("count", [1, 40, 41, 321, 1300])
def test_short_lists_in_two_launches(monkeypatch, count, largest):
    """As where the device does not run a cluster of 16 blocks: given scratch, a short list takes the launches of a long one. Python's form of the call asks for
    as much as a long list does."""
    library = native.lib()
    ask = library.psgd_grad_norm_parts
    long = np.zeros(count, dtype=module.ITEM)
    long["g"], long["n"] = 1 << 40, 1 << 30      # (addresses that nobody reads)
    words = ask(long.tobytes(), count)
    assert words > 0
    asked = []
    monkeypatch.setattr(module, "operators", None)
    monkeypatch.setattr(library, "psgd_grad_norm_parts", lambda *a: asked.append(ask(*a)) or words)
    held = min(count - 1, 60)
    for max_norm in (0.1, 1e9):
        check(make([(3,)] * held + [(0,)] * (count - 1 - held) + [(70, 9)], TYPES, "cuda"), max_norm, largest)
    check(make([(0,)] * (count - 1) + [(1,)], TYPES, "cuda"), 0.1, largest)
    assert asked and not any(asked)     # (this device runs it)


def test_range_of_float64(form):
    check_range_of_float64("cuda")


@pytest.mark.parametrize("numel", [300, 3_000_000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_the_normal_numbers(form, numel, dtype):
    check_small_factors(numel, dtype, "cuda")
