"""Gradients whose memory is another tensor's until they are written."""
import math

import pytest
import torch

from powersgd_b200 import clip_grad_norm, grad_norm
from powersgd_b200.ops import grad_norm as module
from powersgd_b200.ops import host

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
