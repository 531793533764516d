"""Tensors whose address is zero (DTensors and other tensors whose operations Python takes over, tensors whose memory was given back) are refused
before a kernel could be given the address. None of this touches a GPU: tensors that say that they are on one have no memory there."""
import pytest
import torch
import torch.distributed as dist

from powersgd_b200 import clip_grad_norm, grad_norm
from powersgd_b200.ops import adamw, native, scan
from powersgd_b200.ops.attention import check as attention_check
from powersgd_b200.ops.grad_norm import clip_for_step
from powersgd_b200.ops.rotary import rotate_heads, rotate_projection
from powersgd_b200.ops.tokens import check as token_check


class Far(torch.Tensor):
    """Says that it is a tensor of a GPU, and holds nothing."""

    @staticmethod
    def __new__(cls, *shape, dtype=torch.float32, device="cuda:0"):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device=device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError(f"{func} of a tensor without memory")


@pytest.fixture
def mesh():
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        yield dist.init_device_mesh("cpu", (1,))
    finally:
        dist.destroy_process_group()


def parameter(grad):
    p = torch.nn.Parameter(torch.zeros(grad.shape))
    if not isinstance(grad, torch.distributed.tensor.DTensor):
        p.grad = grad
        return p
    p = torch.nn.Parameter(torch.distributed.tensor.zeros(grad.shape, device_mesh=grad.device_mesh, placements=grad.placements))
    p.grad = grad
    return p


def test_sharded_gradients(mesh):
    from torch.distributed.tensor import DTensor, Replicate

    local = [torch.randn(4, 3), torch.randn(5)]
    params = [parameter(DTensor.from_local(t.clone(), mesh, [Replicate()])) for t in local]
    assert params[0].grad.layout == torch.strided and params[0].grad.data_ptr() == 0
    for listed in (params[:1], params, [parameter(torch.ones(2)), params[0]]):
        for call in (lambda: grad_norm(listed), lambda: clip_grad_norm(listed, 0.5), lambda: clip_grad_norm(listed, 0.5, error_if_nonfinite=True),
                     lambda: grad_norm(listed, torch.inf)):
            with pytest.raises(TypeError, match="no memory of its own"):
                call()
    for p, t in zip(params, local):
        assert torch.equal(p.grad.to_local(), t)
    clip_for_step(params, 0.5)      # the library clips them, as before
    norm = torch.cat([t.flatten() for t in local]).norm()
    for p, t in zip(params, local):
        assert torch.allclose(p.grad.to_local(), t * 0.5 / (norm + 1e-6))


def test_sharded_heads(mesh):
    from torch.distributed.tensor import DTensor, Replicate

    plain, at = torch.randn(6, 4, 8), torch.arange(6)
    x, w = DTensor.from_local(plain, mesh, [Replicate()]), DTensor.from_local(torch.ones(8), mesh, [Replicate()])
    for call in (lambda: rotate_heads(x, positions=at), lambda: rotate_heads(plain, positions=at, weight=w), lambda: rotate_projection(x, 2, 1, positions=at),
                 lambda: rotate_projection(plain, 2, 1, positions=at, k_weight=w), lambda: rotate_heads(plain, positions=DTensor.from_local(at, mesh, [Replicate()]))):
        with pytest.raises(TypeError, match="no memory of its own"):
            call()


def test_tensors_that_say_that_they_are_on_a_gpu():
    x = Far(6, 4, 8)
    p = torch.nn.Parameter(torch.zeros(3))
    calls = [lambda: rotate_heads(x, positions=Far(6, dtype=torch.int64)), lambda: rotate_projection(x, 2, 1, offsets=Far(2, dtype=torch.int32)),
             lambda: attention_check(x, x, x, Far(2, dtype=torch.int32), None), lambda: token_check(Far(3, 8), Far(3, dtype=torch.int64), 0, -100, 1.0),
             lambda: adamw.check_lists([x], [x], [[x], [x]], [Far()], 32), lambda: scan.addresses([x]), lambda: scan.addresses([p, x])]
    for call in calls:
        with pytest.raises(TypeError, match="no memory of its own"):
            call()
    for dtype in (torch.float32, torch.bfloat16):
        far = Far(3, dtype=dtype)
        with pytest.raises(TypeError, match="no memory of its own"):
            native.refuse_without_memory("call", None, p, far)


def test_memory_that_was_given_back():
    t = torch.randn(6, 4, 8)
    t.untyped_storage().resize_(0)
    assert t.data_ptr() == 0
    p = torch.nn.Parameter(torch.zeros(6, 4, 8))
    p.grad = t
    for call in (lambda: grad_norm([p]), lambda: clip_grad_norm([p], 0.5), lambda: rotate_heads(t, positions=torch.arange(6))):
        with pytest.raises(RuntimeError, match="was given back"):
            call()


def test_tensors_that_are_not_refused():
    """Subclasses whose operations are PyTorch's, zeros that have no memory, no elements, parameters and views."""

    class Named(torch.Tensor):
        pass

    x, at = torch.randn(6, 4, 8), torch.arange(6)
    want = rotate_heads(x, positions=at)
    assert torch.equal(rotate_heads(x.as_subclass(Named), positions=at), want)
    assert torch.equal(rotate_heads(torch.nn.Parameter(x), positions=at), want)
    assert (rotate_heads(torch._efficientzerotensor((6, 4, 8)), positions=at) == 0).all()
    p = torch.nn.Parameter(torch.zeros(3))
    for grad in (torch.ones(3).as_subclass(Named), torch.ones(6)[::2]):
        p.grad = grad
        assert abs(grad_norm([p]).item() - 3**0.5) <= 2.0**-23
    p.grad = torch._efficientzerotensor((3,))
    assert grad_norm([p]) == 0
    empty = torch.nn.Parameter(torch.zeros(0))
    empty.grad = torch.zeros(0)
    assert grad_norm([empty]) == 0


@pytest.mark.parametrize("count", [1, 2])
def test_clipping_of_a_step_hands_them_to_the_library(count, monkeypatch):
    listed = [Far(3) for _ in range(count)]
    for p in listed:
        p.grad = Far(3)
    assert listed[0].is_cuda
    given = []
    monkeypatch.setattr(torch.nn.utils, "clip_grad_norm_", lambda parameters, max_norm: given.append((parameters, max_norm)))
    clip_for_step(iter(listed), 0.5)
    assert len(given) == 1 and [id(p) for p in given[0][0]] == [id(p) for p in listed] and given[0][1] == 0.5
