"""Calls and backward passes while something watches PyTorch's operations (a counter of operations, selective checkpointing): the tensors are plain ones."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from powersgd_b200 import clip_grad_norm
from powersgd_b200.ops.attention import packed_attention
from powersgd_b200.ops.rotary import rotate_projection
from powersgd_b200.ops.tokens import token_log_probs

pytestmark = pytest.mark.gpu


class Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _rotate(x):
    return torch.cat(rotate_projection(x, 4, 2, positions=torch.arange(x.shape[0], device="cuda")), 1)


def _attention(x):
    return packed_attention(x[:, :4], x[:, 4:6], x[:, 6:], torch.tensor([0, 5, 12], dtype=torch.int32, device="cuda"))


def _tokens(x):
    return token_log_probs(x.flatten(1), torch.arange(12, device="cuda")).log_probs


@pytest.mark.parametrize("call", [_rotate, _attention, _tokens])
@pytest.mark.parametrize("where", ["forward", "backward", "both"])
def test_watched(call, where):
    x = torch.randn(12, 8, 16, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).bfloat16().requires_grad_()

    def run(forward, backward):
        with Watch() if forward else torch.enable_grad():
            out = call(x)
        grad = torch.ones_like(out)
        with Watch() if backward else torch.enable_grad():
            return out, torch.autograd.grad(out, x, grad)[0]

    want = run(False, False)
    got = run(where != "backward", where != "forward")
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_watched_clipping():
    p = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    p.grad = torch.ones(1000, device="cuda")
    with Watch():
        norm = clip_grad_norm([p], 1.0)
    assert abs(norm.item() - 1000**0.5) <= 1e-5 and abs(p.grad.norm().item() - 1) <= 1e-5
