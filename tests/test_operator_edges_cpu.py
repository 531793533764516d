"""token_log_probs, packed_attention and AdamW where they can go wrong, in their forms on the CPU."""
import pytest
import torch

from powersgd_b200.ops.tokens import token_log_probs


@pytest.mark.parametrize("which", ["entropy", "top_log_probs"])
def test_entropy_and_alternatives_do_not_depend_on_the_target(which):
    torch.manual_seed(0)
    z = torch.randn(4, 9, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([-1, 9, 3, -100])
    r = token_log_probs(z, t, top=3, entropy=True)
    want = token_log_probs(z, torch.zeros_like(t), top=3, entropy=True)
    got, = torch.autograd.grad(getattr(r, which).square().sum(), z)
    assert got.isfinite().all() and torch.equal(got, torch.autograd.grad(getattr(want, which).square().sum(), z)[0])
    assert torch.autograd.gradcheck(lambda z: getattr(token_log_probs(z, t, top=3, entropy=True), which), (z,))
    r = token_log_probs(z, t, entropy=True)     # its own gradient does
    grad, = torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), z)
    assert grad[:2].isnan().all() and grad[2:].isfinite().all()
