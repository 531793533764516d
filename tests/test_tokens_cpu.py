"""token_log_probs in torch operations: values, gradients by differences, rows without a distribution, refusals."""
import math

import pytest
import torch

from powersgd_b200.ops.tokens import token_log_probs


def test_values_and_shapes():
    torch.manual_seed(0)
    z = torch.randn(4, 5, 17)
    t = torch.randint(0, 17, (4, 5), dtype=torch.int32)
    t[1, 2] = -100
    r = token_log_probs(z, t, top=4, entropy=True, temperature=0.8)
    want = torch.log_softmax(z.double() / 0.8, -1)
    picked = want.gather(-1, t.clamp_min(0).long()[..., None])[..., 0]
    picked[1, 2] = 0.0
    torch.testing.assert_close(r.log_probs.double(), picked, atol=2e-6, rtol=0)
    torch.testing.assert_close(r.entropy.double(), -(want.exp() * want).sum(-1), atol=4e-6, rtol=0)
    assert r.top_tokens.shape == (4, 5, 4) and r.top_tokens.dtype == torch.int64
    assert torch.equal(r.top_tokens, torch.topk(want, 4, -1).indices)
    plain = token_log_probs(z, t)
    assert plain.entropy is None and plain.top_tokens is None and plain.top_log_probs is None


def test_gradients_by_differences():
    torch.manual_seed(1)
    z = torch.randn(6, 9, dtype=torch.float64, requires_grad=True)
    t = torch.randint(0, 9, (6,))
    t[3] = -100
    assert torch.autograd.gradcheck(lambda z: token_log_probs(z, t, top=3, entropy=True, temperature=0.7)[:3], (z,))
    assert torch.autograd.gradcheck(lambda z: token_log_probs(z, t)[0], (z,))


def test_gradient_of_broadcast_logits():
    z = torch.randn(1, 8, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([1, 5, 5])
    assert torch.autograd.gradcheck(lambda z: token_log_probs(z.expand(3, 8), t, entropy=True)[:2], (z,))


def test_rows_without_a_distribution():
    inf = math.inf
    z = torch.tensor([[-inf] * 5, [0.0, -inf, 1.0, -inf, -inf], [torch.finfo(torch.float32).min] * 5, [0.0, inf, 0.0, 0.0, 0.0],
                      [0.0, math.nan, 0.0, 0.0, 0.0], [0.0] * 5, [0.0] * 5], requires_grad=True)
    t = torch.tensor([1, 0, 4, 0, 0, 5, -1])
    r = token_log_probs(z, t, top=3, entropy=True)
    assert r.log_probs[0] == -inf and r.entropy[0] == 0 and torch.equal(r.top_log_probs[0], torch.full((3,), -inf))
    assert torch.equal(r.top_tokens[0], torch.tensor([0, 1, 2]))
    assert r.top_tokens[1].tolist() == [2, 0, 1] and r.top_log_probs[1, 2] == -inf
    torch.testing.assert_close(r.log_probs[2].item(), -math.log(5), atol=1e-6, rtol=0)
    torch.testing.assert_close(r.entropy[2].item(), math.log(5), atol=1e-6, rtol=0)
    assert r.log_probs[3].isnan() and r.log_probs[4].isnan()
    assert r.log_probs[5].isnan() and r.log_probs[6].isnan()   # targets outside the vocabulary
    assert r.entropy[5].item() == pytest.approx(math.log(5), abs=1e-6)
    (r.log_probs[:3].sum() + r.entropy[:3].sum()).backward()
    assert torch.equal(z.grad[0], torch.zeros(5)) and z.grad[:3].isfinite().all()


def test_nothing_to_do():
    r = token_log_probs(torch.zeros(0, 7), torch.zeros(0, dtype=torch.int64), top=2, entropy=True)
    assert r.log_probs.shape == (0,) and r.top_tokens.shape == (0, 2)
    one = token_log_probs(torch.randn(3, 1), torch.zeros(3, dtype=torch.int64), top=1, entropy=True)
    assert torch.equal(one.log_probs, torch.zeros(3)) and torch.equal(one.entropy, torch.zeros(3))


@pytest.mark.parametrize("change, error", [
    (dict(logits=torch.zeros(3, 8, dtype=torch.int32)), TypeError), (dict(targets=torch.zeros(3)), TypeError), (dict(targets=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(top=9), ValueError), (dict(top=-1), ValueError), (dict(temperature=0.0), ValueError), (dict(temperature=math.inf), ValueError), (dict(temperature=1e-40), ValueError),
    (dict(logits=torch.zeros(3, 0)), ValueError), (dict(logits=torch.zeros(3, 64), top=33), ValueError), (dict(ignore_index=2**63), ValueError),
])
def test_refusals(change, error):
    call = dict(logits=torch.zeros(3, 8), targets=torch.zeros(3, dtype=torch.int64))
    call.update(change)
    with pytest.raises(error):
        token_log_probs(call.pop("logits"), call.pop("targets"), **call)
