"""packed_attention in torch operations: against one sequence at a time, gradients by differences, refusals."""
import math

import pytest
import torch

from powersgd_b200.ops.attention import packed_attention


def _offsets(*lengths):
    return torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)


@pytest.mark.parametrize("causal", [True, False])
def test_each_sequence_by_itself(causal):
    torch.manual_seed(0)
    q, k, v = torch.randn(12, 4, 8), torch.randn(12, 2, 8), torch.randn(12, 2, 8)
    out = packed_attention(q, k, v, _offsets(5, 0, 1, 4), causal=causal)
    for lo, hi in ((0, 5), (5, 6), (6, 10)):
        part = [x[lo:hi].transpose(0, 1) for x in (q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1))]
        want = torch.nn.functional.scaled_dot_product_attention(*part, is_causal=causal).transpose(0, 1)
        torch.testing.assert_close(out[lo:hi], want, atol=1e-6, rtol=0)
    assert (out[10:] == 0).all()      # rows behind the last sequence


@pytest.mark.parametrize("causal", [True, False])
def test_gradients_by_differences(causal):
    torch.manual_seed(1)
    q, k, v = (torch.randn(7, n, 8, dtype=torch.float64, requires_grad=True) for n in (4, 2, 2))
    assert torch.autograd.gradcheck(lambda *x: packed_attention(*x, _offsets(3, 2, 0, 1), causal=causal, scale=0.4), (q, k, v))


def test_shared_and_broadcast_inputs():
    torch.manual_seed(2)
    x = torch.randn(5, 1, 8, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x: packed_attention(x.expand(5, 4, 8), x, x, _offsets(5)), (x,))


def test_rows_outside_may_hold_anything():
    q, k, v = (torch.randn(9, 2, 8) for _ in range(3))
    want = packed_attention(q, k, v, torch.tensor([2, 7], dtype=torch.int32))
    for x in (q, k, v):
        x[:2] = math.nan
        x[7:] = math.inf
    assert torch.equal(packed_attention(q, k, v, torch.tensor([2, 7], dtype=torch.int32)), want)
    assert (want[:2] == 0).all() and (want[7:] == 0).all()


def test_bad_offsets_stay_inside():
    q, k, v = (torch.randn(9, 2, 8) for _ in range(3))
    for bad in ([-5, 4, 100], [0, 20, 3], [50, 60]):
        packed_attention(q, k, v, torch.tensor(bad, dtype=torch.int32))


def test_nothing_to_do():
    q = torch.zeros(0, 2, 8)
    assert packed_attention(q, q, q, _offsets(0)).shape == (0, 2, 8)
    q = torch.ones(3, 2, 8)
    assert (packed_attention(q, q, q, torch.zeros(1, dtype=torch.int32)) == 0).all()


@pytest.mark.parametrize("change, error", [
    (dict(q=torch.zeros(4, 3, 8)), ValueError), (dict(q=torch.zeros(5, 4, 8)), ValueError), (dict(q=torch.zeros(4, 4, 16)), ValueError),
    (dict(v=torch.zeros(4, 4, 8)), ValueError), (dict(k=torch.zeros(4, 2, 8, dtype=torch.float64)), TypeError), (dict(offsets=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(offsets=torch.zeros(0, dtype=torch.int32)), ValueError), (dict(offsets=torch.zeros(2, 2, dtype=torch.int32)), ValueError), (dict(scale=0.0), ValueError),
    (dict(scale=math.nan), ValueError), (dict(q=torch.zeros(4, 4, 12), k=torch.zeros(4, 2, 12), v=torch.zeros(4, 2, 12)), ValueError),
    (dict(q=torch.zeros(4, 4, 136), k=torch.zeros(4, 2, 136), v=torch.zeros(4, 2, 136)), ValueError), (dict(q=torch.zeros(4, 4, 8).int(), k=torch.zeros(4, 2, 8).int(), v=torch.zeros(4, 2, 8).int()), TypeError),
])
def test_refusals(change, error):
    call = dict(q=torch.zeros(4, 4, 8), k=torch.zeros(4, 2, 8), v=torch.zeros(4, 2, 8), offsets=_offsets(4))
    call.update(change)
    with pytest.raises(error):
        packed_attention(call.pop("q"), call.pop("k"), call.pop("v"), call.pop("offsets"), **call)


@pytest.mark.parametrize("scale", [0.0, -1.0, 2.0**-101, 2.0**101, math.inf, math.nan])
def test_refused_scales(scale):
    x = torch.zeros(3, 1, 8)
    with pytest.raises(ValueError, match="scale"):
        packed_attention(x, x, x, torch.tensor([0, 3], dtype=torch.int32), scale=scale)
