"""AdamW in torch operations: against torch.optim, 8-bit moments, checkpoints, refusals."""
import copy
import math

import pytest
import torch

from powersgd_b200 import AdamW, AllReduce, optimizer_step
from powersgd_b200.ops import adamw


def _params(*shapes, dtype=torch.float32):
    gen = torch.Generator().manual_seed(0)
    return [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype)) for s in shapes]


def _grads(params, step):
    gen = torch.Generator().manual_seed(100 + step)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen).to(p.dtype)


def test_same_as_torch():
    ours, theirs = _params((7, 9), (300,), ()), _params((7, 9), (300,), ())
    a, b = AdamW(ours, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1)
    for step in range(30):
        _grads(ours, step), _grads(theirs, step)
        a.step(), b.step()
    for p, q in zip(ours, theirs):
        torch.testing.assert_close(p, q, atol=30 * 2.0**-22, rtol=0)   # a few roundings of numbers up to 4 in each step
    a.load_state_dict(copy.deepcopy(b.state_dict()))   # names and meanings are those of torch.optim
    assert a.param_groups[0]["state_bits"] == 32 and a.state[ours[0]]["step"] == 30


def test_eight_bits_follow_thirty_two():
    narrow, wide = _params((40, 50), (700,)), _params((40, 50), (700,))
    a, b = AdamW(narrow, lr=1e-3, state_bits=8, seed=5), AdamW(wide, lr=1e-3)
    for step in range(50):
        _grads(narrow, step), _grads(wide, step)
        a.step(), b.step()
    state = a.state[narrow[0]]
    assert state["exp_avg"].dtype == torch.float8_e4m3fn and state["exp_avg_scale"].shape == (8,)
    for p, q, start in zip(narrow, wide, _params((40, 50), (700,))):
        moved = (q - start).norm()
        assert (p - q).norm() < 0.15 * moved     # 50 steps, each off by a rounding of up to 2^-3 with mean zero


def test_quantize_keeps_the_mean_and_neighbours():
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(4, 256, generator=gen) * torch.tensor([1e-6, 1.0, 1e5, 0.0])[:, None]
    total = torch.zeros(4, 256, dtype=torch.float64)
    for step in range(400):
        codes, scale = adamw.quantize(x, adamw.random_words(4, 0, step, 1) & 0xFFFF, False)
        y = codes.double() * scale.double()[:, None]
        largest = x.abs().amax(1, keepdim=True).double()
        assert ((y - x).abs() <= x.abs().double() * 2.0**-3 * (1 + 1e-6) + largest / 448 * 2.0**-9 * (1 + 1e-6)).all()   # one step of e4m3
        total += y
    # 400 draws of a two-valued variable whose values lie one step apart: six standard deviations of the mean
    step_size = torch.maximum(x.abs().double() * 2.0**-3, largest / 448 * 2.0**-9)
    assert ((total / 400 - x).abs() <= 6 * step_size * 0.5 / math.sqrt(400)).all()
    codes, scale = adamw.quantize(x.abs(), torch.zeros(4, 256, dtype=torch.int64), True)
    assert (codes.float()[:3] > 0).all() and (codes.float()[3] == 0).all() and scale[3] == 0


def test_no_number_stays_none():
    x = torch.ones(2, 256)
    x[0, 3] = math.nan
    codes, scale = adamw.quantize(x, torch.zeros(2, 256, dtype=torch.int64), False)
    assert codes.float()[0].isnan().any() and scale[0].isnan() and codes.float()[1].isfinite().all()


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpoint_continues_the_run(bits, dtype):
    one, two = _params((13, 31), (5,), dtype=dtype), _params((13, 31), (5,), dtype=dtype)
    a, b = AdamW(one, state_bits=bits, seed=9), AdamW(two, state_bits=bits, seed=9)
    for step in range(3):
        _grads(one, step)
        a.step()
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    for p, q in zip(one, two):
        q.data.copy_(p.data)
        assert {k: v.dtype for k, v in a.state[p].items()} == {k: v.dtype for k, v in b.state[q].items()}
    for step in range(3, 6):
        _grads(one, step), _grads(two, step)
        a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    c = copy.deepcopy(b)
    assert c.state_dict()["param_groups"] == b.state_dict()["param_groups"]


def test_states_of_torch_in_other_types():
    ours, theirs = _params((7, 9), dtype=torch.bfloat16), _params((7, 9), dtype=torch.bfloat16)
    a, b = AdamW(ours, lr=1e-2), torch.optim.AdamW(theirs, lr=1e-2)
    _grads(theirs, 0)
    b.step()
    state = copy.deepcopy(b.state_dict())
    assert state["state"][0]["exp_avg"].dtype == torch.bfloat16
    state["state"][0]["step"] = 1
    a.load_state_dict(state)
    _grads(ours, 1)
    a.step()
    assert a.state[ours[0]]["exp_avg"].dtype == torch.float32 and a.state[ours[0]]["step"] == 2


def test_parameters_without_gradient_and_other_layouts():
    params = _params((6, 4), (8,), (3, 5, 2, 2))
    params[2].data = params[2].data.contiguous(memory_format=torch.channels_last)
    opt = AdamW(params + [torch.nn.Parameter(torch.randn(5, 7).t())])
    last = opt.param_groups[0]["params"][3]
    params[0].grad = torch.ones(6, 4)
    params[2].grad = torch.ones(3, 5, 2, 2)      # laid out otherwise than its parameter
    last.grad = torch.randn(7, 5)
    before = params[1].detach().clone()
    opt.step()
    assert torch.equal(before, params[1]) and params[1] not in opt.state
    assert opt.state[params[0]]["step"] == 1 and opt.state[params[2]]["exp_avg"].stride() == params[2].stride()
    torch.testing.assert_close(opt.state[last]["exp_avg"], 0.1 * last.grad)


def test_behind_an_aggregator():
    params = _params((20, 30), (30,))
    opt = AdamW(params, lr=1e-2)
    _grads(params, 0)
    want = [p.grad.clone() for p in params]
    optimizer_step(opt, AllReduce())
    for p, g in zip(params, want):
        torch.testing.assert_close(opt.state[p]["exp_avg"], 0.1 * g)


@pytest.mark.parametrize("change, error", [
    (dict(lr=-1.0), ValueError), (dict(lr=torch.zeros(2)), ValueError), (dict(betas=(0.9, 1.0)), ValueError), (dict(eps=-1.0), ValueError),
    (dict(weight_decay=math.inf), ValueError), (dict(state_bits=16), ValueError), (dict(seed=2**32), ValueError),
])
def test_refused_settings(change, error):
    with pytest.raises(error):
        AdamW(_params((3,)), **change)


def test_refused_tensors():
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    gap = torch.nn.Parameter(torch.zeros(4, 6)[:, :3])
    gap.grad = torch.zeros(4, 3)
    with pytest.raises(ValueError, match="one piece"):
        AdamW([gap]).step()
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.zeros(4).to_sparse()
    with pytest.raises(TypeError, match="dense"):
        AdamW([p]).step()
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    opt = AdamW([p])
    opt.step()
    opt.param_groups[0]["state_bits"] = 8
    with pytest.raises(ValueError, match="state"):
        opt.step()
    with pytest.raises(ValueError, match="twice"):
        q = torch.nn.Parameter(torch.zeros(4))
        with pytest.warns(UserWarning):
            AdamW([q, q])


def test_parameters_in_the_same_memory_are_refused():
    x = torch.zeros(4, 6)
    for a, b in ((x, x), (x, x[1:3]), (x[2:], x[:3]), (x, x.view(6, 4))):
        with pytest.raises(ValueError, match="0 and 1 share memory"):
            AdamW([torch.nn.Parameter(a), torch.nn.Parameter(b)])
    opt = AdamW([torch.nn.Parameter(x[:2]), torch.nn.Parameter(x[2:]), torch.nn.Parameter(x[:0]), torch.nn.Parameter(torch.zeros(4, 6))])
    assert len(opt.param_groups) == 1
