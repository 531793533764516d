"""The norm of many gradients and clipping, in torch operations, and what both refuse.

Bounds: sums of squares in 64 bits, so a norm is off by its own rounding (2^-24) and a little; a scaled gradient by those of the factor and the product
(2^-24 each) and half a step of its type."""
import math

import pytest
import torch

from powersgd_b200 import clip_grad_norm, grad_norm
from powersgd_b200.ops import grad_norm as module

TYPES = [torch.float32, torch.bfloat16, torch.float16, torch.float64]


def make(shapes, dtypes, device="cpu", scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    params = []
    for i, shape in enumerate(shapes):
        p = torch.nn.Parameter(torch.zeros(shape, dtype=dtypes[i % len(dtypes)], device=device))
        p.grad = (torch.randn(shape, generator=gen, dtype=torch.float64) * torch.exp(torch.randn(shape, generator=gen, dtype=torch.float64)) * scale).to(p.dtype).to(device)
        params.append(p)
    return params


def exact(params, norm_type):
    parts = [p.grad.detach().double().flatten().cpu() for p in params if p.grad is not None]
    flat = torch.cat(parts) if parts else torch.zeros(1, dtype=torch.float64)
    return math.sqrt(math.fsum((flat * flat).tolist())) if norm_type == 2 else flat.abs().max().item()


def check(params, max_norm, norm_type=2.0, call=clip_grad_norm):
    """Clips and compares with 64 bits."""
    before = [None if p.grad is None else p.grad.detach().double().clone() for p in params]
    norm = exact(params, norm_type)
    factor = min(1.0, max_norm / (norm + 1e-6))
    assert abs(grad_norm(params, norm_type).item() - norm) <= norm * 2.0**-23
    got = call(params, max_norm, norm_type)
    wide = any(p.grad is not None and p.grad.dtype == torch.float64 for p in params)
    assert got.shape == () and got.dtype == (torch.float64 if wide else torch.float32)
    assert abs(got.item() - norm) <= norm * (2.0**-50 if wide else 2.0**-23)
    for p, b in zip(params, before):
        if b is None:
            continue
        if factor == 1:
            assert torch.equal(p.grad.double(), b)
            continue
        want, info = b * factor, torch.finfo(p.dtype)
        own = 2.0**-50 if p.dtype == torch.float64 else 2.0**-22.9
        half = 0.0 if p.dtype in (torch.float32, torch.float64) else info.eps / 2
        bound = want.abs() * (half + own) + info.smallest_normal * info.eps     # (below the normal numbers steps do not shrink)
        assert ((p.grad.double() - want).abs() <= bound).all()


SHAPES = [(1,), (3, 5), (), (0,), (257,), (64, 33), (2, 3, 4, 5), (1000, 13)]


@pytest.mark.parametrize("norm_type", [2, 2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("max_norm", [0.0, 0.4, 1e9, math.inf])
def test_against_64_bits(dtypes, max_norm, norm_type):
    check(make(SHAPES, dtypes), max_norm, norm_type)


def test_same_as_torch():
    a, b = make(SHAPES, TYPES[:1]), make(SHAPES, TYPES[:1])
    want = torch.nn.utils.clip_grad_norm_(a, 0.4)
    torch.testing.assert_close(clip_grad_norm(b, 0.4), want, rtol=1e-5, atol=0)
    for p, q in zip(a, b):
        torch.testing.assert_close(q.grad, p.grad, rtol=1e-5, atol=1e-9)


def test_one_tensor_generators_and_none():
    params = make([(5,), (7,)], TYPES[:1])
    params[1].grad = None
    want = exact(params, 2)
    assert grad_norm(params[0]).item() == pytest.approx(want) and grad_norm(p for p in params).item() == pytest.approx(want)
    check(params, 0.1)
    for nothing in ([], [params[1]], make([(0,)], TYPES[:1])):
        out = clip_grad_norm(nothing, 1.0)
        assert out.item() == 0 and out.dtype == torch.float32 and out.shape == ()


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_what_is_not_finite(norm_type):
    def values(bad):
        params = make([(5,), (7,)], TYPES[:1])
        params[0].grad[2] = bad
        return params

    for bad, want in ((math.nan, math.nan), (math.inf, math.inf), (-math.inf, math.inf)):
        params = values(bad)
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="norm of the gradients"):
            clip_grad_norm(params, 1.0, norm_type, error_if_nonfinite=True)
        assert all(torch.equal(p.grad.nan_to_num(5.0), b.nan_to_num(5.0)) for p, b in zip(params, before))
        twin = values(bad)
        got, theirs = clip_grad_norm(params, 1.0, norm_type), torch.nn.utils.clip_grad_norm_(twin, 1.0, norm_type)
        assert got.isnan() if math.isnan(want) else got.item() == want
        assert theirs.isnan() == got.isnan()
        for p, q in zip(params, twin):
            assert torch.equal(p.grad.isnan(), q.grad.isnan()) and torch.equal(p.grad.nan_to_num(7.0), q.grad.nan_to_num(7.0))
    params = values(1.0)
    clip_grad_norm(params, 1.0, norm_type, error_if_nonfinite=True)


def test_large_and_small_gradients():
    """Squares that float32 does not hold."""
    for scale, dtype in ((1e30, torch.float32), (1e-30, torch.float32), (1e30, torch.bfloat16), (1e-30, torch.bfloat16)):
        params = make([(100,), (33, 3)], [dtype], scale=scale)
        norm = exact(params, 2)
        assert abs(grad_norm(params).item() - norm) <= norm * 2.0**-23
        if scale > 1:
            check(params, 0.5 * norm)


def refused(device):
    """Calls that raise and change nothing."""
    p = make([(4, 6)], TYPES[:1], device)[0]
    twin = torch.nn.Parameter(torch.zeros(4, 6, device=device))
    twin.grad = p.grad
    part = torch.nn.Parameter(torch.zeros(2, 6, device=device))
    part.grad = p.grad[1:3]
    same = torch.nn.Parameter(torch.zeros(4, 6, device=device))
    same.grad = torch.ones(6, device=device).expand(4, 6)
    sparse = torch.nn.Parameter(torch.zeros(4, 6, device=device))
    sparse.grad = torch.eye(4, 6, device=device).to_sparse()
    complex_ = torch.nn.Parameter(torch.zeros(4, dtype=torch.complex64, device=device))
    complex_.grad = torch.ones(4, dtype=torch.complex64, device=device)
    yield lambda: clip_grad_norm([p, p], 1e-3), ValueError, "share memory"
    yield lambda: clip_grad_norm([p, twin], 1e-3), ValueError, "share memory"
    yield lambda: clip_grad_norm([part, p], 1e-3), ValueError, "share memory"
    yield lambda: clip_grad_norm([p, same], 1e-3), ValueError, "share memory"
    yield lambda: clip_grad_norm([p, sparse], 1e-3), TypeError, "dense"
    yield lambda: clip_grad_norm([p, complex_], 1e-3), TypeError, "complex64"
    yield lambda: grad_norm([p, complex_]), TypeError, "complex64"
    for bad in (-1.0, math.nan):
        yield lambda bad=bad: clip_grad_norm([p], bad), ValueError, "max_norm"
    for bad in (1, 3.0, 0, -math.inf, math.nan):
        yield lambda bad=bad: clip_grad_norm([p], 1e-3, bad), ValueError, "norm_type"
        yield lambda bad=bad: grad_norm([p], bad), ValueError, "norm_type"
    yield None, p, None


def check_refusals(device):
    calls = list(refused(device))
    p = calls[-1][1]
    before = p.grad.clone()
    for call, error, match in calls[:-1]:
        with pytest.raises(error, match=match):
            call()
        assert torch.equal(p.grad, before)


def test_refusals():
    check_refusals("cpu")


def layouts(device):
    """Gradients in other orders of dimensions, with gaps, negated views and zeros that have no memory."""
    params = []
    for g in (torch.randn(6, 10, device=device).t(), torch.randn(8, 6, 3, 3, device=device).contiguous(memory_format=torch.channels_last), torch.randn(20, 30, device=device)[::2, 3:17],
              torch._neg_view(torch.randn(50, device=device)), torch.randn(101, device=device)[1:], torch._efficientzerotensor((5,), device=device)):
        p = torch.nn.Parameter(torch.zeros(g.shape, device=device, dtype=g.dtype))
        p.grad = g
        params.append(p)
    return params


def check_counted_twice(device):
    p = make([(300,)], TYPES[:1], device)[0]
    twin = torch.nn.Parameter(torch.zeros(100, device=device))
    twin.grad = p.grad[50:150]
    norm = exact([p, p, twin], 2)
    assert abs(grad_norm([p, p, twin]).item() - norm) <= norm * 2.0**-23


def test_counted_twice():
    check_counted_twice("cpu")


def test_layouts():
    check(layouts("cpu"), 0.4)


def test_autograd_knows():
    """A gradient that a later backward pass needs was changed: told, as torch operations tell it."""
    p = make([(4,)], TYPES[:1])[0]
    x = torch.ones(4, requires_grad=True)
    loss = (x * p.grad).sum()
    clip_grad_norm([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_the_item_of_a_list():
    assert module.ITEM.itemsize == 24


def test_language_model_task_and_train_step_clip():
    from powersgd_b200 import AllReduce
    from powersgd_b200.engine import TrainStep

    torch.manual_seed(0)
    model = torch.nn.Linear(8, 4)
    optimizer = torch.optim.SGD(model.parameters(), lr=1.0)
    before = [p.detach().clone() for p in model.parameters()]
    step = TrainStep(model, torch.nn.functional.cross_entropy, optimizer, AllReduce(), grad_clip=1e-3)
    step(100 * torch.randn(16, 8), torch.randint(0, 4, (16,)))
    moved = torch.cat([(p - b).flatten() for p, b in zip(model.parameters(), before)]).double().norm()
    assert abs(moved - 1e-3) <= 1e-4     # weights near one move by a hundredth of that: their own roundings are 6e-8 each
