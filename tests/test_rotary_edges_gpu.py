"""Rows that more warps would share than a launch of gradients has, weights' gradients of many rows, products that leave the range, far positions."""
import pytest
import torch
from test_rotary_cpu import check, values
from test_rotary_edges_cpu import check_far

from powersgd_b200.ops import host, rotary
from powersgd_b200.ops.rotary import rotate_heads

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(rotary, "operators", None)
    else:
        assert host.operators is not None
    return request.param


@pytest.mark.parametrize("heads, keys, values_, size", [(3000, 1096, 0, 256), (1096, 3000, 0, 256), (2400, 1184, 8, 136), (2369, 1, 0, 256), (2050, 2040, 6, 200)])
@pytest.mark.parametrize("rows", [1, 2])
def test_queries_and_keys_share_the_warps_of_a_launch(form, rows, heads, keys, values_, size):
    """Each kind alone may take half of the warps and more; both together have to find room."""
    torch.empty(rows, heads + keys + values_, size, device="cuda").fill_(float("nan"))     # (what an output that is not written may hold)
    check(values(rows, heads + keys + values_, size, torch.float32, "cuda"), heads, keys, lengths=[rows])


@pytest.mark.parametrize("rows, heads", [(2**22, 1), (2**20, 4), (2**19, 40)])
def test_weights_gradients_of_many_rows(form, rows, heads):
    """Products that are all 1 + 2^-17: up to 64 of them add up exactly in 32 bits, and any number in 64, while a sum of 32 bits loses the 2^-17 from 128 on. What
    is left of a bound is the reciprocal root of one, two steps of 2^-23, and the last rounding."""
    x = torch.ones(rows, heads, 8, device="cuda")
    w = torch.ones(8, device="cuda", requires_grad=True)
    z = rotate_heads(x, weight=w, eps=2.0**-100, rotated=0)
    got, = torch.autograd.grad(z, w, torch.full_like(z, 1 + 2.0**-17))
    want = rows * heads * (1 + 2.0**-17)
    assert ((got.double() - want).abs() <= want * (2 * 2.0**-23 + 2.0**-24)).all(), (got.double() / want - 1).abs().max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_gradients_of_large_heads(form, dtype):
    """Products of a gradient and a head leave the range of float32; what they are the mean of, over the head's norm, does not. The same numbers times powers of two
    give the same but for numbers below 2^-126, which are far below a head's largest, and a rounding to the type: the bound leaves room for more."""
    x, g = values(9, 4, 64, dtype, "cuda") * 2.0**50, values(9, 4, 64, dtype, "cuda", seed=1) * 2.0**100
    one, two = ((x * s).requires_grad_() for s in (1.0, 2.0**-50))
    at = torch.arange(9, device="cuda")
    a, = torch.autograd.grad(rotate_heads(one, positions=at, eps=2.0**-100), one, g)
    b, = torch.autograd.grad(rotate_heads(two, positions=at, eps=2.0**-100), two, g * 2.0**-100)
    assert a.isfinite().all()
    assert ((a.double() * 2.0**-50 - b.double()).abs() <= b.double().abs().amax(-1, keepdim=True) * (2.0**-18 + torch.finfo(dtype).eps)).all()


@pytest.mark.parametrize("rotated, interleaved, base", [(16, False, 10000.0), (64, True, 10000.0), (128, False, 500000.0), (8, False, 1.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_far_positions(form, dtype, rotated, interleaved, base):
    check_far(dtype, rotated, interleaved, base, "cuda")


@pytest.mark.parametrize("size", [16, 40, 136, 256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_more_rows_than_are_added_up_at_a_time(form, dtype, size):
    """A warp comes to 84 rows; with and without gradients of weights."""
    rows = 100_000
    check(values(rows, 3, size, dtype, "cuda"), 1, 1, lengths=[rows // 3, rows // 2], rotated=0)
    check(values(rows, 1, size, dtype, "cuda"), 1, 0, lengths=[rows], weights=False, rotated=0)


@pytest.mark.parametrize("scale", [1.0, 2.0**-8, 2.0**18])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_near_the_end_of_the_range(form, dtype, scale):
    """Where their products with a small head leave float32, or where one of them is infinite, the weights' gradients (products with normed elements, here of one row)
    are what they are. Bounds: as for sums of one product (five roundings on the way to a normed element, one of the product, one at the end)."""
    for spoiled in (False, True):
        x = (values(1, 1, 64, dtype, "cuda").abs() + 0.5) * scale
        g = (1 + values(1, 1, 64, dtype, "cuda", seed=1).abs().clamp(max=0.5)) * 2.0**124
        if spoiled:
            g[0, 0, 5] = float("inf")
        w = torch.ones(64, device="cuda", requires_grad=True)
        got, = torch.autograd.grad(rotate_heads(x, weight=w, eps=1e-6, rotated=0), w, g)
        wide = x.double()[0, 0]
        want = g.double()[0, 0] * wide / (wide.square().mean() + 1e-6).sqrt()
        if spoiled:
            assert got[5] == float("inf")
            got, want = got[torch.arange(64) != 5], want[torch.arange(64) != 5]
        assert ((got.double() - want).abs() <= want * 8 * 2.0**-24).all()
