"""Angles of far positions against numbers of 60 digits, which take nothing from the table of frequencies."""
import decimal
import math

import pytest
import torch
from test_rotary_cpu import OWN, magnitudes, values

from powersgd_b200.ops.rotary import rotate_heads

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628621")
FAR = [0, 1, -1, 1023, 2**20 - 1, 2**31 - 1, -(2**31), 2**38, -(2**38) + 7, 2**40 + 12345, 10**13, 10**15 + 7, -(2**50) - 3, 2**62]


def turns(position, i, rotated, base):
    """position * base^(-2i / rotated) / 2 pi without whole turns."""
    with decimal.localcontext() as context:
        context.prec = 60
        t = decimal.Decimal(position) * decimal.Decimal(base) ** (decimal.Decimal(-2 * i) / rotated) / (2 * PI)
        return float(t - t.to_integral_value(decimal.ROUND_FLOOR))


def check_far(dtype, rotated, interleaved, base, device="cpu"):
    """A frequency is rounded to 2^-64 turns, by 2^-65 at most, which the position multiplies; 2^-32 turns are cut off behind that (in 64 bits an angle's own
    roundings, of 2^-50). A pair moves by its magnitude times that angle."""
    x = values(len(FAR), 2, rotated, dtype, device)
    got = rotate_heads(x, positions=torch.tensor(FAR, device=device), eps=None, base=base, interleaved=interleaved).double().cpu()
    angle = 2 * math.pi * torch.tensor([[turns(p, i, rotated, base) for i in range(rotated // 2)] for p in FAR], dtype=torch.float64)[:, None]
    wide = x.double().cpu()
    a, b = (wide[..., 0::2], wide[..., 1::2]) if interleaved else wide.chunk(2, -1)
    parts = a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()
    want = torch.stack(parts, -1).flatten(-2) if interleaved else torch.cat(parts, -1)
    off = torch.tensor([2 * math.pi * (abs(p) * 2.0**-65 + (2.0**-32 if dtype != torch.float64 else 2.0**-50)) for p in FAR], dtype=torch.float64)[:, None, None]
    own = 2.0**-45 if dtype == torch.float64 else OWN
    bound = magnitudes(wide, rotated, interleaved) * (own + off) + (want.abs() * torch.finfo(dtype).eps / 2 if dtype.itemsize == 2 else 0)
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max().item()
    assert off[7].item() <= 2.0**-24      # less than float32's own rounding up to 2^38


@pytest.mark.parametrize("rotated, interleaved, base", [(16, False, 10000.0), (64, True, 10000.0), (128, False, 500000.0), (8, False, 1.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_far_positions(dtype, rotated, interleaved, base):
    check_far(dtype, rotated, interleaved, base)
