"""packed_attention on the GPU where it can go wrong."""
import math

import pytest
import torch

from powersgd_b200.ops.attention import packed_attention

pytestmark = pytest.mark.gpu


def _offsets(lengths, first=0):
    return torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)


def _inputs(tokens, heads, groups, size, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda n: (torch.randn(tokens, n, size, generator=gen, device="cuda") * scale).to(dtype)  # noqa: E731
    return make(heads), make(groups), make(groups), make(heads)


def test_offsets_that_go_down_again_and_again():
    """2^24 and more sequences of 128 tiles each over the same rows: their tiles, more than 2^31, are counted without overflow, and what the grid
    has no room for is left. What such offsets give is not defined, but nothing is written elsewhere."""
    tokens, turns = 2**14, 2**24 + 2**21
    offsets = torch.zeros(2 * turns, device="cuda", dtype=torch.int32)
    offsets[1::2] = tokens
    whole = torch.zeros(3, tokens, 1, 16, device="cuda", dtype=torch.bfloat16)
    q, k, v = whole.unbind(0)
    guard = torch.full((2**26,), 7, device="cuda", dtype=torch.int32)
    packed_attention(q, k, v, offsets)
    torch.cuda.synchronize()
    assert (guard == 7).all() and (whole == 0).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("size", [64, 128])
def test_scores_that_are_no_numbers(size, bad, causal):
    """One key of a sequence: positions that see a score of NaN (or +inf, whose softmax is none) give NaN, as the form in torch operations does,
    wherever in a tile the key lies."""
    for place in (0, 1, 2, 16, 17, 40, 123, 124, 127, 128, 130, 250):
        q, k, v, _ = _inputs(300, 2, 1, size, torch.bfloat16, seed=place)
        k[20 + place] = bad if math.isnan(bad) else k[20 + place]
        if math.isinf(bad):
            k[20 + place, 0, 3] = bad
        offsets = torch.tensor([0, 20, 280, 300], device="cuda", dtype=torch.int32)
        got = packed_attention(q, k, v, offsets, causal=causal)
        want = packed_attention(*(x.cpu().float() for x in (q, k, v)), offsets.cpu(), causal=causal)
        assert torch.equal(got.isnan().cpu(), want.isnan()), place
        fine = ~want.isnan()
        assert want.isnan().any() and fine.any()
        # a weight is off by 2^-8 of itself and 2^-12 (its score), the output by half a step, 2^-8
        assert ((got.cpu().float() - want)[fine].abs() <= (2.0**-7 + 2.0**-11) * v.abs().max().item()).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("until", [128, 150, 256, 300])
def test_scores_of_minus_infinity_come_first(until, size, causal):
    """Keys whose scores are -inf have no weight, also where whole tiles of them come before all others."""
    q, k, v, _ = _inputs(500, 2, 1, size, torch.bfloat16, seed=until)
    q[..., 3] = q[..., 3].abs() + 0.25
    k[:until, :, 3] = -math.inf
    got = packed_attention(q, k, v, _offsets([500]), causal=causal)
    want = packed_attention(*(x.cpu().float() for x in (q, k, v)), _offsets([500]).cpu(), causal=causal)
    assert torch.equal(got.isnan().cpu(), want.isnan()) and want[until:].isfinite().all()
    assert ((got.cpu().float() - want)[until:].abs() <= (2.0**-7 + 2.0**-11) * v.abs().max().item()).all()
