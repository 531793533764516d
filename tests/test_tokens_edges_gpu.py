"""token_log_probs on the GPU where it can go wrong, against float64. Bounds as in test_tokens_gpu.py."""
import math

import pytest
import torch

from powersgd_b200.ops.tokens import token_log_probs

pytestmark = pytest.mark.gpu


def _logits(rows, vocab, dtype, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen, device="cuda") * 2).to(dtype), torch.randint(0, vocab, (rows,), generator=gen, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, vocab", [(1, 4096), (1, 8192), (3, 8195), (1, 32768), (5, 32771), (36, 32768), (37, 50257), (147, 8192)])
def test_rows_shared_by_blocks(rows, vocab, dtype):
    """Few rows: two, four or eight blocks to a row, which bring their parts together in the shared memory of the first. Some rows are ignored: their
    blocks leave at once."""
    z, t = _logits(rows, vocab, dtype)
    log_p = torch.log_softmax(z.double(), 1)
    at = log_p.gather(1, t[:, None])[:, 0]
    base = (vocab / 64 + 24) * 2.0**-24 + 2.0**-22 + 16 * 2.0**-22      # log p of a row's mean: below 16
    best = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :7]
    for _ in range(20):
        plain, both = token_log_probs(z, t), token_log_probs(z, t, top=7, entropy=True)
        for r in (plain, both):
            assert ((r.log_probs.double() - at).abs() <= base + at.abs() * 2.0**-22).all()
        assert torch.equal(both.top_tokens, best)
    ignored = torch.where(torch.arange(rows, device="cuda") % 2 == 0, t, torch.full_like(t, -100))
    assert torch.equal(token_log_probs(z, ignored).log_probs, torch.where(ignored == -100, 0.0, plain.log_probs))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows, vocab", [(4, 700), (3, 5003), (300, 8191), (2, 50257)])
def test_more_equal_logits_than_candidates(rows, vocab, dtype):
    """Every warp then keeps a list, under a bound that all warps of the block raise; the last round of vectors is a partial one."""
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    z = torch.randint(0, 3, (rows, vocab), generator=gen, device="cuda").to(dtype)
    z[:, vocab // 2:] += (torch.arange(vocab - vocab // 2, device="cuda") // 600).to(dtype) / 8      # bounds that rise as the row is read
    t = torch.zeros(rows, device="cuda", dtype=torch.int64)
    for top in (1, 20, 32):
        want = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
        for _ in range(10):
            assert torch.equal(token_log_probs(z, t, top=top).top_tokens, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [40, 5003])
def test_entropy_and_alternatives_do_not_depend_on_the_target(vocab, dtype):
    """Their gradients with targets outside the vocabulary: the same as with any other, and those of 64 bits. p is off by 2^-20 of itself and
    2^-21 for each unit of its logarithm (below 16 where it counts), the gradient by half a step of its type."""
    z, _ = _logits(6, vocab, dtype)
    z.requires_grad_()
    t = torch.tensor([-1, vocab, 3, -100, vocab + 5, -7], device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    gh, gt = torch.randn(6, generator=gen, device="cuda"), torch.randn(6, 4, generator=gen, device="cuda")
    log_p = torch.log_softmax(z.detach().double(), 1)
    p = log_p.exp()
    h = torch.special.entr(p).sum(1, keepdim=True)
    best = torch.sort(z.detach(), dim=1, descending=True, stable=True).indices[:, :4]
    for which, g, want, size in (("entropy", gh, gh[:, None].double() * (torch.special.entr(p) - p * h), gh[:, None].double().abs() * (torch.special.entr(p) + p * h)),
                                 ("top_log_probs", gt, torch.zeros_like(p).scatter_(1, best, gt.double()) - p * gt.double().sum(1, keepdim=True),
                                  torch.zeros_like(p).scatter_(1, best, gt.double().abs()) + p * gt.double().abs().sum(1, keepdim=True))):
        got, = torch.autograd.grad(getattr(token_log_probs(z, t, top=4, entropy=True), which), z, g)
        other, = torch.autograd.grad(getattr(token_log_probs(z, torch.zeros_like(t), top=4, entropy=True), which), z, g)
        assert torch.equal(got, other)
        least = 2.0**-25 if dtype == torch.float16 else 1e-36
        bound = size * (2.0**-17 + (vocab / 64 + 24) * 2.0**-22) + want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + least
        assert ((got.double() - want).abs() <= bound).all()
