"""token_log_probs on the GPU against float64. Bounds count roundings: a log of a sum of V exponentials has at most
V / 256 + 16 additions in a row (2^-24 each), exponentials of 2^-22 and arguments of 2^-23 |z - m| / T; a gradient has
twice that relative to its terms, and half a step of its own type."""
import math

import pytest
import torch

from powersgd_b200.ops.tokens import _grad_like, _rows, token_log_probs

pytestmark = pytest.mark.gpu


def _reference(z, t, top, temperature, ignore_index=-100):
    z = z.detach().double()
    log_p = torch.log_softmax(z / temperature, -1)
    p = log_p.exp()
    entropy = torch.special.entr(p).sum(-1)
    known = (t != ignore_index)
    lp = torch.where(known, log_p.gather(-1, t.clamp_min(0).long()[..., None])[..., 0], 0.0)
    tokens = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :top]
    return log_p, p, lp, entropy, tokens


def _check(z, t, top=0, entropy=False, temperature=1.0, gradients=("g",), ignore_index=-100):
    leaf = z.detach().requires_grad_() if gradients else z
    r = token_log_probs(leaf, t, top=top, entropy=entropy, temperature=temperature, ignore_index=ignore_index)
    log_p, p, lp, h, tokens = _reference(z, t, top, temperature, ignore_index)
    vocab = z.shape[-1]
    spread = torch.where(log_p.isfinite(), log_p, 0.0).abs()
    base = (vocab / 64 + 24) * 2.0**-24 + 2.0**-22 + (p * spread).sum(-1) * 2.0**-22      # log s
    assert ((r.log_probs.double() - lp).abs() <= base + lp.abs() * 2.0**-22).all()
    if entropy:
        assert ((r.entropy.double() - h).abs() <= 4 * base * (1 + h) + 1e-6).all()
    if top:
        assert torch.equal(r.top_tokens, tokens)
        want = log_p.gather(-1, tokens)
        fine = want.isfinite()
        assert torch.equal(fine, r.top_log_probs.isfinite())
        assert ((r.top_log_probs.double() - want).abs()[fine] <= (base[..., None] + want.abs() * 2.0**-22)[fine]).all()
    if not gradients:
        return
    outs, grads = [], []
    dz = torch.zeros_like(p)
    size = torch.zeros_like(p)
    gen = torch.Generator(device="cuda").manual_seed(3)
    live = (t != ignore_index)
    if "g" in gradients:
        g = torch.randn(t.shape, generator=gen, device="cuda")
        outs.append(r.log_probs), grads.append(g)
        one = torch.zeros_like(p).scatter_(-1, t.clamp_min(0).long()[..., None], live.double()[..., None])
        dz += g.double()[..., None] * (one - p * live[..., None])
        size += g.double().abs()[..., None] * p
    if "h" in gradients:
        gh = torch.randn(t.shape, generator=gen, device="cuda")
        outs.append(r.entropy), grads.append(gh)
        dz += gh.double()[..., None] * (torch.special.entr(p) - p * h[..., None])
        size += gh.double().abs()[..., None] * (torch.special.entr(p) + p * h[..., None])
    if "top" in gradients:
        gt = torch.randn(r.top_log_probs.shape, generator=gen, device="cuda")
        outs.append(r.top_log_probs), grads.append(gt)
        dz += torch.zeros_like(p).scatter_(-1, tokens, gt.double()) - p * gt.double().sum(-1, keepdim=True)
        size += p * gt.double().abs().sum(-1, keepdim=True)
    dz /= temperature
    got, = torch.autograd.grad(outs, leaf, grads)
    assert got.dtype == z.dtype and got.shape == z.shape
    rel = 4 * base[..., None] + spread * 2.0**-21 + 2.0**-20
    smallest = {torch.float32: 1e-36, torch.bfloat16: 1e-36, torch.float16: 2.0**-25}[z.dtype]
    bound = size / temperature * rel + dz.abs() * (torch.finfo(z.dtype).eps / 2 + 2.0**-22) + smallest
    off = (got.double() - dz).abs()
    assert (off <= bound).all(), (off / bound).max().item()


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 2), (2, 7), (5, 31), (1, 300), (7, 512), (3, 2049), (2, 4099), (9, 10007), (1, 50257), (2, 65536), (5, 131072)])
def test_sizes(rows, vocab, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows * 1000 + vocab)
    z = (torch.randn(rows, vocab, generator=gen, device="cuda") * 3).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    top = min(vocab, 8)
    _check(z, t)
    _check(z, t, top=top, entropy=True, gradients=("g", "h", "top"), temperature=0.7)
    _check(z, t, top=min(vocab, 32), gradients=("top",))
    _check(z, t, entropy=True, gradients=("h",))
    _check(z, t, top=1, gradients=())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 30, 150, 400, 1200])
def test_numbers_of_rows(rows, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows)
    z = (torch.randn(rows, 9001, generator=gen, device="cuda") * 2).to(dtype)
    t = torch.randint(0, 9001, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    t[::3] = -100
    _check(z, t, top=5, entropy=True, gradients=("g", "h"))
    _check(z, t)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    gen = torch.Generator(device="cuda").manual_seed(7)
    whole = torch.randn(6, 5, 1031, generator=gen, device="cuda").to(dtype)
    t = torch.randint(0, 1000, (6, 5), generator=gen, device="cuda")
    for z in (whole[..., :1000], whole[..., 1:1001], whole[..., 3:1004], whole[:, ::2, :1000], whole.transpose(0, 1)[..., :1000], whole.new_zeros(6, 1000, 5).transpose(1, 2),
              whole[:1, :, :1000].expand(6, 5, 1000)):
        _check(z, t[:, : z.shape[1]] if z.shape[0] == 6 else t.t(), top=3, entropy=True, gradients=("g", "h", "top"))
    shifted = whole[..., 1:1001]
    grad, rows = _grad_like(shifted, _rows(shifted))
    assert grad.shape == shifted.shape and (rows.data_ptr() - _rows(shifted).data_ptr()) % 16 == 0


def test_gradient_is_accumulated_over_a_broadcast():
    z = torch.randn(1, 777, device="cuda", requires_grad=True)
    t = torch.tensor([4, 700, 4], device="cuda")
    token_log_probs(z.expand(3, 777), t).log_probs.sum().backward()
    p = torch.softmax(z.detach().double(), 1)
    want = -3 * p
    want[0, 4] += 2
    want[0, 700] += 1
    torch.testing.assert_close(z.grad.double(), want, atol=1e-5, rtol=0)


@pytest.mark.parametrize("vocab", [5, 5000, 40000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_a_distribution(dtype, vocab):
    inf = math.inf
    z = torch.zeros(9, vocab, device="cuda", dtype=dtype)
    z[0] = -inf
    z[1, 1:] = -inf
    z[2] = torch.finfo(dtype).min
    z[3, 1] = inf
    z[4, vocab - 1] = math.nan
    z[7, : vocab - 2] = torch.finfo(dtype).min
    z.requires_grad_()
    t = torch.tensor([1, 0, 4, 0, 0, vocab, -1, vocab - 1, -100], device="cuda")
    r = token_log_probs(z, t, top=3, entropy=True)
    assert r.log_probs[0] == -inf and r.entropy[0] == 0 and (r.top_log_probs[0] == -inf).all() and r.top_tokens[0].tolist() == [0, 1, 2]
    assert r.log_probs[1] == 0 and r.entropy[1] == 0 and r.top_tokens[1].tolist() == [0, 1, 2] and r.top_log_probs[1].tolist() == [0, -inf, -inf]
    for row in (2, 5, 8):
        assert r.entropy[row].item() == pytest.approx(math.log(vocab), abs=1e-4) and r.top_tokens[row].tolist() == [0, 1, 2]
    assert r.log_probs[2].item() == pytest.approx(-math.log(vocab), abs=1e-4)
    assert r.log_probs[7].item() == pytest.approx(-math.log(2), abs=1e-6) and r.entropy[7].item() == pytest.approx(math.log(2), abs=1e-6)
    assert r.log_probs[3:7].isnan().all() and r.entropy[3].isnan() and r.entropy[4].isnan() and r.log_probs[8] == 0
    assert ((r.top_tokens >= 0) & (r.top_tokens < vocab)).all()
    grad, = torch.autograd.grad((r.log_probs, r.entropy, r.top_log_probs), z, (torch.ones(9, device="cuda"), torch.ones(9, device="cuda"), torch.ones(9, 3, device="cuda")))
    assert (grad[0] == 0).all() and grad[:3].isfinite().all() and grad[7:].isfinite().all() and grad[3:7].isnan().all()
    alone = token_log_probs(z, t).log_probs      # rows that are ignored are not even read
    torch.testing.assert_close(alone, r.log_probs.detach(), equal_nan=True, atol=2e-5, rtol=0)
    grad, = torch.autograd.grad(token_log_probs(z, t).log_probs, z, torch.ones(9, device="cuda"))
    assert (grad[8] == 0).all() and (grad[0] == 0).all()


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few"])
@pytest.mark.parametrize("rows, vocab", [(2, 50257), (400, 5003), (3, 300)])
def test_orders_of_the_largest(kind, rows, vocab):
    z = {"equal": torch.zeros(vocab), "rising": torch.arange(vocab) / 64.0, "falling": -torch.arange(vocab) / 64.0, "few": (torch.arange(vocab) * 7919 % 5).float()}[kind]
    for dtype in DTYPES:
        if kind in ("rising", "falling") and dtype == torch.float16 and vocab > 60000:
            continue
        _check(z.to("cuda", dtype).expand(rows, vocab).contiguous(), torch.full((rows,), vocab // 2, device="cuda"), top=32, entropy=True, gradients=("top",))


def test_zeros_of_both_signs_are_equal():
    for rows, vocab in ((1, 40), (3, 5000)):
        z = torch.zeros(rows, vocab, device="cuda")
        z[:, ::2] = -0.0
        r = token_log_probs(z, torch.zeros(rows, dtype=torch.int64, device="cuda"), top=5)
        assert (r.top_tokens == torch.arange(5, device="cuda")).all()


def test_streams_and_graphs():
    gen = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(64, 5003, generator=gen, device="cuda", requires_grad=True)
    t = torch.randint(0, 5003, (64,), generator=gen, device="cuda")

    def call():
        r = token_log_probs(z, t, top=4, entropy=True)
        return (*[x for x in r], *torch.autograd.grad((r.log_probs.sum() + r.entropy.sum()), z))

    want = [x.detach().clone() for x in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
        got = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    z.data.copy_(z.data.flip(0))
    t.copy_(t.flip(0))
    graph.replay()
    got = [x.detach().clone() for x in got]
    assert not torch.equal(got[0], want[0])
    assert all(torch.equal(a, b) for a, b in zip([x.detach() for x in call()], got))   # (the same rows at the same addresses: the same order of sums)


def test_more_elements_than_thirty_two_bits_count():
    """Rows that begin behind 2^31 elements: the same as those rows by themselves."""
    rows, vocab = 43000, 50257     # 2^31 = 42730.2 x 50257
    z = torch.empty(rows, vocab, device="cuda", dtype=torch.bfloat16).normal_(generator=torch.Generator(device="cuda").manual_seed(0)).requires_grad_()
    t = torch.arange(rows, device="cuda") % vocab
    r = token_log_probs(z, t, top=3, entropy=True)
    grad, = torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), z)
    last = z.detach()[-300:].clone().requires_grad_()
    want = token_log_probs(last, t[-300:], top=3, entropy=True)
    # Not bit for bit: the 42700th row begins 8 bytes behind a 16-byte boundary and its copy on one, so that threads sum other elements.
    # A sum of 197 terms in a thread and 8 levels above: 205 x 2^-24 of s, an exponential 2^-22 and its argument 16 x 2^-24 off: for two
    # such sums 2 (205 + 4 + 16) 2^-24 < 2.7e-5; the rest of log p (of 14) 2^-20. In H what is off by 2.7e-5 has a weight of |d| <= 14.
    # A gradient is p (< 2e-3) times what is off by less than both together, 5e-4, and is rounded once on either side.
    off = 2.7e-5 + 2.0**-20
    for a, b, atol in zip(r[:3], want[:3], (off, 15 * off, off)):
        assert ((a[-300:] - b).abs() <= atol).all()
    assert torch.equal(r.top_tokens[-300:], want.top_tokens)
    expected = torch.autograd.grad(want.log_probs.sum() + want.entropy.sum(), last)[0].double()
    assert ((grad[-300:].double() - expected).abs() <= 1e-6 + 2.0**-7 * expected.abs()).all()
