"""Heads normed and turned by position, in torch operations, against complex numbers in 64 bits and against differences; and what is refused.

Bounds in float32: a result is a sum of two products, each with at most ten roundings of 2^-24 (norm, weight, cosine, the products and the sum), relative to the
magnitudes of its two terms."""
import math

import pytest
import torch

from powersgd_b200.models import GPT2, GPT2Config
from powersgd_b200.ops.rotary import frequencies, rotate_heads, rotate_projection

OWN = 12 * 2.0**-24    # relative to the pair's magnitude


def places(lengths, rows, device="cpu"):
    """Offsets of sequences of these lengths, positions of the rows and which of them belong to one."""
    offsets = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device=device)
    position, held = torch.zeros(rows, dtype=torch.int64), torch.zeros(rows, dtype=torch.bool)
    for lo, n in zip(offsets.tolist(), lengths):
        position[lo : lo + n], held[lo : lo + n] = torch.arange(n), True
    return offsets, position.to(device), held.to(device)


def exact(x, position, held, weight, eps, base, rotated, interleaved):
    """In 64 bits, differentiable; angles as exact as whole turns can be taken out beforehand."""
    y = x if eps is None else x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + eps)
    y = y if weight is None else y * weight
    if rotated:
        table = frequencies(rotated, base)
        turns = [[(int(p) * int.from_bytes(table[8 * i : 8 * i + 8], "little")) % 2**64 / 2**64 for i in range(rotated // 2)] for p in position.tolist()]
        angle = 2 * math.pi * torch.tensor(turns, dtype=torch.float64, device=x.device).view(-1, 1, rotated // 2)
        head = y[..., :rotated]
        pairs = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
        y = torch.cat(((z if interleaved else z.transpose(-1, -2)).flatten(-2), y[..., rotated:]), -1)
    return torch.where(held[:, None, None], y, torch.zeros_like(y))


def magnitudes(x, rotated, interleaved):
    """Of each element with the one that it is turned with."""
    y = x.abs().clone()
    if rotated:
        head = y[..., :rotated]
        pairs = head.unflatten(-1, (-1, 2)) if interleaved else head.unflatten(-1, (2, -1)).transpose(-1, -2)
        both = pairs.norm(dim=-1, keepdim=True).expand(pairs.shape)
        y[..., :rotated] = (both if interleaved else both.transpose(-1, -2)).flatten(-2)
    return y


def compare(got, want, dtype, rotated, interleaved, scale=1.0, floor=0.0):
    info = torch.finfo(dtype)
    own = 2.0**-45 if dtype == torch.float64 else OWN
    bound = magnitudes(want, rotated, interleaved) * own * scale + want.abs() * (info.eps / 2 if dtype.itemsize == 2 else 0) + info.smallest_normal * info.eps + floor
    off = (got.double() - want).abs()
    assert (off <= bound).all(), (off / bound).max().item()


def check(x, heads, keys, lengths=None, position=None, weights=True, eps=1e-6, base=10000.0, rotated=None, interleaved=False, weight_type=torch.float32, only=None):
    """Forward and backward of one call against 64 bits. `only`: which of the results have a gradient."""
    rows, _, size = x.shape
    device, dtype = x.device, x.dtype
    rotated = size if rotated is None else rotated
    gen = torch.Generator().manual_seed(5)
    w = [(1 + 0.3 * torch.randn(size, generator=gen)).to(weight_type).to(device).requires_grad_() if weights and eps is not None else None for _ in range(2 if keys else 1)]
    held = torch.ones(rows, dtype=torch.bool, device=device)
    options = dict(eps=eps, base=base, rotated=rotated, interleaved=interleaved)
    if lengths is not None:
        options["offsets"], position, held = places(lengths, rows, device)
    else:
        options["positions"] = position
    x = x.detach().requires_grad_()
    if keys:
        outs = rotate_projection(x, heads, keys, q_weight=w[0], k_weight=w[1], **options)
    else:
        outs = (rotate_heads(x, weight=w[0], **options),)
    wide = [None if t is None else t.detach().double().requires_grad_() for t in (x, *w)]
    wants = []
    for lo, n, weight in ((0, heads, wide[1]), (heads, keys, wide[-1])):
        if n:
            wants.append(exact(wide[0][:, lo : lo + n], position, held, weight, eps, base, rotated, interleaved))
    for got, want in zip(outs, wants):
        assert got.dtype == dtype and got.is_contiguous()
        compare(got, want, dtype, rotated, interleaved)
    if keys:
        wants.append(wide[0][:, heads + keys :])
        assert torch.equal(outs[2], x[:, heads + keys :]) and outs[2].data_ptr() == x[:, heads + keys :].data_ptr()
    only = range(len(outs)) if only is None else only
    grads = [torch.randn(o.shape, generator=gen).to(dtype).to(device) for o in outs]
    leaves = [t for t in (x, *w) if t is not None]
    got = torch.autograd.grad([outs[i] for i in only], leaves, [grads[i] for i in only], allow_unused=True)
    want = torch.autograd.grad([wants[i] for i in only], [t for t in wide if t is not None], [grads[i].double() for i in only], allow_unused=True)
    # dx: the difference of dn and its part along n; both are as large as w r and a head's gradients
    with torch.no_grad():
        r = 1.0 if eps is None else torch.rsqrt(wide[0].square().mean(-1, keepdim=True) + eps)
        largest = max([1.0] + [t.detach().abs().max().item() for t in w if t is not None])
        head_grad = torch.cat([g.double().abs().amax(-1, keepdim=True) if i in only else torch.zeros_like(g[..., :1]).double() for i, g in enumerate(grads)], 1)
        terms = head_grad * r * largest * 2 * size**0.5    # |n_i| <= sqrt(size), mean(dn n) <= |dn| |n| / size <= max |dn|
        info = torch.finfo(dtype)
        own = 2.0**-45 if dtype == torch.float64 else 8 * 2.0**-24
        bound = terms * own + want[0].abs() * (info.eps / 2 if dtype.itemsize == 2 else 0) + info.smallest_normal * info.eps
        off = (got[0].double() - want[0]).abs()
        assert got[0].shape == x.shape and (off <= bound).all(), (off / bound).max().item()
        if not held.all():
            assert (got[0][~held][:, : heads + keys] == 0).all()
        # dw: sums over rows and heads of products of normed elements and gradients, of which none is larger than the following
        for i, (g, t) in enumerate(zip(got[1:], want[1:])):
            n = (heads, keys)[i]
            if t is None:
                assert g is None or (g == 0).all()
                continue
            part = wide[0][:, (0, heads)[i] : (0, heads)[i] + n] * (r if eps is None else r[:, (0, heads)[i] : (0, heads)[i] + n])
            size_of = (magnitudes(grads[i].double(), rotated, interleaved) * part.abs() * held[:, None, None]).sum((0, 1))
            terms = max(rows * n, 2)
            own = (12 + math.log2(terms) + terms**0.5) * 2.0**-24 if weight_type != torch.float64 else 2.0**-40     # in blocks, whose errors go either way
            bound = size_of * own + t.abs() * (torch.finfo(weight_type).eps / 2 if weight_type.itemsize == 2 else 2.0**-24) + 1e-30
            assert g.dtype == weight_type and ((g.double() - t).abs() <= bound).all()
    return outs, got


def values(rows, heads, size, dtype, device="cpu", seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, heads, size, generator=gen) * torch.exp(torch.randn(rows, heads, 1, generator=gen))).to(dtype).to(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("size, rotated, interleaved", [(8, 8, False), (16, 16, True), (40, 16, False), (64, 64, False), (80, 40, True), (24, 0, False)])
def test_against_64_bits(size, rotated, interleaved, dtype):
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    check(values(20, 8, size, dtype), 4, 2, lengths=[3, 0, 9, 1], rotated=rotated, interleaved=interleaved, weight_type=wide)
    check(values(20, 3, size, dtype), 3, 0, position=torch.randint(-1000, 2**20, (20,)), rotated=rotated, interleaved=interleaved, weight_type=dtype)
    check(values(20, 3, size, dtype), 3, 0, lengths=[20], eps=None, rotated=rotated, interleaved=interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("eps", [1e-6, None])
def test_against_differences(eps, interleaved):
    torch.manual_seed(0)
    x = torch.randn(7, 5, 16, dtype=torch.float64, requires_grad=True)
    w = [torch.randn(16, dtype=torch.float64, requires_grad=True) if eps else None for _ in range(2)]
    offsets = torch.tensor([1, 4, 4, 6], dtype=torch.int32)
    call = lambda x, *w: rotate_projection(x, 2, 1, offsets=offsets, q_weight=w[0] if w else None, k_weight=w[1] if w else None, eps=eps, rotated=8, interleaved=interleaved)  # noqa: E731
    assert torch.autograd.gradcheck(call, (x, *w) if eps else (x,))
    assert torch.autograd.gradcheck(lambda x: rotate_heads(x, offsets=offsets, eps=eps, interleaved=interleaved), (x,))


def test_positions_far_out():
    """As exact as near zero: the formula in numbers of any length."""
    from fractions import Fraction

    far = [0, 1, -1, 2**31 - 1, -(2**31), 2**40 + 12345, 10**15 + 7]
    table = frequencies(16, 10000.0)
    assert len(table) == 64
    for i in range(8):
        f = Fraction(int.from_bytes(table[8 * i : 8 * i + 8], "little"), 2**64)
        assert abs(float(f) * 2 * math.pi / 10000.0 ** (-i / 8) - 1) < 1e-14
    check(values(len(far), 2, 16, torch.float32), 2, 0, position=torch.tensor(far))
    check(values(len(far), 2, 16, torch.float64), 2, 0, position=torch.tensor(far), weight_type=torch.float64)


def check_offsets(device, dtype=torch.float32, form=None):
    """Offsets outside the rows, rows before the first and behind the last sequence, none at all."""
    x = values(12, 3, 16, dtype, device)
    for offsets, position in (([-3, 4, 4, 9], [0, 1, 2, 3, 0, 1, 2, 3, 4, None, None, None]), ([2, 5, 100], [None, None, 0, 1, 2, 0, 1, 2, 3, 4, 5, 6]), ([0], [None] * 12),
                              ([12, 12], [None] * 12), ([5, 5, 5, 5, 7], [None] * 5 + [0, 1] + [None] * 5)):
        offsets = torch.tensor(offsets, dtype=torch.int32, device=device)
        held = torch.tensor([p is not None for p in position], device=device)
        bad = x.clone()
        bad[~held] = math.nan
        bad.requires_grad_()
        w = torch.linspace(0.5, 2, 16, device=device).requires_grad_()
        got = rotate_heads(bad, offsets=offsets, weight=w)
        want = rotate_heads(x, positions=torch.tensor([p or 0 for p in position], device=device), weight=w.detach())
        assert torch.equal(got[held], want[held]) and (got[~held] == 0).all()
        grad = torch.full_like(got, 0.5)
        grad[~held] = math.nan
        dx, dw = torch.autograd.grad(got, (bad, w), grad)
        assert (dx[~held] == 0).all() and dx.isfinite().all() and dw.isfinite().all()


def test_offsets():
    check_offsets("cpu")


def check_sizes_at_the_border(device):
    """Heads of zeros, of numbers whose squares leave the range of float32, and of what is no number."""
    x = torch.ones(6, 2, 16, device=device)
    x[0], x[1, 0], x[2], x[3, 1, 5], x[4, 0, 3] = 0, 1e30, -3e38, math.nan, math.inf
    out = rotate_heads(x, positions=torch.zeros(6, dtype=torch.int32, device=device))
    assert (out[0] == 0).all() and (out[1, 0] - 1).abs().max() <= 1e-6 and (out[2] + 1).abs().max() <= 1e-6 and (out[5] - 1).abs().max() <= 1e-6
    assert out[3, 1].isnan().all() and out[4, 0, 3].isnan() and (out[4, 0, [0, 1, 2]] == 0).all() and out[3, 0].isfinite().all() and out[4, 1].isfinite().all()
    x = x[[0, 1, 2, 5]].requires_grad_()
    dx, = torch.autograd.grad(rotate_heads(x, positions=torch.zeros(4, dtype=torch.int32, device=device)), x, torch.ones_like(x))
    assert dx.isfinite().all()


def test_sizes_at_the_border():
    check_sizes_at_the_border("cpu")


def check_some_gradients(device, dtype):
    """Where not all results are used, and where only the weights are asked for."""
    for only in ([0], [1], [2], [0, 2], [1, 2]):
        check(values(9, 6, 16, dtype, device), 2, 2, lengths=[5, 4], only=only)
    x, w = values(9, 6, 16, dtype, device), torch.ones(16, device=device, requires_grad=True)
    q, k, v = rotate_projection(x, 2, 2, positions=torch.arange(9, device=device), q_weight=w, k_weight=w)
    a, = torch.autograd.grad((q, k), w, (q.detach(), k.detach()))
    y = x.clone().requires_grad_()
    q, k, v = rotate_projection(y, 2, 2, positions=torch.arange(9, device=device), q_weight=w, k_weight=w)
    b, dy = torch.autograd.grad((q, k), (w, y), (q.detach(), k.detach()))
    assert torch.equal(a, b) and (dy[:, 4:] == 0).all() and (q * k).sum().isfinite()


def test_some_gradients():
    check_some_gradients("cpu", torch.float32)


def refused(device):
    x = torch.randn(6, 4, 16, device=device)
    at = torch.arange(6, device=device)
    o = torch.tensor([0, 6], dtype=torch.int32, device=device)
    w = torch.ones(16, device=device)
    p = lambda *a, **k: lambda: rotate_projection(*a, **k)  # noqa: E731
    h = lambda *a, **k: lambda: rotate_heads(*a, **k)  # noqa: E731
    yield h(x[0], positions=at), ValueError
    yield h(x[..., :12], positions=at), ValueError
    yield h(torch.randn(6, 1, 264, device=device), positions=at), ValueError
    yield h(x, positions=at, rotated=12), ValueError
    yield h(torch.zeros(6, 4097, 8, device=device), positions=at), ValueError
    yield h(x, positions=at, rotated=24), ValueError
    yield h(x, positions=at, rotated=-8), ValueError
    yield h(x, positions=at, rotated=8.0), ValueError
    yield h(x), ValueError
    yield h(x, positions=at, offsets=o), ValueError
    yield h(x, rotated=0, positions=at, offsets=o), ValueError
    yield h(x, positions=at[:5]), ValueError
    yield h(x, positions=at.float()), ValueError
    yield h(x, positions=at[:, None]), ValueError
    yield h(x, offsets=o.long()), ValueError
    yield h(x, offsets=o[:0]), ValueError
    yield h(x, offsets=o[None]), ValueError
    yield h(x, positions=at, eps=0.0), ValueError
    yield h(x, positions=at, eps=-1.0), ValueError
    yield h(x, positions=at, eps=math.nan), ValueError
    yield h(x, positions=at, base=0.5), ValueError
    yield h(x, positions=at, base=math.inf), ValueError
    yield h(x, positions=at, base=math.nan), ValueError
    yield h(x, positions=at, weight=w, eps=None), ValueError
    yield h(x, positions=at, weight=w[:8]), ValueError
    yield h(x, positions=at, weight=w.double()), TypeError
    yield h(x.long(), positions=at), TypeError
    yield p(x, 2, 2, positions=at, q_weight=w, k_weight=w.bfloat16()), TypeError
    yield p(x.bfloat16(), 2, 2, positions=at, q_weight=w, k_weight=w.bfloat16()), TypeError
    yield p(x, 0, 2, positions=at), ValueError
    yield p(x, 2, 0, positions=at), ValueError
    yield p(x, 2, 3, positions=at), ValueError
    yield p(x, -1, 2, positions=at), ValueError


def test_refusals():
    for call, error in refused("cpu"):
        with pytest.raises(error):
            call()


def tangents(device):
    import torch.autograd.forward_ad as fw

    x, w, at = torch.randn(6, 4, 16, device=device), torch.ones(16, device=device), torch.arange(6, device=device)
    for f, t in ((lambda x: rotate_heads(x, positions=at), x), (lambda w: rotate_heads(x, positions=at, weight=w), w)):
        for leaf in (False, True):
            def dual(f=f, t=t, leaf=leaf):
                with fw.dual_level():
                    f(fw.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t)))

            yield dual

        def handed_in(f=f, t=t):
            leaf = t.clone().requires_grad_()
            out = f(leaf)
            with fw.dual_level():
                torch.autograd.grad(out, leaf, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))

        yield handed_in


def test_tangents_and_second_derivatives_are_refused():
    for call in tangents("cpu"):
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode"):
            call()
    x = torch.randn(6, 4, 16, requires_grad=True)
    g, = torch.autograd.grad(rotate_heads(x, positions=torch.arange(6)).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def check_no_rows_and_no_values(device):
    for rows in (0, 1):
        x = torch.randn(rows, 4, 16, device=device, requires_grad=True)
        w = torch.ones(16, device=device, requires_grad=True)
        q, k, v = rotate_projection(x, 3, 1, positions=torch.arange(rows, device=device), q_weight=w, k_weight=w)
        assert v.shape == (rows, 0, 16)
        dx, dw = torch.autograd.grad((q.sum() + k.sum()), (x, w))
        assert dx.shape == x.shape and (rows or (dw == 0).all())
        assert rotate_heads(x.detach(), offsets=torch.zeros(1, dtype=torch.int32, device=device)).shape == (rows, 4, 16)


def test_no_rows_and_no_values():
    check_no_rows_and_no_values("cpu")


def check_one_weight(device):
    """Only one of the weights is given, or learns; the other's heads are the same as without it."""
    x, at = values(9, 6, 16, torch.float32, device), torch.arange(9, device=device)
    w = [torch.linspace(0.5, 2, 16, device=device), torch.linspace(2, 0.5, 16, device=device)]
    grads = [torch.randn(9, 2, 16, device=device) for _ in range(3)]

    def call(learns, given=(True, True)):
        leaves = [t.clone().requires_grad_(i in learns) if g else None for i, (t, g) in enumerate(zip(w, given))]
        out = rotate_projection(x, 2, 2, positions=at, q_weight=leaves[0], k_weight=leaves[1])
        return out, torch.autograd.grad(out, [leaves[i] for i in learns], grads) if learns else ()

    both = call((0, 1))
    for i in (0, 1):
        assert torch.equal(call((i,))[1][0], both[1][i])
        out, grad = call((i,), given=(i == 0, i == 1))
        assert torch.equal(out[i], both[0][i]) and torch.equal(grad[0], both[1][i])
        assert torch.equal(out[1 - i], rotate_heads(x[:, 2 - 2 * i : 4 - 2 * i], positions=at))
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(call(())[0], both[0]))


def test_one_weight():
    check_one_weight("cpu")


@pytest.mark.parametrize("rotary, qk_norm", [(True, False), (False, True), (True, True)])
def test_gpt2_same_as_document_by_document(rotary, qk_norm):
    from test_packed_training_cpu import _by_document, _documents

    torch.manual_seed(0)
    model = GPT2(GPT2Config(vocab_size=512, n_positions=64, n_embd=64, n_layer=2, n_head=4, rotary=rotary, qk_norm=qk_norm))
    names = {name for name, _ in model.named_parameters()}
    assert ("wpe.weight" in names) != rotary and ("h.0.q_norm" in names) == qk_norm
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "_norm" in name:
                p.copy_(torch.linspace(0.5, 2.0, p.numel()))
    tokens, targets, offsets = _documents([9, 0, 1, 30, 17], 60)
    params = list(model.parameters())
    loss, want = model.loss(tokens, targets, offsets), _by_document(model, tokens, targets, offsets)
    torch.testing.assert_close(loss, want, rtol=1e-5, atol=0)     # float32 sums of up to 512 terms in other orders, through two layers
    for g, w in zip(torch.autograd.grad(loss, params), torch.autograd.grad(want, params)):
        assert (g - w).norm() <= 1e-4 * w.norm() + 1e-7
    assert rotary is False or model(torch.randint(0, 512, (1, 100))).isfinite().all()      # no last position
    batch = torch.randint(0, 512, (3, 20))
    one_by_one = torch.cat([model(row[None]) for row in batch])
    torch.testing.assert_close(model(batch), one_by_one, rtol=1e-4, atol=1e-5)


def test_gpt2_positions_matter_only_by_their_distance():
    """What rotary attention of a first token says does not change with the tokens before it being elsewhere: rows before a document change nothing."""
    torch.manual_seed(0)
    model = GPT2(GPT2Config(vocab_size=512, n_positions=8, n_embd=64, n_layer=2, n_head=4, rotary=True))
    tokens = torch.randint(0, 512, (30,))
    a = model(tokens, torch.tensor([0, 12, 30], dtype=torch.int32))[12:]
    b = model(tokens[12:], torch.tensor([0, 18], dtype=torch.int32))
    torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def check_small(device):
    """Heads of zeros and of very small numbers under a small eps: r^3 would leave the range of float32."""
    x = torch.zeros(3, 1, 16, device=device)
    x[1, 0, 3], x[2] = 2.0**-60, 2.0**-50
    w = torch.linspace(0.5, 2, 16, device=device).requires_grad_()
    x.requires_grad_()
    grad = torch.ones(3, 1, 16, device=device)
    out = rotate_heads(x, positions=torch.zeros(3, dtype=torch.int32, device=device), weight=w, eps=2.0**-100)
    dx, dw = torch.autograd.grad(out, (x, w), grad)
    wide, ww = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = wide / (wide.square().mean(-1, keepdim=True) + 2.0**-100).sqrt() * ww
    wants = torch.autograd.grad(want, (wide, ww), grad.double())
    torch.testing.assert_close(out.double(), want, rtol=1e-5, atol=0)
    torch.testing.assert_close(dw.double(), wants[1], rtol=1e-5, atol=0)
    torch.testing.assert_close(dx.double(), wants[0], rtol=1e-4, atol=1e-5 * 2.0**50)    # differences of terms as large as w r, r up to 2^50


def test_small():
    check_small("cpu")
