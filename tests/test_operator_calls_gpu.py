"""token_log_probs and packed_attention through the extension (csrc/host/operators.cpp) and through Python: the same results,
gradients and refusals."""
import pytest
import torch

from powersgd_b200.ops import attention, host, tokens

pytestmark = pytest.mark.gpu


def test_the_extension_is_there():
    assert host.operators is not None


def _both(monkeypatch, module, call):
    results = []
    for operators in (host.operators, None):
        monkeypatch.setattr(module, "operators", operators)
        results.append(call())
    return results


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape and x.stride() == y.stride() and x.requires_grad == y.requires_grad
            assert torch.equal(x.detach(), y.detach())


@pytest.mark.parametrize("top, entropy", [(0, False), (0, True), (5, False), (5, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_tokens(dtype, top, entropy, monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(0)
    whole = torch.randn(4, 6, 1033, generator=gen, device="cuda").to(dtype)
    t = torch.randint(0, 1000, (4, 6), generator=gen, device="cuda")
    for z in (whole[..., :1000], whole[..., 1:1001], whole[:, ::2, :1000], whole[..., :1000].contiguous(), whole[:, :, :1000].transpose(0, 1), whole[0], whole[0, 0], whole[:1, :, :1000].expand(4, 6, 1000)):
        targets = t.new_zeros(z.shape[:-1]) + 3

        def call():
            leaf = z.detach().requires_grad_()
            r = tokens.token_log_probs(leaf, targets, top=top, entropy=entropy, temperature=0.9)
            plain = tokens.token_log_probs(z, targets.int(), top=top, entropy=entropy)
            loss = r.log_probs.sum() + (r.entropy.square().sum() if entropy else 0) + (r.top_log_probs.sum() if top else 0)
            return [*r, *plain, *torch.autograd.grad(loss, leaf)]

        _same(*_both(monkeypatch, tokens, call))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_attention(dtype, monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(300, 8, 64, generator=gen, device="cuda").to(dtype)
    offsets = torch.tensor([0, 100, 290], device="cuda", dtype=torch.int32)
    attention.packed_attention(x, x, x, offsets)   # (a device's first call goes through Python)
    odd = torch.randn(300 * 2 * 64 + 1, generator=gen, device="cuda").to(dtype)[1:].view(300, 2, 64)
    for q, k, v in ((x[:, :4], x[:, 4:6], x[:, 6:]), (x[:, :4].contiguous(), odd, x[:, :2]), (x[:, :1].expand(300, 4, 64), x[:, 4:6], x[:, 6:])):
        for causal, scale in ((True, None), (False, 0.3)):

            def call():
                leaves = [y.detach().requires_grad_() for y in (q, k, v)]
                out = attention.packed_attention(*leaves, offsets, causal=causal, scale=scale)
                return [attention.packed_attention(q, k, v, offsets, causal=causal, scale=scale), out, *torch.autograd.grad(out.float().square().sum(), leaves)]

            _same(*_both(monkeypatch, attention, call))


def test_empty(monkeypatch):
    def call():
        q = torch.zeros(0, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = attention.packed_attention(q, q, q, torch.zeros(3, device="cuda", dtype=torch.int32))
        k = torch.ones(5, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        none = attention.packed_attention(k, k, k, torch.zeros(1, device="cuda", dtype=torch.int32))
        return [out, *torch.autograd.grad(out.sum(), q), none, *torch.autograd.grad(none.sum(), k)]

    _same(*_both(monkeypatch, attention, call))

    def call():
        z = torch.zeros(0, 9, device="cuda", requires_grad=True)
        r = tokens.token_log_probs(z, torch.zeros(0, device="cuda", dtype=torch.int64), top=2, entropy=True)
        return [*r, *torch.autograd.grad(r.log_probs.sum(), z)]

    _same(*_both(monkeypatch, tokens, call))


def test_differentiated_once(monkeypatch):
    def twice():
        z = torch.randn(3, 50, device="cuda", requires_grad=True)
        g, = torch.autograd.grad(tokens.token_log_probs(z, torch.zeros(3, device="cuda", dtype=torch.int64)).log_probs.square().sum(), z, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()
        return []

    _both(monkeypatch, tokens, twice)


def test_changed_inputs_are_noticed(monkeypatch):
    def changed():
        z = torch.randn(3, 50, device="cuda", requires_grad=True)
        t = torch.zeros(3, device="cuda", dtype=torch.int64)
        r = tokens.token_log_probs(z, t)
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            r.log_probs.sum().backward()
        return []

    _both(monkeypatch, tokens, changed)


def test_subclasses_and_refusals(monkeypatch):
    class Sub(torch.Tensor):
        pass

    z, t = torch.randn(3, 50, device="cuda"), torch.zeros(3, device="cuda", dtype=torch.int64)
    assert host.operators.token_log_probs(z.as_subclass(Sub), t, 0, False, -100, 1.0) is None
    assert host.operators.token_log_probs(z, t, "x", False, -100, 1.0) is None

    def refused():
        for call, error in ((lambda: tokens.token_log_probs(z, t, top=51), ValueError), (lambda: tokens.token_log_probs(z.double(), t), TypeError),
                            (lambda: tokens.token_log_probs(z, t, temperature=-1.0), ValueError), (lambda: tokens.token_log_probs(z, t.cpu()), ValueError),
                            (lambda: tokens.token_log_probs(z, t, ignore_index=2**70), ValueError)):
            with pytest.raises(error):
                call()
        return []

    _both(monkeypatch, tokens, refused)


def test_a_wait_that_ran_out_is_told(monkeypatch):
    """The status word that kernels write is set from the host."""
    x = torch.randn(10, 1, 64, device="cuda").bfloat16()
    offsets = torch.tensor([0, 10], device="cuda", dtype=torch.int32)
    attention.packed_attention(x, x, x, offsets)
    for operators in (host.operators, None):
        monkeypatch.setattr(attention, "operators", operators)
        attention._statuses[x.device][0][0] = 3
        with pytest.raises(RuntimeError, match="ran out"):
            attention.packed_attention(x, x, x, offsets)
        attention.packed_attention(x, x, x, offsets)


def test_gradients_of_some(monkeypatch):
    """Only some inputs want a gradient; one tensor is all three of them."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(200, 2, 64, generator=gen, device="cuda").bfloat16() for _ in range(3))
    offsets = torch.tensor([0, 70, 200], device="cuda", dtype=torch.int32)

    def call():
        out = []
        whole = [x.detach().requires_grad_() for x in (q, k, v)]
        want = torch.autograd.grad(attention.packed_attention(*whole, offsets).float().square().sum(), whole)
        for i in range(3):
            given = [x.detach().requires_grad_() if i == j else x for j, x in enumerate((q, k, v))]
            got, = torch.autograd.grad(attention.packed_attention(*given, offsets).float().square().sum(), given[i])
            assert torch.equal(got, want[i])
            out.append(got)
        apart = [q.detach().requires_grad_() for _ in range(3)]
        parts = torch.autograd.grad(attention.packed_attention(*apart, offsets).float().square().sum(), apart)
        same = q.detach().requires_grad_()
        got, = torch.autograd.grad(attention.packed_attention(same, same, same, offsets).float().square().sum(), same)
        # sums of three, rounded at each addition, in any order: each rounding is half a step of a partial sum
        size = sum(x.double().abs() for x in parts)
        assert ((got.double() - sum(x.double() for x in parts)).abs() <= 2 * 2.0**-8 * size).all()
        return out + [got]

    _same(*_both(monkeypatch, attention, call))
