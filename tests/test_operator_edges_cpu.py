"""token_log_probs, packed_attention and AdamW where they can go wrong, in their forms on the CPU."""
import copy

import pytest
import torch

from powersgd_b200 import AdamW
from powersgd_b200.models import GPT2, GPT2Config
from powersgd_b200.ops.attention import packed_attention
from powersgd_b200.ops.tokens import token_log_probs


@pytest.mark.parametrize("which", ["entropy", "top_log_probs"])
def test_entropy_and_alternatives_do_not_depend_on_the_target(which):
    torch.manual_seed(0)
    z = torch.randn(4, 9, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([-1, 9, 3, -100])
    r = token_log_probs(z, t, top=3, entropy=True)
    want = token_log_probs(z, torch.zeros_like(t), top=3, entropy=True)
    got, = torch.autograd.grad(getattr(r, which).square().sum(), z)
    assert got.isfinite().all() and torch.equal(got, torch.autograd.grad(getattr(want, which).square().sum(), z)[0])
    assert torch.autograd.gradcheck(lambda z: getattr(token_log_probs(z, t, top=3, entropy=True), which), (z,))
    r = token_log_probs(z, t, entropy=True)     # its own gradient does
    grad, = torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), z)
    assert grad[:2].isnan().all() and grad[2:].isfinite().all()


def _tangent_calls(device):
    """Calls of both operators with a tangent at one input, or at the gradient that is handed in."""
    import torch.autograd.forward_ad as fw

    z, t = torch.randn(3, 8, device=device), torch.tensor([0, 5, -100], device=device)
    x = torch.randn(6, 2, 8, device=device).bfloat16()
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device=device)
    tokens = lambda z: token_log_probs(z, t, top=2, entropy=True)[:3]  # noqa: E731
    places = [lambda y: packed_attention(y, x, x, offsets), lambda y: packed_attention(x, y, x, offsets), lambda y: packed_attention(x, x, y, offsets)]
    calls = []
    for f, at in [(tokens, z), *((f, x) for f in places)]:
        def jvp(f=f, at=at):
            torch.func.jvp(f, (at,), (torch.ones_like(at),))

        def dual(f=f, at=at, grad=False):
            with fw.dual_level():
                f(fw.make_dual(at.clone().requires_grad_() if grad else at, torch.ones_like(at)))

        def unrecorded(dual=dual):
            with torch.no_grad():
                dual()

        def handed_in(f=f, at=at):
            leaf = at.clone().requires_grad_()
            out = f(leaf)
            out = out if isinstance(out, torch.Tensor) else out[0]
            with fw.dual_level():
                torch.autograd.grad(out, leaf, fw.make_dual(torch.ones_like(out), torch.ones_like(out)))

        calls += [jvp, dual, lambda dual=dual: dual(grad=True), unrecorded, handed_in]
    calls.append(lambda: torch.func.jacfwd(lambda z: token_log_probs(z, t).log_probs)(z))
    return calls


def test_tangents_are_refused():
    """Forward-mode differentiation would find results without tangents, which it takes for zeros."""
    for call in _tangent_calls("cpu"):
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp|setup_context"):
            call()


@pytest.mark.parametrize("change, error", [(dict(amsgrad=True), ValueError), (dict(maximize=True), ValueError), (dict(lr=-1.0), ValueError),
                                           (dict(betas=(0.9, 1.0)), ValueError), (dict(state_bits=16), ValueError), (dict(seed=-1), ValueError)])
def test_a_state_that_is_refused_changes_nothing(change, error):
    def optimizer(lr):
        p = [torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(3))]
        opt = AdamW([dict(params=p[:1]), dict(params=p[1:], lr=0.5)], lr=lr)
        for x in p:
            x.grad = torch.full_like(x, lr)
        opt.step()
        return opt

    a, state = optimizer(0.1), copy.deepcopy(optimizer(0.2).state_dict())
    before = copy.deepcopy(a.state_dict())
    state["param_groups"][1].update(change)
    with pytest.raises(error):
        a.load_state_dict(state)
    after = a.state_dict()
    assert after["param_groups"] == before["param_groups"]
    for i, moments in before["state"].items():
        assert all(torch.equal(x, after["state"][i][name]) for name, x in moments.items())


def check_orders_of_dimensions(device):
    """A parameter whose order of dimensions changes after steps were made, and a state that was saved before it did: the same steps as
    those of torch. In 8 bits, where elements share scales in the order of memory, the step is refused."""
    torch.manual_seed(0)
    start = torch.randn(6, 4, 3, 3, device=device)
    grads = [torch.randn(6, 4, 3, 3, device=device) for _ in range(4)]
    last = torch.channels_last

    def steps(make, change):
        p = torch.nn.Parameter(start.clone())
        opt = make([p])
        for i, g in enumerate(grads):
            if i == 2 and change == "data":
                p.data = p.data.contiguous(memory_format=last)
            if i == 2 and change == "load":
                state, q = copy.deepcopy(opt.state_dict()), torch.nn.Parameter(p.detach().contiguous(memory_format=last))
                p, opt = q, make([q])
                opt.load_state_dict(state)
            p.grad = g.clone()
            opt.step()
        return p.detach(), opt

    want, _ = steps(lambda p: torch.optim.AdamW(p, lr=0.1, foreach=False), "none")
    for change in ("data", "load"):
        got, opt = steps(lambda p: AdamW(p, lr=0.1), change)
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
        assert next(iter(opt.state.values()))["exp_avg"].is_contiguous(memory_format=last)
        with pytest.raises(ValueError, match="strides"):
            steps(lambda p: AdamW(p, lr=0.1, state_bits=8), change)


def test_orders_of_dimensions():
    check_orders_of_dimensions("cpu")


def test_positions_of_documents_with_offsets_outside():
    """Offsets outside the rows are taken for the nearer end, by attention and by positions."""
    torch.manual_seed(0)
    model, tokens = GPT2(GPT2Config.tiny()), torch.randint(0, 512, (30,))
    for bad, good in (([-5, 9, 30], [0, 9, 30]), ([-9, -3, 20, 99], [0, 0, 20, 30]), ([4, 12, 40], [4, 12, 30])):
        bad, good = (torch.tensor(x, dtype=torch.int32) for x in (bad, good))
        assert torch.equal(model(tokens, bad), model(tokens, good))
