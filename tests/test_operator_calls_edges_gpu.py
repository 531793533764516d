"""Calls of token_log_probs, packed_attention and AdamW on the GPU that go through the extension (csrc/host/operators.cpp) or through Python: both
refuse, raise and answer alike."""
import pytest
import torch
from test_operator_edges_cpu import _tangent_calls, check_orders_of_dimensions

from powersgd_b200 import AdamW, Config, PowerSGD
from powersgd_b200.engine import TrainStep
from powersgd_b200.ops import attention, host, scan, tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(tokens, "operators", None)
        monkeypatch.setattr(attention, "operators", None)
    else:
        assert host.operators is not None
        x = torch.zeros(1, 1, 8, device="cuda", dtype=torch.bfloat16)
        attention.packed_attention(x, x, x, torch.tensor([0, 1], device="cuda", dtype=torch.int32))   # (a device's first call goes through Python)
    return request.param


def test_tangents_are_refused(form):
    for call in _tangent_calls("cuda"):
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode|jvp|setup_context"):
            call()


@pytest.mark.parametrize("gradient", [False, True])
def test_tracing_is_refused(form, gradient):
    """A trace would hold an empty tensor and no kernel."""
    z, t = torch.randn(3, 8, device="cuda", requires_grad=gradient), torch.tensor([0, 5, -100], device="cuda")
    x = torch.randn(6, 2, 8, device="cuda").bfloat16().requires_grad_(gradient)
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")
    for f, args in ((lambda z, t: tokens.token_log_probs(z, t).log_probs, (z, t)), (lambda x, o: attention.packed_attention(x, x, x, o), (x, offsets))):
        with pytest.raises(NotImplementedError, match="jit.trace"):
            torch.jit.trace(f, args)


def test_requests_for_too_much_memory_are_told_as_such(form):
    """Copies and results beyond any GPU's memory: torch.OutOfMemoryError, which programs catch, through either form."""
    z = torch.zeros(1, 50257, device="cuda", dtype=torch.bfloat16).expand(2**23, 50257)
    with pytest.raises(torch.OutOfMemoryError):
        tokens.token_log_probs(z, torch.zeros(2**23, device="cuda", dtype=torch.int32))
    x = torch.zeros(1, 1, 128, device="cuda", dtype=torch.bfloat16).expand(2**20, 2**13, 128)
    with pytest.raises(torch.OutOfMemoryError):
        attention.packed_attention(x, x[:, :1], x[:, :1], torch.tensor([0, 5], device="cuda", dtype=torch.int32))


def _negated(x):
    """-x as a tensor that only says so, as the imaginary part of a conjugate does."""
    assert torch.complex(x, x).conj().imag.is_neg()
    return torch._neg_view(x)


def test_tensors_that_only_say_that_they_are_negated(form):
    z, t = torch.randn(3, 80, device="cuda"), torch.tensor([0, 5, -100], device="cuda")

    def both(z, g):
        leaf = z.detach().requires_grad_()
        r = tokens.token_log_probs(leaf, t, entropy=True)
        return [r.log_probs, r.entropy, *torch.autograd.grad((r.log_probs, r.entropy), leaf, (g, g))]

    g = torch.randn(3, device="cuda")
    for got in (both(_negated(z), g), both((-z).requires_grad_(), _negated(-g))):
        assert all(torch.equal(a, b) for a, b in zip(both(-z, g), got))
    zero = torch._efficientzerotensor((3,), device="cuda")
    assert (both(z, zero)[2] == 0).all()

    x, g = torch.randn(6, 2, 8, device="cuda").half(), torch.randn(6, 2, 8, device="cuda").half()
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda")

    def grads(x, g):
        leaf = x.detach().requires_grad_()
        out = attention.packed_attention(leaf, leaf, leaf, offsets)
        return [out, *torch.autograd.grad(out, leaf, g)]

    for got in (grads(torch._neg_view(x), g), grads(-x, torch._neg_view(-g))):
        assert all(torch.equal(a, b) for a, b in zip(grads(-x, g), got))
    assert (grads(x, torch._efficientzerotensor(x.shape, device="cuda", dtype=x.dtype))[1] == 0).all()


@pytest.mark.parametrize("listed", [True, False])
def test_gradients_that_only_say_that_they_are_negated(listed, monkeypatch):
    if not listed:
        monkeypatch.setattr(scan, "_native", None)
    start, g = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    results = []
    for grad in (-g, _negated(g)):
        p = torch.nn.Parameter(start.clone())
        optimizer = AdamW([p], lr=0.1)
        for _ in range(2):      # the first step makes the state
            p.grad = grad
            optimizer.step()
        results.append(p.detach())
    assert torch.equal(*results)


def test_orders_of_dimensions():
    check_orders_of_dimensions("cuda")


def test_a_wait_that_ran_out_is_told_behind_the_last_call(form):
    """The status word that kernels write is set from the host."""
    x = torch.zeros(4, 1, 8, device="cuda", dtype=torch.bfloat16)
    attention.packed_attention(x, x, x, torch.tensor([0, 4], device="cuda", dtype=torch.int32))
    torch.cuda.synchronize()
    attention.check_waits()
    attention._statuses[x.device][0][0] = 3
    with pytest.raises(RuntimeError, match="ran out"):
        attention.check_waits()
    attention.check_waits()


@pytest.mark.parametrize("bits", [32, 8])
def test_train_step_with_adamw(bits):
    """Every step runs eagerly, on weights that became channels_last; moments in 32 bits may be older than that."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Conv2d(3, 16, 3), torch.nn.ReLU(), torch.nn.Conv2d(16, 16, 3), torch.nn.AdaptiveAvgPool2d(1), torch.nn.Flatten(), torch.nn.Linear(16, 10)).cuda()
    params = list(model.parameters())
    optimizer = AdamW(params, lr=1e-2, state_bits=bits)
    if bits == 32:
        for p in params:
            p.grad = torch.randn_like(p)
        optimizer.step()
        optimizer.zero_grad()
    step = TrainStep(model, torch.nn.functional.cross_entropy, optimizer, PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=1)))
    x, y = torch.randn(32, 3, 16, 16, device="cuda"), torch.randint(0, 10, (32,), device="cuda")
    before = [p.detach().clone() for p in params]
    assert all(step(x, y).isfinite() for _ in range(5)) and not step._graphs
    assert all(p.isfinite().all() and not torch.equal(p, b) for p, b in zip(params, before))
    assert all(optimizer.state[p]["step"] == (6 if bits == 32 else 5) for p in params)
