"""Calls of token_log_probs, packed_attention and AdamW on the GPU that go through the extension (csrc/host/operators.cpp) or through Python: both
refuse, raise and answer alike."""
import pytest
import torch
from test_operator_edges_cpu import _tangent_calls

from powersgd_b200.ops import attention, host, tokens

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
