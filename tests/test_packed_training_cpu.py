"""GPT-2 on packed documents, token log probabilities and AdamW together, in torch operations: the same as document by document."""
import pytest
import torch

from powersgd_b200 import AdamW, Config, PowerSGD, optimizer_step
from powersgd_b200.models import GPT2, GPT2Config


def _documents(lengths, rows):
    gen = torch.Generator().manual_seed(0)
    tokens = torch.randint(0, 512, (rows,), generator=gen)
    offsets = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32)
    targets = torch.full((rows,), -100)
    for lo, hi in zip(offsets.tolist(), offsets.tolist()[1:]):
        targets[lo : max(hi - 1, lo)] = tokens[lo + 1 : max(hi, lo + 1)]
    return tokens, targets, offsets


def _by_document(model, tokens, targets, offsets):
    total, count = 0.0, 0
    for lo, hi in zip(offsets.tolist(), offsets.tolist()[1:]):
        if hi > lo:
            logits = model(tokens[None, lo:hi])[0]
            total = total + torch.nn.functional.cross_entropy(logits, targets[lo:hi], ignore_index=-100, reduction="sum")
            count += int((targets[lo:hi] != -100).sum())
    return total / max(count, 1)


def test_same_as_document_by_document():
    torch.manual_seed(0)
    model = GPT2(GPT2Config.tiny())
    tokens, targets, offsets = _documents([9, 0, 1, 30, 17], 60)
    loss = model.loss(tokens, targets, offsets)
    grads = torch.autograd.grad(loss, list(model.parameters()))
    want = _by_document(model, tokens, targets, offsets)
    want_grads = torch.autograd.grad(want, list(model.parameters()))
    # float32 sums of up to 512 terms in other orders, through two layers
    torch.testing.assert_close(loss, want, rtol=1e-5, atol=0)
    for g, w in zip(grads, want_grads):
        assert (g - w).norm() <= 1e-4 * w.norm() + 1e-7
    r = model.score(tokens, targets, offsets, top=3, entropy=True)
    torch.testing.assert_close(-r.log_probs.sum() / (targets != -100).sum(), loss)
    assert r.top_tokens.shape == (60, 3)


def test_without_offsets_as_before():
    torch.manual_seed(0)
    model = GPT2(GPT2Config.tiny())
    tokens, targets = torch.randint(0, 512, (2, 8)), torch.randint(0, 512, (2, 8))
    want = torch.nn.functional.cross_entropy(model(tokens).view(-1, 512).float(), targets.reshape(-1))
    assert torch.equal(model.loss(tokens, targets), want)
    torch.testing.assert_close(-model.score(tokens, targets).log_probs.mean(), want, rtol=1e-5, atol=0)


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_behind_powersgd(bits):
    torch.manual_seed(0)
    model = GPT2(GPT2Config.tiny())
    params = list(model.parameters())
    opt = AdamW(params, lr=1e-3, state_bits=bits)
    agg = PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=1))
    tokens, targets, offsets = _documents([9, 0, 1, 30, 17], 60)
    for step in range(3):
        model.loss(tokens, targets, offsets).backward()
        optimizer_step(opt, agg)
    assert all(p.isfinite().all() for p in params) and all(opt.state[p]["step"] == 3 for p in params)


def test_refusals():
    model = GPT2(GPT2Config(vocab_size=512, n_positions=64, n_embd=64, n_layer=1, n_head=4, dropout=0.1))
    tokens, targets, offsets = _documents([9], 9)
    with pytest.raises(ValueError, match="dropout"):
        model.loss(tokens, targets, offsets)
    model.eval().loss(tokens, targets, offsets)
    with pytest.raises(ValueError, match="tokens"):
        model.loss(tokens[None], targets, offsets)
    with pytest.raises(ValueError, match="tokens"):
        model(tokens)
