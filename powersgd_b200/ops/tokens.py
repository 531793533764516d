"""Log probabilities of given tokens, with the entropy of each row and its most likely tokens (csrc/token_logprob.cu).

What a language model's training and evaluation take from its logits, without a float copy of them: the loss
(`-log_probs.mean()`), perplexity, an entropy bonus, the alternatives to a token. The logits are read once in
their own type, and the gradient is written once in it. On the CPU (or on CUDA without the native library
where PSGD_B200_ALLOW_FALLBACK=1 allows it) the same comes from torch operations.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch

from . import native
from .host import operators

MOST_TOP = 32
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class TokenLogProbs(NamedTuple):
    log_probs: torch.Tensor                     # float32, shaped like the targets
    entropy: Optional[torch.Tensor]             # float32, shaped like the targets
    top_log_probs: Optional[torch.Tensor]       # float32, [*targets.shape, top], descending
    top_tokens: Optional[torch.Tensor]          # int64; of equal logits the lowest index first


def token_log_probs(logits: torch.Tensor, targets: torch.Tensor, *, top: int = 0, entropy: bool = False, ignore_index: int = -100,
                    temperature: float = 1.0) -> TokenLogProbs:
    """Of the distribution softmax(logits / temperature) over the last dimension: the log probability of each target, the entropy (in nats),
    and the `top` (at most 32) most likely tokens with their log probabilities. All but the tokens are differentiable (once, backwards).

    `logits`: float32, bfloat16 or float16, [*targets.shape, vocabulary]; `targets`: int64 or int32.
    A target equal to `ignore_index` has log probability zero and no gradient; entropy and alternatives are those of its row all
    the same. A target outside the vocabulary has log probability NaN, whose gradient is NaN too: nothing is read for it. Masked tokens have logits of
    -inf; a row that has only those is no distribution: log probability -inf, entropy zero, no gradient. A row that
    holds +inf or NaN gives NaN, and any tokens. Returned statistics are float32."""
    out = operators.token_log_probs(logits, targets, top, entropy, ignore_index, temperature) if operators is not None else None
    if out is not None:
        return TokenLogProbs(*out)
    check(logits, targets, top, ignore_index, temperature)
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _TokenLogProbs.apply(logits, targets, int(top), bool(entropy), int(ignore_index), float(temperature))
        return TokenLogProbs(*out)
    return TokenLogProbs(*_forward(logits, targets, int(top), bool(entropy), int(ignore_index), float(temperature))[:4])


def check(logits, targets, top, ignore_index, temperature) -> None:
    native.refuse_tracing("token_log_probs", logits)
    if logits.is_cuda:
        native.refuse_without_memory("token_log_probs", logits, targets)
    if logits.dtype not in DTYPES and not (logits.dtype == torch.float64 and not logits.is_cuda):
        raise TypeError(f"token_log_probs: logits are {logits.dtype}; float32, bfloat16 and float16 are supported")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_log_probs: targets are {targets.dtype}; int64 and int32 are supported")
    if logits.dim() < 1 or logits.shape[:-1] != targets.shape:
        raise ValueError(f"token_log_probs: logits {tuple(logits.shape)} and targets {tuple(targets.shape)} do not belong together")
    vocab = logits.shape[-1]
    if not 1 <= vocab < 2**31 - 2**16:
        raise ValueError(f"token_log_probs: a vocabulary of {vocab}")
    if logits.device != targets.device:
        raise ValueError(f"token_log_probs: logits on {logits.device}, targets on {targets.device}")
    if not 0 <= top <= min(MOST_TOP, vocab):
        raise ValueError(f"token_log_probs: top = {top}; 0 to {min(MOST_TOP, vocab)} for a vocabulary of {vocab}")
    if not 2.0**-100 <= temperature <= 2.0**100:
        raise ValueError(f"token_log_probs: temperature {temperature}; 2^-100 to 2^100")
    if not -(2**63) <= ignore_index < 2**63:
        raise ValueError(f"token_log_probs: ignore_index {ignore_index}")
    native.refuse_tangents("token_log_probs", logits)


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """The logits as [rows, vocabulary] with elements of a row side by side and rows apart: a view where they lie so, else a copy."""
    logits, vocab = native.in_memory(logits), logits.shape[-1]
    if logits.is_contiguous():
        return logits.view(-1, vocab)
    if logits.stride(-1) == 1 or vocab == 1:
        try:
            rows = logits.view(-1, vocab)
            if rows.shape[0] <= 1 or rows.stride(0) >= vocab:
                return rows
        except RuntimeError:
            pass
    return logits.contiguous().view(-1, vocab)


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and native.use_for_cuda()


def _forward(logits, targets, top, entropy, ignore_index, temperature):
    """log_probs, entropy, top_log_probs, top_tokens, and the statistics (maximum, log of the sum) that the gradient needs."""
    shape, device = targets.shape, logits.device
    if not _native(logits):
        return _forward_torch(logits, targets, top, entropy, ignore_index, temperature)
    z, t = _rows(logits), targets.contiguous()
    n, vocab = z.shape
    log_probs = torch.empty(shape, dtype=torch.float32, device=device)
    stats = torch.empty(n, 2, dtype=torch.float32, device=device)
    h = torch.empty(shape, dtype=torch.float32, device=device) if entropy else None
    values = torch.empty((*shape, top), dtype=torch.float32, device=device) if top else None
    tokens = torch.empty((*shape, top), dtype=torch.int64, device=device) if top else None
    if n:
        with native.on_device(device) as stream:
            code = native.lib().psgd_token_logprob(
                z.data_ptr(), DTYPES[z.dtype], n, vocab, z.stride(0), t.data_ptr(), t.dtype == torch.int64, ignore_index, 1.0 / temperature, top,
                log_probs.data_ptr(), stats.data_ptr(), h.data_ptr() if entropy else None, values.data_ptr() if top else None,
                tokens.data_ptr() if top else None, stream,
            )
        native.check(code, "psgd_token_logprob")
    return log_probs, h, values, tokens, stats


def _backward(logits, targets, stats, entropy, tokens, g, g_entropy, g_top, ignore_index, temperature):
    if not _native(logits):
        return _backward_torch(logits, targets, stats, entropy, tokens, g, g_entropy, g_top, ignore_index, temperature)
    z, t = _rows(logits), targets.contiguous()
    n, vocab = z.shape
    grad, rows = _grad_like(logits, z)
    if n:
        g, g_entropy, g_top = (None if x is None else native.in_memory(x).contiguous() for x in (g, g_entropy, g_top))
        at = lambda x: None if x is None else x.data_ptr()  # noqa: E731
        with native.on_device(logits.device) as stream:
            code = native.lib().psgd_token_logprob_grad(
                z.data_ptr(), DTYPES[z.dtype], n, vocab, z.stride(0), rows.data_ptr(), rows.stride(0), t.data_ptr(), t.dtype == torch.int64,
                ignore_index, 1.0 / temperature, 0 if tokens is None else tokens.shape[-1], stats.data_ptr(), at(entropy), at(tokens), at(g), at(g_entropy),
                at(g_top), stream,
            )
        native.check(code, "psgd_token_logprob_grad")
    return grad


def _grad_like(logits: torch.Tensor, z: torch.Tensor):
    """Room for the gradient of the rows `z`, shaped like the logits, and the same as rows. Each row lies as far from a 16-byte boundary as
    that of `z` does, so that both are moved in the same vectors: contiguous where `z` is and begins on one, else with a few elements
    between the rows."""
    n, vocab = z.shape
    size = z.element_size()
    lead = z.data_ptr() % 16 // size
    between = (z.stride(0) - vocab) % (16 // size) if n > 1 else 0
    if lead == 0 and between == 0:
        grad = torch.empty(logits.shape, dtype=z.dtype, device=z.device)
        return grad, grad.view(n, vocab)
    pitch = vocab + between
    rows = torch.empty(lead + n * pitch, dtype=z.dtype, device=z.device).as_strided((n, vocab), (pitch, 1), lead)
    strides, step = [], pitch
    for size_of in reversed(logits.shape[:-1]):
        strides.append(step)
        step *= size_of
    return rows.as_strided(logits.shape, (*reversed(strides), 1), lead), rows


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, entropy, ignore_index, temperature):
        log_probs, h, values, tokens, stats = _forward(logits, targets, top, entropy, ignore_index, temperature)
        ctx.save_for_backward(logits, targets, stats, h, tokens)
        ctx.ignore_index, ctx.temperature = ignore_index, temperature
        ctx.set_materialize_grads(False)
        if tokens is not None:
            ctx.mark_non_differentiable(tokens)
        return log_probs, h, values, tokens

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, g_entropy, g_top, _):
        native.refuse_tangents("token_log_probs", g, g_entropy, g_top)
        logits, targets, stats, entropy, tokens = ctx.saved_tensors
        if logits.is_cuda:
            native.refuse_without_memory("token_log_probs", g, g_entropy, g_top)
        if g is None and g_entropy is None and g_top is None:
            return (None,) * 6
        if g_entropy is None:
            entropy = None
        if g_top is None:
            tokens = None
        return _backward(logits, targets, stats, entropy, tokens, g, g_entropy, g_top, ctx.ignore_index, ctx.temperature), None, None, None, None, None


# ---- the same in torch operations --------------------------------------------------------------
def _scaled(logits, stats, temperature):
    """log softmax of the rows (-inf throughout where a row has no distribution), and whether it has none."""
    z = logits.reshape(-1, logits.shape[-1]).to(stats.dtype)
    m, log_s = stats[:, :1], stats[:, 1:]
    empty = (m == -math.inf) & (log_s == 0)
    return (z - torch.where(m == -math.inf, torch.zeros_like(m), m)) / temperature - log_s, empty


def _forward_torch(logits, targets, top, entropy, ignore_index, temperature):
    shape, vocab = targets.shape, logits.shape[-1]
    z = logits.detach().reshape(-1, vocab)
    z = z if z.dtype == torch.float64 else z.float()
    t = targets.reshape(-1, 1).long()
    m = z.amax(1, keepdim=True)
    base = torch.where(m == -math.inf, torch.zeros_like(m), m)
    s = torch.exp((z - base) / temperature).sum(1, keepdim=True)
    stats = torch.cat([m, torch.where((m == -math.inf) & (s == 0), torch.zeros_like(s), torch.log(s))], 1)
    log_p, empty = _scaled(z, stats, temperature)
    known, ignored = (t >= 0) & (t < vocab), t == ignore_index
    log_probs = torch.where(known, log_p.gather(1, t.clamp(0, vocab - 1)), torch.full_like(m, math.nan))
    log_probs = torch.where(ignored, torch.zeros_like(m), log_probs)
    h = None
    if entropy:
        p = torch.exp(log_p)
        h = -torch.where(p == 0, torch.zeros_like(p), p * log_p).sum(1)
        h = h.view(shape)
    values = tokens = None
    if top:
        tokens = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]
        values = log_p.gather(1, tokens).view(*shape, top)
        tokens = tokens.reshape(*shape, top).contiguous()
    return log_probs.view(shape), h, values, tokens, stats


def _backward_torch(logits, targets, stats, entropy, tokens, g, g_entropy, g_top, ignore_index, temperature):
    vocab = logits.shape[-1]
    log_p, empty = _scaled(logits.detach(), stats, temperature)
    p = torch.exp(log_p)
    t = targets.reshape(-1, 1).long()
    known, ignored = (t >= 0) & (t < vocab), t == ignore_index
    zero = torch.zeros_like(stats[:, :1])
    all_of = zero.clone()
    at_target = zero
    if g is not None:
        at_target = torch.where(ignored, zero, g.reshape(-1, 1).to(zero.dtype))
        at_target = torch.where(known | ignored, at_target, torch.full_like(zero, math.nan))   # (entropy and alternatives do not depend on the target)
    all_of = all_of + at_target
    if g_top is not None:
        g_top = g_top.reshape(p.shape[0], -1).to(zero.dtype)
        all_of = all_of + g_top.sum(1, keepdim=True)
    dz = -p * all_of
    if g_entropy is not None:
        p_log_p = torch.where(p == 0, torch.zeros_like(p), p * log_p)
        dz = dz - g_entropy.reshape(-1, 1).to(zero.dtype) * (p_log_p + p * entropy.reshape(-1, 1))
    dz.scatter_add_(1, t.clamp(0, vocab - 1), torch.where(known, at_target, zero))
    if g_top is not None:
        dz.scatter_add_(1, tokens.reshape(p.shape[0], -1), g_top)
    return (torch.where(empty, torch.zeros_like(dz), dz) / temperature).to(logits.dtype).view(logits.shape)
