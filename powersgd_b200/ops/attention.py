"""Attention over packed sequences (csrc/attention.cu): sequences of different lengths one behind another in one tensor,
without padding, with a backward pass and with fewer key heads than query heads where wanted.

On the CPU (or on CUDA without the native library where PSGD_B200_ALLOW_FALLBACK=1 allows it) the same comes from torch
operations, one sequence after another.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import native
from .host import operators

DTYPES = {torch.bfloat16: 1, torch.float16: 2}
MOST_SIZE = 128

_statuses: dict = {}   # device -> status word that kernels write when a wait of theirs runs out


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets: torch.Tensor, *, causal: bool = True,
                     scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of each sequence by itself; a position sees those up to its own (`causal`) or all of its sequence.

    `q`: [tokens, heads, size]; `k`, `v`: [tokens, key heads, size], where the query heads h n to (h + 1) n - 1 share key head h,
    n = heads / key heads. bfloat16 or float16 on the GPU; size up to 128, a multiple of 8. `offsets`: int32,
    [sequences + 1], on the tensors' device, never decreasing: sequence s has the rows offsets[s] to offsets[s + 1], and may have none.
    It is read by the kernels and not by the host: a call neither waits nor checks it, values outside [0, tokens] are taken for the
    nearer end, and what sequences that overlap give is not defined. Rows that belong to no sequence give zeros, whatever they
    hold. `scale`: 1 / sqrt(size) unless given; 2^-100 to 2^100.

    Differentiable (once, backwards) in q, k and v, whose gradients have the shapes of these; all three are computed where one is asked for. Until
    then a second tensor as large as the output is kept, what rounding took from it. The result and the gradients are the same
    in every run. Tensors may be views, as parts of one projection are: rows and heads that do not begin on 16-byte boundaries, or
    elements that do not lie side by side, are copied first. Under float16 a gradient beyond its range becomes infinite. Positions that
    see a score which is no number give NaN; where a row of q, k, v or a gradient is not finite, any other of its sequence may."""
    if operators is not None and (scale is None or scale > 0):
        out = operators.packed_attention(q, k, v, offsets, causal, 0.0 if scale is None else scale)
        if out is not None:
            return out
    check(q, k, v, offsets, scale)
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _PackedAttention.apply(q, k, v, offsets, bool(causal), scale)
    return _forward(q, k, v, offsets, bool(causal), scale, False)[0]


def check(q, k, v, offsets, scale) -> None:
    native.refuse_tracing("packed_attention", q)
    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together; [tokens, heads, size] is expected")
    heads, groups, size = q.shape[1], k.shape[1], q.shape[2]
    if groups < 1 or heads < 1 or heads % groups:
        raise ValueError(f"packed_attention: {heads} query heads over {groups} key heads")
    if not 8 <= size <= MOST_SIZE or size % 8:
        raise ValueError(f"packed_attention: heads of {size}; multiples of 8 up to {MOST_SIZE} are supported")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise TypeError(f"packed_attention: q, k and v are {q.dtype}, {k.dtype} and {v.dtype}")
    if q.dtype not in DTYPES and (q.is_cuda or not q.dtype.is_floating_point):
        raise TypeError(f"packed_attention: {q.dtype}; bfloat16 and float16 are supported")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"packed_attention: offsets are {offsets.dtype} {tuple(offsets.shape)}; int32 [sequences + 1] is expected")
    if not (q.device == k.device == v.device == offsets.device):
        raise ValueError(f"packed_attention: tensors on {q.device}, {k.device}, {v.device} and {offsets.device}")
    if q.shape[0] >= 2**31 - 2**16:
        raise ValueError(f"packed_attention: {q.shape[0]} tokens")
    if offsets.shape[0] > 2**31 - 2**16:
        raise ValueError(f"packed_attention: {offsets.shape[0] - 1} sequences")
    if scale is not None and not 2.0**-100 <= scale <= 2.0**100:
        raise ValueError(f"packed_attention: scale {scale}; 2^-100 to 2^100")
    native.refuse_tangents("packed_attention", q, k, v)


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and native.use_for_cuda()


def _status(device: torch.device):
    """The device's status word: raises if a wait has run out since the last call."""
    word = _statuses.get(device)
    if word is None:
        host, dev = ctypes.POINTER(ctypes.c_int)(), ctypes.POINTER(ctypes.c_int)()
        with native.relaxed_capture():
            native.check(native.lib().psgd_status_alloc(ctypes.byref(host), ctypes.byref(dev)), "psgd_status_alloc")
        word = _statuses[device] = (host, ctypes.cast(dev, ctypes.c_void_p).value)
        if operators is not None:
            operators.status(device.index, ctypes.cast(host, ctypes.c_void_p).value, word[1])
    code = word[0][0]
    if code:
        word[0][0] = 0
        raise RuntimeError(f"packed_attention: a wait of an earlier call ran out on {device} (status {code}); its results are not valid")
    return word[1]


def check_waits() -> None:
    """Raises RuntimeError if a wait inside an attention kernel has run out, on any device, in what has ended by now. Every call of `packed_attention`
    asks this of the calls before it; a program asks it behind its last call and behind replays of a graph, once these have ended."""
    for device in list(_statuses):
        _status(device)


def _usable(t: torch.Tensor) -> torch.Tensor:
    """As the kernels address it: elements of a head side by side, rows and heads on 16-byte boundaries and apart. A copy if need be."""
    t = native.in_memory(t)
    tokens, heads, size = t.shape
    row, head, one = t.stride()
    if (one == 1 or size == 1) and t.data_ptr() % 16 == 0 and (tokens == 1 or (row % 8 == 0 and row >= size)) and (heads == 1 or (head % 8 == 0 and head >= size)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(*tensors) -> ctypes.Array:
    """Of rows and heads; where there is only one of them, any that is allowed."""
    out = []
    for t in tensors:
        tokens, heads, size = t.shape
        out += [t.stride(0) if tokens > 1 else heads * size, t.stride(1) if heads > 1 else size]
    return (ctypes.c_longlong * len(out))(*out)


def _plan(sequences: int, tokens: int, device: torch.device) -> Optional[torch.Tensor]:
    """Scratch for the order of the tiles, where there are many sequences."""
    ints = native.lib().psgd_attention_plan_ints(sequences, tokens)
    return torch.empty(ints, dtype=torch.int32, device=device) if ints else None


def _forward(q, k, v, offsets, causal, scale, gradient: bool):
    """The output, and for a backward pass the logarithms of the sums and what rounding took from the output."""
    if not _native(q):
        return _forward_torch(q, k, v, offsets, causal, scale)
    tokens, heads, size = q.shape
    sequences = offsets.shape[0] - 1
    out = torch.empty((tokens, heads, size), dtype=q.dtype, device=q.device)
    if tokens == 0 or sequences == 0:
        return out.zero_(), None, None
    lse = torch.empty((heads, tokens), dtype=torch.float32, device=q.device)
    rest = torch.empty_like(out) if gradient else None
    q, k, v, offsets, plan = _usable(q), _usable(k), _usable(v), offsets.contiguous(), _plan(sequences, tokens, q.device)
    with native.on_device(q.device) as stream:
        code = native.lib().psgd_attention(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), _strides(q, k, v), offsets.data_ptr(), sequences, tokens, heads, k.shape[1], size, DTYPES[q.dtype],
            causal, scale, out.data_ptr(), rest.data_ptr() if gradient else None, lse.data_ptr(), None if plan is None else plan.data_ptr(),
            _status(q.device), stream,
        )
    native.check(code, "psgd_attention")
    return out, lse, rest


def _backward(q, k, v, offsets, out, lse, rest, grad, causal, scale):
    if not _native(q):
        return _backward_torch(q, k, v, offsets, out, grad, causal, scale)
    tokens, heads, size = q.shape
    groups, sequences = k.shape[1], offsets.shape[0] - 1
    dq = torch.empty((tokens, heads, size), dtype=q.dtype, device=q.device)
    dk = torch.empty((tokens, groups, size), dtype=q.dtype, device=q.device)
    dv = torch.empty_like(dk)
    if tokens == 0 or sequences == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    delta = torch.empty((2 * heads + groups if q.dtype == torch.float16 else heads, tokens), dtype=torch.float32, device=q.device)   # scratch
    q, k, v, grad, offsets, plan = _usable(q), _usable(k), _usable(v), _usable(grad), offsets.contiguous(), _plan(sequences, tokens, q.device)
    with native.on_device(q.device) as stream:
        code = native.lib().psgd_attention_backward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), grad.data_ptr(), _strides(q, k, v, grad), offsets.data_ptr(), sequences, tokens, heads, groups, size,
            DTYPES[q.dtype], causal, scale, out.data_ptr(), rest.data_ptr(), lse.data_ptr(), delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            None if plan is None else plan.data_ptr(), _status(q.device), stream,
        )
    native.check(code, "psgd_attention_backward")
    return dq, dk, dv


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets, causal, scale):
        out, lse, rest = _forward(q, k, v, offsets, causal, scale, True)
        ctx.save_for_backward(q, k, v, offsets, out, lse, rest)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        native.refuse_tangents("packed_attention", grad)
        q, k, v, offsets, out, lse, rest = ctx.saved_tensors
        return (*_backward(q, k, v, offsets, out, lse, rest, grad, ctx.causal, ctx.scale), None, None, None)


# ---- the same in torch operations --------------------------------------------------------------
def _sequences(offsets: torch.Tensor, tokens: int):
    ends = offsets.clamp(0, tokens).tolist()
    return [(lo, hi) for lo, hi in zip(ends, ends[1:]) if hi > lo]


def _wide(t: torch.Tensor, repeat: int = 1) -> torch.Tensor:
    """[rows, heads, size] as [heads, rows, size] in float32 (float64 stays)."""
    t = t.detach().transpose(0, 1)
    t = t if t.dtype == torch.float64 else t.float()
    return t.repeat_interleave(repeat, 0) if repeat > 1 else t


def _weights(q, k, causal, scale):
    s = q @ k.transpose(1, 2) * scale
    if causal:
        n = q.shape[1]
        s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), -math.inf)
    return torch.softmax(s, -1)


def _forward_torch(q, k, v, offsets, causal, scale):
    out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    group = q.shape[1] // k.shape[1]
    for lo, hi in _sequences(offsets, q.shape[0]):
        p = _weights(_wide(q[lo:hi]), _wide(k[lo:hi], group), causal, scale)
        out[lo:hi] = (p @ _wide(v[lo:hi], group)).transpose(0, 1).to(q.dtype)
    return out, None, None


def _backward_torch(q, k, v, offsets, out, grad, causal, scale):
    group = q.shape[1] // k.shape[1]
    dq, dk, dv = (torch.zeros(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
    for lo, hi in _sequences(offsets, q.shape[0]):
        qq, kk, vv, g = _wide(q[lo:hi]), _wide(k[lo:hi], group), _wide(v[lo:hi], group), _wide(grad[lo:hi])
        p = _weights(qq, kk, causal, scale)
        ds = p * (g @ vv.transpose(1, 2) - (g * (p @ vv)).sum(-1, keepdim=True)) * scale
        shared = lambda x: x.view(k.shape[1], group, *x.shape[1:]).sum(1).transpose(0, 1)  # noqa: E731
        dq[lo:hi] = (ds @ kk).transpose(0, 1).to(q.dtype)
        dk[lo:hi] = shared(ds.transpose(1, 2) @ qq).to(q.dtype)
        dv[lo:hi] = shared(p.transpose(1, 2) @ g).to(q.dtype)
    return dq, dk, dv
