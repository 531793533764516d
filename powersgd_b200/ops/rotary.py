"""Heads normed and turned by their row's position (csrc/rotary.cuh): what a transformer does to its queries and keys between
their projection and the attention.

On the CPU (or on CUDA without the native library where PSGD_B200_ALLOW_FALLBACK=1 allows it) the same comes from torch
operations.
"""
from __future__ import annotations

import ctypes
import decimal
import functools
import math
from typing import Optional, Tuple

import torch

from . import native
from .attention import _strides, _usable
from .host import operators

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MOST_SIZE = 256
MOST_HEADS = 4096


class Call(ctypes.Structure):
    """PsgdRotate, see csrc/rotary.cuh."""

    _fields_ = [("x", ctypes.c_void_p), ("grad", ctypes.c_void_p * 3), ("weight", ctypes.c_void_p * 2), ("offsets", ctypes.c_void_p), ("positions", ctypes.c_void_p),
                ("out", ctypes.c_void_p * 2), ("dx", ctypes.c_void_p), ("dweight", ctypes.c_void_p * 2), ("parts", ctypes.c_void_p), ("frequencies", ctypes.c_void_p),
                ("x_row", ctypes.c_longlong), ("x_head", ctypes.c_longlong), ("grad_row", ctypes.c_longlong * 3), ("grad_head", ctypes.c_longlong * 3),
                *((name, ctypes.c_int) for name in ("rows", "sequences", "heads", "keys", "values", "size", "rotated", "pairs", "type", "weight_type", "wide", "norm")),
                ("eps", ctypes.c_float), ("pad", ctypes.c_int)]


assert ctypes.sizeof(Call) == 240 and Call.x_row.offset == 120 and Call.rows.offset == 184


def rotate_heads(x: torch.Tensor, *, offsets: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None,
                 eps: Optional[float] = 1e-6, base: float = 10000.0, rotated: Optional[int] = None, interleaved: bool = False) -> torch.Tensor:
    """Each head of `x` divided by the root of its mean square and multiplied with `weight`, and its first `rotated` elements turned pair by
    pair by position * base^(-2 i / rotated), i = 0 to rotated / 2 - 1.

    `x`: [rows, heads, size], float32, bfloat16 or float16 on the GPU; size a multiple of 8 up to 256, up to 4096 heads. `rotated`: a multiple of 8, all of the head
    unless given, or 0. Pairs are (i, i + rotated / 2), or (2 i, 2 i + 1) with `interleaved`. `eps` is added to the mean square, 2^-100 to 1; None: no
    norm. `weight`: [size], float32 or of the type of x; None: ones.

    Positions come from `offsets` (int32, [sequences + 1], as `packed_attention` takes them: a sequence's rows are counted from zero; rows that
    belong to no sequence give zeros, whatever they hold) or from `positions` (int32 or int64, [rows], below zero too). Both are read by the kernels and not by the host. Without a
    rotation neither is needed. Angles are off by |position| * 2^-65 turns, in float32 and less by 2^-32 more: for positions up to 2^38 (some 2.7e11) less than a float32's rounding, 1.7e-4 radians at
    10^15, and of no meaning from some 2^60 on.

    Differentiable (once, backwards) in x and weight. The result and the gradients are the same in every run. `x` may be a view; rows and
    heads that do not begin on 16-byte boundaries are copied first. A head that holds what is no number is spoiled, and with it the weight's gradient."""
    return _rotate("rotate_heads", x, x.shape[1] if x.dim() == 3 else 0, 0, offsets, positions, weight, None, eps, base, rotated, interleaved)[0]


def rotate_projection(qkv: torch.Tensor, heads: int, key_heads: int, *, offsets: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                      q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: Optional[float] = 1e-6, base: float = 10000.0,
                      rotated: Optional[int] = None, interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Queries, keys and values of one projection, the first two as `rotate_heads` makes them.

    `qkv`: [rows, heads + key_heads + value heads, size], in this order. The values are a view of it, whose memory they keep. Its gradient is written
    once, in one piece: nothing has to be put together behind the attention's three. The weights have one type."""
    return _rotate("rotate_projection", qkv, heads, key_heads, offsets, positions, q_weight, k_weight, eps, base, rotated, interleaved)


def _rotate(what, x, heads, keys, offsets, positions, q_weight, k_weight, eps, base, rotated, interleaved):
    rotated = x.shape[-1] if rotated is None and x.dim() else rotated
    if isinstance(rotated, int) and 0 <= rotated <= MOST_SIZE and rotated % 8 == 0 and 1 <= base <= 1e30 and (eps is None or 2.0**-100 <= eps <= 1):
        table = frequencies(rotated, float(base))
        if operators is not None and (keys > 0 or what == "rotate_heads"):
            out = operators.rotate(x, heads, keys, offsets, positions, q_weight, k_weight, -1.0 if eps is None else eps, rotated, interleaved, table)
            if out is not None:
                return out
    check(what, x, heads, keys, offsets, positions, q_weight, k_weight, eps, base, rotated)
    arguments = (heads, keys, eps, rotated, bool(interleaved), float(base))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, q_weight, k_weight)):
        return _Rotate.apply(x, q_weight, k_weight, offsets, positions, *arguments)
    return _forward(x, q_weight, k_weight, offsets, positions, *arguments)


def check(what, x, heads, keys, offsets, positions, q_weight, k_weight, eps, base, rotated) -> None:
    native.refuse_tracing(what, x)
    native.refuse_without_memory(what, x, q_weight, k_weight, offsets, positions)
    if x.dim() != 3:
        raise ValueError(f"{what}: {tuple(x.shape)}; [rows, heads, size] is expected")
    rows, have, size = x.shape
    if heads < 1 or keys < 0 or (keys < 1 and what != "rotate_heads") or heads + keys > have:
        raise ValueError(f"{what}: {heads} query heads and {keys} key heads of {have}")
    if not 8 <= size <= MOST_SIZE or size % 8:
        raise ValueError(f"{what}: heads of {size}; multiples of 8 up to {MOST_SIZE} are supported")
    if not isinstance(rotated, int) or not 0 <= rotated <= size or rotated % 8:
        raise ValueError(f"{what}: {rotated} elements of {size} turned; a multiple of 8 is expected")
    if x.dtype not in DTYPES and (x.is_cuda or not x.dtype.is_floating_point):
        raise TypeError(f"{what}: {x.dtype}; float32, bfloat16 and float16 are supported")
    if rows >= 2**31 - 2**16 or have > MOST_HEADS:
        raise ValueError(f"{what}: {rows} rows of {have} heads")
    if not (math.isfinite(base) and 1 <= base <= 1e30):
        raise ValueError(f"{what}: base {base}; 1 to 1e30")
    if eps is not None and not 2.0**-100 <= eps <= 1:
        raise ValueError(f"{what}: eps {eps}; 2^-100 to 1, or None")
    if offsets is not None and positions is not None or rotated and offsets is None and positions is None:
        raise ValueError(f"{what}: one of offsets and positions is expected")
    if offsets is not None and (offsets.dtype != torch.int32 or offsets.dim() != 1 or not 1 <= offsets.shape[0] <= 2**31 - 2**16):
        raise ValueError(f"{what}: offsets are {offsets.dtype} {tuple(offsets.shape)}; int32 [sequences + 1] is expected")
    if positions is not None and (positions.dtype not in (torch.int32, torch.int64) or positions.shape != (rows,)):
        raise ValueError(f"{what}: positions are {positions.dtype} {tuple(positions.shape)}; int32 or int64 [{rows}] is expected")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if eps is None:
            raise ValueError(f"{what}: weights without a norm (eps is None)")
        if w.shape != (size,):
            raise ValueError(f"{what}: weights {tuple(w.shape)}; [{size}] is expected")
        if w.dtype not in (torch.float32, x.dtype) or w.dtype != weights[0].dtype:
            raise TypeError(f"{what}: weights are {w.dtype}; all float32 or all {x.dtype} is expected")
    for t in (*weights, offsets, positions):
        if t is not None and t.device != x.device:
            raise ValueError(f"{what}: tensors on {x.device} and {t.device}")
    native.refuse_tangents(what, x, *weights)


@functools.lru_cache(maxsize=64)
def frequencies(rotated: int, base: float) -> bytes:
    """base^(-2 i / rotated) in turns per position: 64-bit fractions, rounded once."""
    with decimal.localcontext() as context:
        context.prec = 50
        turn = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582")
        fractions = [decimal.Decimal(base) ** (decimal.Decimal(-2 * i) / rotated) / turn for i in range(rotated // 2)]
        return b"".join(int((f * 2**64).to_integral_value()).to_bytes(8, "little") for f in fractions)


def _call(x, q_weight, k_weight, offsets, positions, heads, keys, eps, rotated, pairs, table) -> Call:
    call = Call()
    call.x, (call.x_row, call.x_head) = x.data_ptr(), _strides(x)
    for i, w in enumerate((q_weight, k_weight)):
        if w is not None:
            call.weight[i], call.weight_type = w.data_ptr(), DTYPES[w.dtype]
    if offsets is not None:
        call.offsets, call.sequences = offsets.data_ptr(), offsets.shape[0] - 1
    if positions is not None:
        call.positions, call.wide = positions.data_ptr(), positions.dtype == torch.int64
    call.frequencies = ctypes.cast(table, ctypes.c_void_p)
    call.rows, call.heads, call.keys, call.values, call.size = x.shape[0], heads, keys, x.shape[1] - heads - keys, x.shape[2]
    call.rotated, call.pairs, call.type = rotated, pairs, DTYPES[x.dtype]
    call.norm, call.eps = eps is not None, 0.0 if eps is None else eps
    return call


def _laid(*tensors):
    return [None if t is None else native.in_memory(t).contiguous() for t in tensors]


def _native(t: torch.Tensor) -> bool:
    return t.is_cuda and native.use_for_cuda()


def _forward(x, q_weight, k_weight, offsets, positions, heads, keys, eps, rotated, pairs, base):
    if not _native(x):
        return _forward_torch(x, q_weight, k_weight, offsets, positions, heads, keys, eps, rotated, pairs, base)
    rows, _, size = x.shape
    q = torch.empty((rows, heads, size), dtype=x.dtype, device=x.device)
    k = torch.empty((rows, keys, size), dtype=x.dtype, device=x.device) if keys else None
    laid, table = _usable(x), frequencies(rotated, base)
    tensors = _laid(q_weight, k_weight, offsets, positions)
    call = _call(laid, *tensors, heads, keys, eps, rotated, pairs, table)
    call.out[0] = q.data_ptr()
    if keys:
        call.out[1] = k.data_ptr()
    with native.on_device(x.device) as stream:
        code = native.lib().psgd_rotate(ctypes.byref(call), stream)
    native.check(code, "psgd_rotate")
    return (q, k, x[:, heads + keys :]) if keys else (q,)


def _backward(x, q_weight, k_weight, offsets, positions, grads, needs, heads, keys, eps, rotated, pairs, base):
    """The gradients of x and the weights, those that `needs` says."""
    if not _native(x):
        return _backward_torch(x, q_weight, k_weight, offsets, positions, grads, needs, heads, keys, eps, rotated, pairs, base)
    laid, table = _usable(x), frequencies(rotated, base)
    tensors = _laid(q_weight, k_weight, offsets, positions)
    call = _call(laid, *tensors, heads, keys, eps, rotated, pairs, table)
    grads = [None if g is None else _usable(g) for g in grads]
    for i, g in enumerate(grads):
        if g is not None:
            call.grad[i], (call.grad_row[i], call.grad_head[i]) = g.data_ptr(), _strides(g)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if needs[0] else None
    if dx is not None:
        call.dx = dx.data_ptr()
    dweights, parts = [None, None], None
    for i, w in enumerate(tensors[:2]):
        if w is not None and needs[1 + i]:
            dweights[i] = torch.empty_like(w) if x.shape[0] else torch.zeros_like(w)
            call.dweight[i] = dweights[i].data_ptr()
            parts = torch.empty(native.lib().psgd_rotate_parts(x.shape[2]), dtype=torch.float64, device=x.device) if parts is None else parts
            call.parts = parts.data_ptr()
    with native.on_device(x.device) as stream:
        code = native.lib().psgd_rotate_grad(ctypes.byref(call), stream)
    native.check(code, "psgd_rotate_grad")
    return dx, *dweights


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, q_weight, k_weight, offsets, positions, *arguments):
        ctx.save_for_backward(x, q_weight, k_weight, offsets, positions)
        ctx.arguments = arguments
        ctx.set_materialize_grads(False)
        return _forward(x, q_weight, k_weight, offsets, positions, *arguments)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        native.refuse_without_memory("rotate_heads", *grads)
        native.refuse_tangents("rotate_heads", *grads)
        return (*_backward(*ctx.saved_tensors, grads, ctx.needs_input_grad, *ctx.arguments), *[None] * (2 + len(ctx.arguments)))


# ---- the same in torch operations --------------------------------------------------------------
def _wide(t: torch.Tensor) -> torch.Tensor:
    t = t.detach()
    return t if t.dtype == torch.float64 else t.float()


def _angles(x, offsets, positions, rotated, base):
    """Cosines and sines of the rows' angles, and which rows belong to a sequence."""
    rows, device = x.shape[0], x.device
    held = torch.ones(rows, 1, 1, dtype=torch.bool, device=device)
    if offsets is not None:
        row = torch.arange(rows, device=device)
        sequence = torch.searchsorted(offsets.long(), row, right=True)
        held = ((sequence > 0) & (sequence < offsets.shape[0]))[:, None, None]
        positions = row - offsets.long()[(sequence - 1).clamp_min(0)].clamp_min(0)
    if not rotated:
        return None, None, held
    table = frequencies(rotated, base)
    fraction = torch.tensor([int.from_bytes(table[i : i + 8], "little", signed=True) for i in range(0, len(table), 8)], device=device)
    angle = ((positions.long()[:, None] * fraction).double() * (2 * math.pi / 2**64))[:, None]     # (whole turns are beyond the 64 bits)
    dtype = _wide(x[:0]).dtype
    return angle.cos().to(dtype), angle.sin().to(dtype), held


def _turn(y, cosine, sine, rotated, pairs):
    if not rotated:
        return y
    a, b = (y[..., 0:rotated:2], y[..., 1:rotated:2]) if pairs else (y[..., : rotated // 2], y[..., rotated // 2 : rotated])
    a, b = a * cosine - b * sine, b * cosine + a * sine
    turned = torch.stack((a, b), -1).flatten(-2) if pairs else torch.cat((a, b), -1)
    return torch.cat((turned, y[..., rotated:]), -1)


def _normed(part, eps):
    """x r and r; heads whose squares leave the range are made smaller first."""
    down = torch.where(part.abs().amax(-1, keepdim=True) < 2.0**60, 1.0, 2.0**-70).to(part.dtype)
    part = part * down
    r = torch.rsqrt(part.square().mean(-1, keepdim=True) + eps * down.double().square().to(part.dtype))
    return part * r, r * down


def _kinds(x, q_weight, k_weight, heads, keys):
    return [(x[:, :heads], q_weight)] + ([(x[:, heads : heads + keys], k_weight)] if keys else [])


def _forward_torch(x, q_weight, k_weight, offsets, positions, heads, keys, eps, rotated, pairs, base):
    cosine, sine, held = _angles(x, offsets, positions, rotated, base)
    out = []
    for part, weight in _kinds(x, q_weight, k_weight, heads, keys):
        y = _wide(part)
        if eps is not None:
            y, _ = _normed(y, eps)
        if weight is not None:
            y = y * _wide(weight)
        y = _turn(y, cosine, sine, rotated, pairs)
        out.append(torch.where(held, y, torch.zeros_like(y)).to(x.dtype))
    return (*out, x[:, heads + keys :]) if keys else tuple(out)


def _backward_torch(x, q_weight, k_weight, offsets, positions, grads, needs, heads, keys, eps, rotated, pairs, base):
    cosine, sine, held = _angles(x, offsets, positions, rotated, base)
    dx, dweights = [], []
    for (part, weight), grad in zip(_kinds(x, q_weight, k_weight, heads, keys), grads):
        d = torch.zeros_like(_wide(part)) if grad is None else _wide(grad)
        d = _turn(d, cosine, None if sine is None else -sine, rotated, pairs)
        n, r = _normed(_wide(part), eps) if eps is not None else (None, None)
        dweights.append(None if weight is None else torch.where(held, d * n, torch.zeros_like(n)).sum((0, 1)).to(weight.dtype))
        if weight is not None:
            d = d * _wide(weight)
        if eps is not None:
            d = (d - n * (d * n).mean(-1, keepdim=True)) * r
        dx.append(torch.where(held, d, torch.zeros_like(d)).to(x.dtype))
    if keys:
        dx.append(torch.zeros_like(x[:, heads + keys :]) if grads[2] is None else grads[2])
    dweights += [None] * (2 - len(dweights))
    return torch.cat(dx, 1) if needs[0] else None, *[w if need else None for w, need in zip(dweights, needs[1:3])]
