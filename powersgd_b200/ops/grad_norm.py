"""The norm of many gradients taken together, and clipping (csrc/grad_norm.cu).

On the CPU (or on CUDA without the native library where PSGD_B200_ALLOW_FALLBACK=1 allows it) the same comes from torch
operations, one tensor after another.
"""
from __future__ import annotations

import math
from typing import Iterable, List, Union

import numpy as np
import torch

from . import native, scan
from .adamw import in_one_piece
from .host import operators

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}

# one tensor of a list, see PsgdNormTensor
ITEM = np.dtype([("g", "u8"), ("n", "i8"), ("type", "u4"), ("piece_end", "u4")])
assert ITEM.itemsize == 24


def grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all gradients of `parameters` as if they were one vector: the root of the sum of squares, or the largest magnitude
    (`norm_type` infinity). See `clip_grad_norm`; a parameter that is listed twice counts twice, and gradients may lie in each other's memory."""
    return _norm(_listed(parameters), _largest("grad_norm", norm_type), None)


def clip_grad_norm(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                   error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales the gradients of `parameters` by max_norm / (norm + 1e-6) where that is below one, and returns their norm before that: a tensor without
    dimensions on their device, float32 (float64 where a gradient is), zero where there are none. As `torch.nn.utils.clip_grad_norm_`, in one launch or two for
    up to 1200 tensors (two more for each 1200 after them) and without waiting for the GPU.

    Gradients are plain tensors (no DTensors), dense, float32, bfloat16, float16 or float64, in one list if need be, of one device, and none lies in another's
    memory (a parameter is listed once). Those that do not lie in one piece are copied to and fro. Squares are added in float64; a
    gradient is rounded once. Where the norm is no number all gradients become NaN, where it is infinite finite ones become zero:
    with `error_if_nonfinite` a RuntimeError is raised instead and nothing is changed; it waits for the GPU. A norm that float32 does not hold is
    returned as infinity, and gradients are scaled by what it is. Squares of float64 gradients leave the range from 1.3e154 on: their norm is infinite, as
    the library's is (the largest magnitude has no such bound).

    May be recorded in a CUDA graph, which reads the gradients where they lay, and `max_norm` as it was, at every replay."""
    largest = _largest("clip_grad_norm", norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm: max_norm {max_norm}; zero or more is expected")
    listed = _listed(parameters)
    if error_if_nonfinite:
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("clip_grad_norm: error_if_nonfinite waits for the GPU, which cannot be recorded")
        norm = _norm(listed, largest, None)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"clip_grad_norm: the norm of the gradients is {norm.item()}; nothing was scaled")
    return _norm(listed, largest, max_norm)


def clip_for_step(parameters: Iterable[torch.Tensor], max_norm: float) -> torch.Tensor:
    """What a training loop of this package clips with: `clip_grad_norm` on the GPU. Gradients on the CPU, and lists that it refuses (complex
    gradients, DTensors, several devices), go to the library, which refuses sparse ones too."""
    listed = _listed(parameters)
    if any(p.is_cuda for p in listed):
        try:
            return clip_grad_norm(listed, max_norm)
        except (TypeError, ValueError):     # (nothing was changed)
            pass
    return torch.nn.utils.clip_grad_norm_(listed, max_norm)


def _largest(what: str, norm_type: float) -> bool:
    if norm_type not in (2, math.inf):
        raise ValueError(f"{what}: norm_type {norm_type}; 2 and infinity are supported")
    return norm_type != 2


def _listed(parameters) -> List[torch.Tensor]:
    return [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)


def _norm(parameters: List[torch.Tensor], largest: bool, max_norm) -> torch.Tensor:
    """The norm; gradients are scaled unless `max_norm` is None."""
    if operators is not None:
        out = operators.grad_norm(parameters, largest, max_norm is not None, 0.0 if max_norm is None else max_norm)
        if out is not None:
            return out
    with torch.no_grad():
        return _norm_checked("grad_norm" if max_norm is None else "clip_grad_norm", parameters, largest, max_norm)


def _norm_checked(what: str, parameters: List[torch.Tensor], largest: bool, max_norm) -> torch.Tensor:
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else None)
    native.refuse_tracing(what, grads[0])
    native.refuse_without_memory(what, *grads)
    for i, g in enumerate(grads):
        if g.layout != torch.strided:
            raise TypeError(f"{what}: gradient {i} is {g.layout}; dense gradients are supported")
        if g.dtype not in DTYPES:
            raise TypeError(f"{what}: gradient {i} is {g.dtype}; float32, bfloat16, float16 and float64 are supported")
        if g.device != grads[0].device:
            raise ValueError(f"{what}: gradients on {grads[0].device} and {g.device}")
    native.refuse_tangents(what, *grads)
    if max_norm is not None:
        _refuse_overlaps(what, grads)
    if not (grads[0].is_cuda and native.use_for_cuda()):
        return _norm_torch(grads, largest, max_norm)
    # as the kernels take them: in one piece (that a tensor says to be negated does not matter here)
    laid = [g if in_one_piece(g) and not g._is_zerotensor() else native.in_memory(g).contiguous() for g in grads]
    items = np.zeros(len(laid), dtype=ITEM)
    items["g"] = np.frombuffer(scan.addresses(laid), dtype=np.uint64)
    items["n"] = [g.numel() for g in laid]
    items["type"] = [DTYPES[g.dtype] for g in laid]
    device, wide, listed = grads[0].device, any(g.dtype == torch.float64 for g in grads), items.tobytes()
    out = torch.empty((), dtype=torch.float64 if wide else torch.float32, device=device)
    with native.on_device(device) as stream:
        words = native.lib().psgd_grad_norm_parts(listed, len(laid))     # (asks what the device runs)
        parts = torch.empty(words, dtype=torch.float64, device=device)
        code = native.lib().psgd_grad_norm(listed, len(laid), largest, max_norm is not None, 0.0 if max_norm is None else max_norm, parts.data_ptr() if words else None,
                                           out.data_ptr(), wide, stream)
    native.check(code, "psgd_grad_norm")
    if max_norm is not None:
        for g, t in zip(grads, laid):
            if t is not g and not g._is_zerotensor():
                g.copy_(t)
        torch.autograd.graph.increment_version([g for g, t in zip(grads, laid) if t is g and not g.is_inference()])   # (torch operations do so themselves)
    return out


def _refuse_overlaps(what: str, grads: List[torch.Tensor]) -> None:
    places = []
    for i, g in enumerate(grads):
        if g.numel() == 0 or g._is_zerotensor() or g.device.type not in ("cpu", "cuda"):
            continue
        if any(n > 1 and s == 0 for n, s in zip(g.shape, g.stride())):
            raise ValueError(f"{what}: gradient {i} has elements that share memory (shape {tuple(g.shape)}, strides {g.stride()})")
        if in_one_piece(g):    # (views with gaps may lie in each other's)
            places.append((g.data_ptr(), g.data_ptr() + g.numel() * g.element_size(), i))
    places.sort()
    for (_, end, i), (start, _, j) in zip(places, places[1:]):
        if start < end:
            raise ValueError(f"{what}: gradients {min(i, j)} and {max(i, j)} share memory; a parameter is listed once")


# ---- the same in torch operations --------------------------------------------------------------
def _norm_torch(grads: List[torch.Tensor], largest: bool, max_norm) -> torch.Tensor:
    parts = [g.abs().max().double() if largest else g.double().square().sum() for g in grads if g.numel()]
    total = torch.stack(parts) if parts else torch.zeros(1, dtype=torch.float64, device=grads[0].device)
    norm = total.max() if largest else total.sum().sqrt()
    if max_norm is not None:
        factor = max_norm / (norm + 1e-6)
        factor = torch.where(factor >= 1, torch.ones_like(factor), factor)
        down = torch.where(factor < 2.0**-126, torch.full_like(factor, 2.0**-126), torch.ones_like(factor))      # (below the normal numbers of 32 bits few digits would be left)
        for g in grads:
            if not g._is_zerotensor():
                g.copy_(g * factor if g.dtype == torch.float64 else g.float() * down.float() * (factor / down).float())
    return norm if any(g.dtype == torch.float64 for g in grads) else norm.float()
