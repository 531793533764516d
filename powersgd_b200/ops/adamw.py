"""One AdamW step over a list of tensors (csrc/adamw.cu), with moments in 32 bits or in 8.

`adamw_step` takes lists as `torch.optim`'s functional forms do and changes them in place; `AdamW` (optim.py)
calls it for each of its parameter groups. On the CPU (or on CUDA without the native library where
PSGD_B200_ALLOW_FALLBACK=1 allows it) the same step is made of torch operations, the rounding of 8-bit moments included.

Moments in 8 bits are e4m3 tensors of the parameter's shape with one float32 scale per 256 elements in the order of
memory: the first moment, and the root of the second (its range is half as many octaves). They are rounded up or down by
random bits that are a hash of `seed`, the number of steps and the element's place in the list.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import native, scan
from .host import operators

BLOCK = 256             # elements that share a scale
E4M3_MAX = 448.0
E4M3_LEAST = 2.0**-9    # smallest value above zero
LEAST_SCALED = 2.0**-100   # blocks whose largest magnitude is below are taken for zeros
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

# one tensor of a list, see PsgdAdamTensor
ITEM = np.dtype([("p", "u8"), ("g", "u8"), ("m", "u8"), ("v", "u8"), ("m_scale", "u8"), ("v_scale", "u8"), ("step", "u8"), ("n", "i8"),
                 ("block0", "u4"), ("chunk_end", "u4")])


def blocks_of(numel: int) -> int:
    return -(-numel // BLOCK)


def state_names(bits: int):
    """Names of a parameter's moments in the optimizer's state."""
    return ("exp_avg", "exp_avg_sq") if bits == 32 else ("exp_avg", "exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale")


def new_state(p: torch.Tensor, bits: int) -> dict:
    """Moments of a parameter that has made no step."""
    dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
    state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
    for name in state_names(bits):
        if name.endswith("_scale"):
            state[name] = torch.zeros(blocks_of(p.numel()), dtype=torch.float32, device=p.device)
        else:
            state[name] = torch.zeros_like(p, dtype=dtype, memory_format=torch.preserve_format)
    return state


def in_one_piece(t: torch.Tensor) -> bool:
    """Does the tensor fill its stretch of memory, each element once, in whatever order of dimensions?"""
    if t.is_contiguous() or t.numel() == 0:
        return True
    expected = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expected:
            return False
        expected *= n
    return True


def laid_like(t: torch.Tensor, p: torch.Tensor) -> bool:
    return t.shape == p.shape and all(n == 1 or a == b for n, a, b in zip(p.shape, t.stride(), p.stride()))


def lay_like(state: dict, p: torch.Tensor) -> None:
    """Moments in 32 bits in the order of their parameter's dimensions, which may have changed (a model that became channels_last, a state
    saved before it did). Recorded graphs keep what they refer to."""
    strides = p.stride()
    for name in state_names(32):
        t = state.get(name)
        if t is not None and t.stride() != strides and t.shape == p.shape and not laid_like(t, p) and not (p.is_cuda and torch.cuda.is_current_stream_capturing()):
            state[name] = torch.empty_like(p, dtype=t.dtype, memory_format=torch.preserve_format).copy_(t)


def check_lists(params, grads, moments, steps, bits: int) -> None:
    names = state_names(bits)
    for i, p in enumerate(params):
        if p.dtype not in DTYPES:
            raise TypeError(f"AdamW: parameter {i} is {p.dtype}; float32, bfloat16 and float16 are supported")
        if not in_one_piece(p):
            raise ValueError(f"AdamW: parameter {i} (shape {tuple(p.shape)}, strides {p.stride()}) does not lie in one piece")
        g = grads[i]
        if g.layout != torch.strided:
            raise TypeError(f"AdamW: the gradient of parameter {i} is {g.layout}; dense gradients are supported")
        if g.dtype != p.dtype or g.device != p.device or not laid_like(g, p):
            raise ValueError(f"AdamW: the gradient of parameter {i} has another type, device or layout than the parameter")
        for name, t in zip(names, (m[i] for m in moments)):
            scale = name.endswith("_scale")
            dtype = torch.float32 if bits == 32 or scale else torch.float8_e4m3fn
            fits = t.numel() == blocks_of(p.numel()) and t.is_contiguous() if scale else laid_like(t, p)
            if t.dtype != dtype or t.device != p.device or not fits:
                raise ValueError(f"AdamW: {name} of parameter {i} is {t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}; expected {dtype} for "
                                 f"{tuple(p.shape)}, strides {p.stride()}, on {p.device}")
        if steps[i].dtype != torch.float32 or steps[i].numel() != 1 or steps[i].device != p.device:
            raise ValueError(f"AdamW: the number of steps of parameter {i} must be one float32 on {p.device}")


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], moments: Sequence[Sequence[torch.Tensor]], steps: Sequence[torch.Tensor],
               *, bits: int, lr, beta1: float, beta2: float, eps: float, weight_decay: float, seed: int = 0,
               first_blocks: Optional[Sequence[int]] = None, ticket: Optional[torch.Tensor] = None) -> None:
    """One step for all tensors of one type and device, in place. `moments`: lists in the order of `state_names(bits)`.
    `first_blocks[i]`: where tensor i begins in the stream of random numbers, in blocks of 256 (default: one behind
    another). `ticket`: an int32 tensor of the device that is zero and that no other launch uses at the same time. Gradients
    have their parameter's type and layout."""
    if not params:
        return
    check_lists(params, grads, moments, steps, bits)
    if first_blocks is None:
        first_blocks = np.concatenate([[0], np.cumsum([blocks_of(p.numel()) for p in params])[:-1]]).tolist()
    device = params[0].device
    if any(p.device != device or p.dtype != params[0].dtype for p in params):
        raise ValueError("adamw_step: a list holds tensors of one type and one device")
    if device.type == "cuda" and native.use_for_cuda():
        items = np.zeros(len(params), dtype=ITEM)
        for field, tensors in zip(("p", "g", "step", "m", "v", "m_scale", "v_scale"), (params, grads, steps, *moments)):
            items[field] = np.frombuffer(scan.addresses(list(tensors)), dtype=np.uint64)
        items["n"] = [p.numel() for p in params]
        items["block0"] = first_blocks
        if ticket is None:
            raise ValueError("adamw_step: a ticket is needed on CUDA")
        launch(items.tobytes(), len(params), device, DTYPES[params[0].dtype], bits=bits, lr=lr, beta1=beta1, beta2=beta2, eps=eps,
               weight_decay=weight_decay, seed=seed, ticket=ticket)
        torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])   # (torch operations do so themselves)
        return
    lr = float(lr)
    for i, p in enumerate(params):
        _step_torch(p, grads[i], [m[i] for m in moments], steps[i], bits, lr, beta1, beta2, eps, weight_decay, seed, int(first_blocks[i]))


def launch(items: bytes, count: int, device: torch.device, dtype: int, *, bits, lr, beta1, beta2, eps, weight_decay, seed, ticket) -> None:
    """The native step for a list of `ITEM`s."""
    lr_at = None
    if isinstance(lr, torch.Tensor):
        if lr.is_cuda:
            if lr.device != device or lr.dtype != torch.float32 or lr.numel() != 1:
                raise ValueError(f"AdamW: a learning rate on the GPU must be one float32 on {device}")
            lr_at, lr = lr, 0.0
        else:
            lr = float(lr)
    call = (items, count, dtype, bits, lr, 0 if lr_at is None else lr_at.data_ptr(), beta1, beta2, math.log(beta1) if beta1 > 0 else -math.inf,
            math.log(beta2) if beta2 > 0 else -math.inf, eps, weight_decay, seed, ticket.data_ptr())
    if operators is not None:
        code = operators.adamw_step(*call[:2], device.index, *call[2:])
    else:
        with native.on_device(device) as stream:
            code = native.lib().psgd_adamw_step(*call, stream)
    if code:
        native.check(code, "psgd_adamw_step")


# ---- the step in torch operations --------------------------------------------------------------
def _mix(x: torch.Tensor) -> torch.Tensor:
    """The finalizer of MurmurHash3 (32 bits) in int64 tensors."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_words(blocks: int, first_block: int, step: int, seed: int, device=None) -> torch.Tensor:
    """32 random bits for each element of `blocks` blocks, [blocks, 256] int64."""
    key = _mix(torch.tensor(seed & 0xFFFFFFFF, device=device) ^ _mix(torch.tensor(step, device=device)))
    block = _mix(key ^ ((torch.arange(blocks, device=device) + first_block) & 0xFFFFFFFF))
    return _mix((block[:, None] + torch.arange(BLOCK, device=device)) & 0xFFFFFFFF)


def quantize(x: torch.Tensor, random16: torch.Tensor, least: bool):
    """`x` [blocks, 256] float32 as e4m3 codes and a scale per block; `random16` decides which way a value is rounded. With
    `least`, what is not zero stays above zero."""
    most = x.abs().amax(1, keepdim=True)
    zero = most < LEAST_SCALED
    y = x.abs() * torch.where(zero, torch.zeros_like(most), most.reciprocal() * E4M3_MAX)
    low = y < 2.0**-6
    t = torch.where(low, y + 2.0**-6, y)   # the steps below 2^-6 are those right above it
    t = ((t.view(torch.int32) + (random16 * 16 + 8).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    t = torch.where(low, t - 2.0**-6, t).clamp_max(E4M3_MAX)
    if least:
        t = torch.where(y > 0, t.clamp_min(E4M3_LEAST), t)
    return torch.copysign(t, x).to(torch.float8_e4m3fn), torch.where(zero, torch.zeros_like(most), most * (1.0 / E4M3_MAX))[:, 0]


def _in_memory_order(t: torch.Tensor) -> torch.Tensor:
    return t.as_strided((t.numel(),), (1,))


def _in_blocks(flat: torch.Tensor) -> torch.Tensor:
    n = flat.numel()
    out = flat.new_zeros(blocks_of(n) * BLOCK)
    out[:n] = flat
    return out.view(-1, BLOCK)


@torch.no_grad()
def _step_torch(p, g, moments: List[torch.Tensor], step, bits, lr, beta1, beta2, eps, weight_decay, seed, first_block) -> None:
    step += 1.0
    t = float(step)
    if p.numel() == 0:
        return
    flat_p, flat_g = _in_memory_order(p.detach()), _in_memory_order(g.detach()).float()
    if bits == 32:
        m, v = _in_memory_order(moments[0]), _in_memory_order(moments[1])
    else:
        m8, r8 = _in_memory_order(moments[0]), _in_memory_order(moments[1])
        m = (_in_blocks(m8.float()) * moments[2][:, None]).view(-1)[: p.numel()]
        v = (_in_blocks(r8.float()) * moments[3][:, None]).view(-1)[: p.numel()].square()
    m = m * beta1 + flat_g * (1 - beta1)
    v = v * beta2 + flat_g * flat_g * (1 - beta2)
    root = v.sqrt()
    update = m / (root / math.sqrt(1 - beta2**t) + eps)
    flat_p.copy_(flat_p.float() * (1 - lr * weight_decay) - update * (lr / (1 - beta1**t)))
    if bits == 32:
        _in_memory_order(moments[0]).copy_(m)
        _in_memory_order(moments[1]).copy_(v)
        return
    words = random_words(blocks_of(p.numel()), first_block, int(t), seed, p.device)
    for codes, scale, x, random, least in ((m8, moments[2], m, words & 0xFFFF, False), (r8, moments[3], root, words >> 16, True)):
        new, new_scale = quantize(_in_blocks(x), random, least)
        codes.copy_(new.view(-1)[: p.numel()])
        scale.copy_(new_scale)
