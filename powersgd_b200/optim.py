"""Optimizer glue (powersgd/__init__.py:7-25) and AdamW on the native kernels."""
from __future__ import annotations

import math
from typing import Iterable, Tuple, Union

import torch

from .aggregators import Aggregator
from .ops import adamw as _adamw
from .ops import native, scan
from .ops.recording import keep_with_graph, outside_capture
from .utils import params_in_optimizer


def optimizer_step(optimizer: torch.optim.Optimizer, aggregator: Aggregator) -> None:
    """Aggregate the gradients over workers, step the optimizer with the aggregate, and
    leave each parameter's `.grad` holding its local residual.

    The next `backward()` accumulates onto that residual, which is how error feedback is
    realised — so the caller must NOT call `optimizer.zero_grad()` between steps.

    With the native back end and a plain `torch.optim.SGD`, aggregation, error feedback and
    the parameter update run as one fused sequence of kernels (`PowerSGD.fused_step`).
    """
    fused = getattr(aggregator, "supports_fused_step", None)
    if fused is not None and fused(optimizer):
        aggregator.fused_step(optimizer)
        return
    params = params_in_optimizer(optimizer)
    residuals = [p.grad.data for p in params]
    averaged = aggregator.aggregate(residuals)  # `residuals` now hold what was not sent
    for p, g in zip(params, averaged):
        p.grad = g
    optimizer.step()
    for p, g in zip(params, residuals):
        p.grad = g


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay: all tensors of a parameter group in one launch.

        optimizer = AdamW(model.parameters(), lr=3e-4, weight_decay=0.1, state_bits=8)
        optimizer_step(optimizer, powersgd)        # or optimizer.step() with gradients of one's own

    `state_bits=32`: float32 moments under the names of `torch.optim.AdamW` (`exp_avg`, `exp_avg_sq`, `step`).
    `state_bits=8`: two bytes per parameter instead of eight; `exp_avg` and `exp_avg_sq_root` are e4m3 tensors with a
    scale per 256 elements (`ops/adamw.py`), rounded by random bits that follow from `seed` and the number of steps,
    so that a run can be repeated. A gradient that is infinite or no number spoils the moments of its 256 elements.

    Parameters are float32, bfloat16 or float16 tensors that lie in one piece (any order of dimensions), each in memory of its own. The
    arithmetic is float32. A step may be recorded in a CUDA graph: the number of steps is counted on the device; a learning rate
    that is to change between replays is given as a float32 tensor on the GPU. The optimizer outlives the graph.
    On the CPU the same step runs in torch operations.
    """

    def __init__(self, params: Iterable, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0):
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, seed=seed))
        self._own()

    def _own(self) -> None:
        self._tickets = {}   # device -> counter of finished blocks, zero between launches
        self._held = {}      # what recorded graphs refer to

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self._own()

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check(group)
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> None:
        lr = group["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.numel() != 1:
                raise ValueError("AdamW: a learning rate that is a tensor must have one element")
        elif not (math.isfinite(lr) and lr >= 0):
            raise ValueError(f"AdamW: learning rate {lr}")
        if not all(0.0 <= b < 1.0 for b in group["betas"]) or len(group["betas"]) != 2:
            raise ValueError(f"AdamW: betas {group['betas']}")
        for name in ("eps", "weight_decay"):
            if not (math.isfinite(group[name]) and group[name] >= 0):
                raise ValueError(f"AdamW: {name} {group[name]}")
        if group["state_bits"] not in (8, 32):
            raise ValueError(f"AdamW: state_bits {group['state_bits']}; moments are held in 32 bits or in 8")
        if not 0 <= group["seed"] < 2**32:
            raise ValueError(f"AdamW: seed {group['seed']}; 0 to 2^32 - 1")
        if len({id(p) for p in group["params"]}) != len(group["params"]):
            raise ValueError("AdamW: a parameter is listed twice")
        for i, p in enumerate(group["params"]):
            if p.dtype not in _adamw.DTYPES:
                raise TypeError(f"AdamW: parameter {i} is {p.dtype}; float32, bfloat16 and float16 are supported")
        # one launch steps all of a group at once: none may lie in another's memory
        taken = {}
        for i, p in enumerate(group["params"]):
            if p.numel() and p.device.type in ("cpu", "cuda") and _adamw.in_one_piece(p):
                taken.setdefault(p.device, []).append((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size(), i))
        for pieces in taken.values():
            pieces.sort()
            for (_, end, i), (start, _, j) in zip(pieces, pieces[1:]):
                if start < end:
                    raise ValueError(f"AdamW: parameters {min(i, j)} and {max(i, j)} share memory")

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first_block = 0    # of each parameter in the stream of random numbers
        for group in self.param_groups:
            first_block = self._step_group(group, first_block)
        return loss

    def _step_group(self, group: dict, first_block: int) -> int:
        """One step of a group; its parameters begin at `first_block` of the stream of random numbers. Returns where the next begin."""
        bits, names = group["state_bits"], _adamw.state_names(group["state_bits"])
        known = scan.adam_items(group["params"], self.state, ("step", *names), first_block)
        if known is not None:   # one type, one GPU, everything as the kernel takes it
            items, count, device, dtype, end = known
            if count and native.use_for_cuda():
                device = torch.device("cuda", device)
                ticket = self._ticket(device)
                if torch.cuda.is_current_stream_capturing():
                    self._keep(group, group["params"], [self.state[p] for p in group["params"] if p.grad is not None], ticket)
                beta1, beta2 = group["betas"]
                _adamw.launch(items, count, device, dtype, bits=bits, lr=group["lr"], beta1=beta1, beta2=beta2, eps=group["eps"],
                              weight_decay=group["weight_decay"], seed=group["seed"], ticket=ticket)
                return end
        lists, at = {}, first_block
        for p in group["params"]:
            if p.grad is not None:
                state = self.state[p]
                if not state:
                    with outside_capture(p.device) if p.is_cuda else _nothing():
                        state.update(_adamw.new_state(p, bits))
                elif bits == 32:
                    _adamw.lay_like(state, p)
                g = p.grad
                if g.layout == torch.strided:
                    g = native.in_memory(g)
                if g.layout == torch.strided and g.dtype == p.dtype and not _adamw.laid_like(g, p):
                    g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
                lists.setdefault((p.device, p.dtype), []).append((p, g, state, at))
            at += _adamw.blocks_of(p.numel())
        for (device, _), entries in lists.items():
            params, grads, states, blocks = zip(*entries)
            ticket = None
            if device.type == "cuda" and native.use_for_cuda():
                ticket = self._ticket(device)
                if torch.cuda.is_current_stream_capturing():
                    self._keep(group, params, states, ticket)
            missing = [name for name in ("step", *names) if any(name not in s for s in states)]
            if missing:
                raise ValueError(f"AdamW: the state has no {missing[0]}; it belongs to moments of another number of bits than {bits}")
            _adamw.adamw_step(params, grads, [[s[name] for s in states] for name in names], [s["step"] for s in states], bits=bits, lr=group["lr"],
                              beta1=group["betas"][0], beta2=group["betas"][1], eps=group["eps"], weight_decay=group["weight_decay"],
                              seed=group["seed"], first_blocks=blocks, ticket=ticket)
        return at

    def _ticket(self, device: torch.device) -> torch.Tensor:
        ticket = self._tickets.get(device)
        if ticket is None:
            with outside_capture(device):
                ticket = self._tickets[device] = torch.zeros(1, dtype=torch.int32, device=device)
        return ticket

    def _keep(self, group: dict, params, states, ticket: torch.Tensor) -> None:
        """What the graph that is being recorded refers to stays, whatever is loaded or set later."""
        keep_with_graph(self._held, *params, *[t for s in states for t in s.values()], ticket, group["lr"])

    def load_state_dict(self, state_dict: dict) -> None:
        """As in `torch.optim`, except that moments and numbers of steps keep their own types. What is refused changes nothing. Moments in 32 bits
        take the order of dimensions that their parameter has; those in 8 bits share scales in the order that they were saved in and keep it."""
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for group, own in zip(state_dict["param_groups"], self.param_groups):
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("AdamW: a state of torch.optim.AdamW with amsgrad or maximize does not carry over")
            self._check({**self.defaults, **group, "params": own["params"]})
        super().load_state_dict(state_dict)
        for i, p in zip(saved, params_in_optimizer(self)):
            for name, value in state_dict["state"].get(i, {}).items():
                if name == "step":      # (a number in old states)
                    self.state[p][name] = torch.as_tensor(value, dtype=torch.float32).detach().reshape(()).to(p.device, copy=True)
                elif isinstance(value, torch.Tensor):   # (torch.optim has moments of the parameter's type)
                    dtype = torch.float32 if name in ("exp_avg", "exp_avg_sq") and value.dtype in (torch.bfloat16, torch.float16) else value.dtype
                    self.state[p][name] = value.to(p.device, dtype, copy=True)
        for group in self.param_groups:
            for name, value in self.defaults.items():   # what a state of torch.optim.AdamW does not have
                group.setdefault(name, value)


class _nothing:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False
