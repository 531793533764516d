"""powersgd_b200 — PowerSGD low-rank gradient compression, built for B200 (sm_100a).

Public surface (same names as the reference's `powersgd` package, powersgd/__init__.py:3-7):
`PowerSGD`, `Config`, `AllReduce`, `Aggregator`, `optimizer_step`; besides them `AdamW`, an optimizer to give it, and `clip_grad_norm`, which
scales gradients that are too large together, with `grad_norm`.
"""
from .aggregators import Aggregator, AllReduce, BasicConfig, BasicPowerSGD, Config, PowerSGD
from .ops.grad_norm import clip_grad_norm, grad_norm
from .optim import AdamW, optimizer_step
from .utils import params_in_optimizer

__version__ = "0.1.0"

__all__ = [
    "AdamW",
    "Aggregator",
    "AllReduce",
    "BasicConfig",
    "BasicPowerSGD",
    "Config",
    "PowerSGD",
    "clip_grad_norm",
    "grad_norm",
    "optimizer_step",
    "params_in_optimizer",
]
