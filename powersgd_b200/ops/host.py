"""Calls of the language-model operators without the interpreter in between: csrc/host/operators.cpp, where it is built."""
from __future__ import annotations

import ctypes
import importlib.util
import os

from ..csrc.build import operators_lib, scan_target
from . import native

ENTRY_POINTS = ("psgd_last_error", "psgd_token_logprob", "psgd_token_logprob_grad", "psgd_attention", "psgd_attention_backward", "psgd_adamw_step",
                "psgd_attention_plan_ints", "psgd_grad_norm", "psgd_grad_norm_parts", "psgd_rotate", "psgd_rotate_grad", "psgd_rotate_parts")


def _load():
    """The extension, bound to the native library; None where either is missing or was built for another PyTorch or Python."""
    path = operators_lib()
    if not os.path.exists(path) or not native.available():
        return None
    try:
        spec = importlib.util.spec_from_file_location("_operators", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except ImportError:   # symbols or libraries that are not there
        return None
    if getattr(module, "target", None) != scan_target() or getattr(module, "entry_points", 0) != len(ENTRY_POINTS):
        return None   # of another PyTorch, or of an earlier state of the sources
    module.bind(*[ctypes.cast(getattr(native.lib(), name), ctypes.c_void_p).value for name in ENTRY_POINTS])
    return module


operators = _load()
