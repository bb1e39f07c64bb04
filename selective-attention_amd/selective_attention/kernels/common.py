"""Host-side helpers shared by the kernel launchers."""
from __future__ import annotations

import torch

from .. import _lib

_ACT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def act_dtype_code(dtype: torch.dtype) -> int:
    """Kernel dtype code for activations (u, B, C, delta_raw, q/k/v)."""
    try:
        return _ACT_DTYPES[dtype]
    except KeyError:
        raise TypeError(f"unsupported activation dtype {dtype}; expected float32 or bfloat16")


def as_dtype(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    if t is None or t.dtype == dtype:
        return t
    return t.to(dtype)


def require_device(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError(
                f"tensor on {t.device}: the HIP kernels need device tensors (no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"tensors on different devices: {dev} vs {t.device}")
    return dev


def require_one_device(*tensors: torch.Tensor | None) -> None:
    """require_device for the decode steps' calls: without the device objects,
    which for a dozen tensors take longer than a launch."""
    dev = -2
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != dev:
                if d < 0 or dev != -2:
                    require_device(*tensors)    # says what is wrong
                dev = d


def call_on(t: torch.Tensor, name: str, *args) -> None:
    """_lib.call with t's device current (its stream belongs to that device)."""
    if torch._C._cuda_getDevice() == t.device.index:
        return _lib.call(name, *args)
    with torch.cuda.device(t.device):
        return _lib.call(name, *args)


def limits(delta_limit) -> tuple[float, float]:
    lo, hi = float(delta_limit[0]), float(delta_limit[1])
    return lo, hi


def needs_torch_ops(*ts: torch.Tensor) -> bool:
    """Whether something has to see torch's own ops on ts, which a kernel launch
    hides or cannot serve: forward-mode AD, a dispatch mode, tracing, a functorch
    transform, or a legacy batched tensor (is_grads_batched)."""
    return (torch._C._are_functorch_transforms_active()
            or torch.autograd.forward_ad._current_level >= 0
            or torch._C._len_torch_dispatch_stack() > 0
            or torch.compiler.is_compiling() or torch.jit.is_tracing()
            # (on the tensors too: a GPU backward runs on a thread of its own)
            or any(torch._C._functorch.is_functorch_wrapped_tensor(t)
                   or torch._C._functorch.is_legacy_batchedtensor(t) for t in ts))


def in_forward_mode() -> bool:
    """Whether a dual level of forward-mode AD is open: a kernel launch would drop
    the tangents without a word.  (Wrapped and batched tensors refuse the launch
    by themselves, having no address.)"""
    return torch.autograd.forward_ad._current_level >= 0
