"""Launchers of the 4-bit linear layers (csrc/int4.hip; the reference's layers
are nn.Linear in the model's dtype)."""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .common import call_on, require_device

GROUPS = (32, 64, 128)
MAX_ROWS = 64      # rows of one launch; more go through the widened weights
MAX_MATRICES = 4


def group_size(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None) -> int:
    """The group size that the tensors' shapes say, checked."""
    if packed.dim() != 4 or tuple(packed.shape[2:]) != (64, 16) or packed.dtype != torch.uint8:
        raise ValueError(f"int4: packed must be (tiles, blocks, 64, 16) uint8, got "
                         f"{tuple(packed.shape)} {packed.dtype}")
    nt, kb = packed.shape[:2]
    if nt == 0 or kb == 0:
        raise ValueError("int4: empty weight")
    if scales.dim() != 3 or scales.shape[0] != nt or scales.shape[2] != 16:
        raise ValueError(f"int4: scales must be ({nt}, groups, 16), got {tuple(scales.shape)}")
    G = 128 * kb // max(scales.shape[1], 1)
    if G not in GROUPS or G * scales.shape[1] != 128 * kb:
        raise ValueError(f"int4: {scales.shape[1]} groups over {128 * kb} columns are groups of "
                         f"none of {GROUPS}")
    if zeros is not None and zeros.shape != scales.shape:
        raise ValueError(f"int4: zeros must be {tuple(scales.shape)}, got {tuple(zeros.shape)}")
    for t, name in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and t.dtype != torch.bfloat16:
            raise TypeError(f"int4: {name} must be bfloat16, got {t.dtype}")
    for t, name in ((packed, "packed"), (scales, "scales"), (zeros, "zeros")):
        if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
            raise ValueError(f"int4: {name} must be contiguous on a 16-byte boundary")
    return G


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x (..., K) as (M, K) rows that the kernel reads: 16-byte aligned, the row
    length padded with zeros to a multiple of 8."""
    x = x.reshape(-1, K)
    if K % 8:
        return torch.nn.functional.pad(x, (0, 8 - K % 8))
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def int4_linear_multi(x, weights, biases, sizes, G, xscale=None):
    """x (..., K) bf16 of 1..64 rows; weights: [(packed, scales, zeros or None)],
    1..4 of them with one group size; biases: [(N_i,) bf16 or None]; sizes: [N_i]
    -> [(..., N_i)], one launch."""
    require_device(x, xscale, *[t for w in weights for t in w], *biases)
    K, n = x.shape[-1], len(weights)
    xr = _rows(x, K)
    xs = None if xscale is None else _rows(xscale, K)
    M = xr.shape[0]
    ys = [torch.empty(*x.shape[:-1], N, dtype=torch.bfloat16, device=x.device) for N in sizes]
    bs = [None if b is None else b.contiguous() for b in biases]
    arr = ctypes.c_void_p * n
    call_on(x, "sa_int4_linear_bf16", _lib.ptr(xr), _lib.ptr(xs), M, K, xr.shape[1], G, n,
            arr(*[w[0].data_ptr() for w in weights]), arr(*[w[1].data_ptr() for w in weights]),
            None if weights[0][2] is None else arr(*[w[2].data_ptr() for w in weights]),
            arr(*[_lib.ptr(b) for b in bs]), (ctypes.c_int * n)(*sizes),
            arr(*[y.data_ptr() for y in ys]), _lib.stream_of(x))
    return ys


def dequantize_int4(packed, scales, zeros, N, K, G):
    """(N, K) bf16: what the packed weights stand for, rounded."""
    require_device(packed, scales, zeros)
    out = torch.empty(N, K, dtype=torch.bfloat16, device=packed.device)
    call_on(packed, "sa_int4_dequant_bf16", _lib.ptr(packed), _lib.ptr(scales), _lib.ptr(zeros), N,
            K, G, _lib.ptr(out), _lib.stream_of(packed))
    return out
