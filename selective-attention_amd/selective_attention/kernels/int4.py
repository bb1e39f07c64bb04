"""Launchers of the 4-bit linear layers (csrc/int4.hip; the reference's layers
are nn.Linear in the model's dtype)."""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .common import call_on, require_device, require_one_device

GROUPS = (32, 64, 128)
MAX_ROWS = 64      # rows of one launch; more go through the widened weights
MAX_MATRICES = 4
MAX_STRIDE = 1 << 23


def group_size(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None) -> int:
    """The group size that the tensors' shapes say, checked."""
    shape, f = packed.shape, scales.shape
    if len(shape) != 4 or shape[2] != 64 or shape[3] != 16 or packed.dtype != torch.uint8:
        raise ValueError(f"int4: packed must be (tiles, blocks, 64, 16) uint8, got "
                         f"{tuple(shape)} {packed.dtype}")
    nt, kb = shape[0], shape[1]
    if nt == 0 or kb == 0:
        raise ValueError("int4: empty weight")
    if len(f) != 3 or f[0] != nt or f[2] != 16:
        raise ValueError(f"int4: scales must be ({nt}, groups, 16), got {tuple(f)}")
    G = 128 * kb // max(f[1], 1)
    if G not in GROUPS or G * f[1] != 128 * kb:
        raise ValueError(f"int4: {f[1]} groups over {128 * kb} columns are groups of none of {GROUPS}")
    if zeros is not None and zeros.shape != f:
        raise ValueError(f"int4: zeros must be {tuple(f)}, got {tuple(zeros.shape)}")
    for t, name in ((packed, "packed"), (scales, "scales"), (zeros, "zeros")):
        if t is not None:
            if t is not packed and t.dtype != torch.bfloat16:
                raise TypeError(f"int4: {name} must be bfloat16, got {t.dtype}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"int4: {name} must be contiguous on a 16-byte boundary")
    return G


def _rows(x: torch.Tensor, K: int) -> torch.Tensor:
    """x (..., K) as (M, K) rows of one stride; slices of longer rows as they lie."""
    if x.dim() != 2:
        x = x.reshape(-1, K)
    return x if x.is_contiguous() or _strided(x, K) else x.contiguous()


def _strided(x: torch.Tensor, K: int) -> bool:
    return x.stride(1) == 1 and K <= x.stride(0) <= MAX_STRIDE


def int4_linear_multi(x, weights, biases, sizes, G, xscale=None):
    """x (..., K) bf16 of 1..64 rows; weights: [(packed, scales, zeros or None)],
    1..4 of them with one group size; biases: [(N_i,) bf16 or None]; sizes: [N_i]
    -> [(..., N_i)], one launch."""
    for w in weights:
        require_one_device(x, *w)
    require_one_device(x, xscale, *biases)
    K, n = x.shape[-1], len(weights)
    xr = _rows(x, K)
    xs = None if xscale is None else _rows(xscale, K)
    M = xr.shape[0]
    if M == 1:
        ld = K
    else:
        ld = xr.stride(0)
        if xs is not None and xs.stride(0) != ld:
            xr, xs, ld = xr.contiguous(), xs.contiguous(), K
    ys, words, kept = [], [], []
    for (packed, scales, zeros), b, N in zip(weights, biases, sizes):
        y = torch.empty((*x.shape[:-1], N), dtype=torch.bfloat16, device=x.device)
        if b is not None and not b.is_contiguous():
            b = b.contiguous()
            kept.append(b)
        words += (packed.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
                  0 if b is None else b.data_ptr(), y.data_ptr(), N)
        ys.append(y)
    call_on(x, "sa_int4_linear_bf16", xr.data_ptr(), _lib.ptr(xs), M, K, ld, G, n,
            (ctypes.c_int64 * (6 * n))(*words), _lib.stream_of(x))
    return ys


def dequantize_int4(packed, scales, zeros, N, K, G):
    """(N, K) bf16: what the packed weights stand for, rounded."""
    require_device(packed, scales, zeros)
    out = torch.empty(N, K, dtype=torch.bfloat16, device=packed.device)
    call_on(packed, "sa_int4_dequant_bf16", _lib.ptr(packed), _lib.ptr(scales), _lib.ptr(zeros), N,
            K, G, _lib.ptr(out), _lib.stream_of(packed))
    return out
