"""Linear layers with 4-bit weights and group scales.

    y = x W^T + bias,   W[n, k] = scales[n, k // group] (code[n, k] - zero[n, k // group])

with codes 0..15, zero = 8 where no zero points are given, and groups of 32, 64
or 128 columns.  pack_int4 and quantize_int4 lay a weight out once; int4_linear
takes it as it lies.  Up to 64 rows (decode steps) one kernel reads the codes
and keeps the group's factors in fp32: W is exact, and the output's rounding the
only one to fewer bits.  More rows, and rows that take a gradient, go through the
weights widened to bfloat16 and a plain matrix product: every W[n, k] is rounded
there, by up to 2^-8 of it, so that a row's result moves by up to 2^-8 sum_k
|x_k W[n, k]| where a 65th row comes to stand beside it.

x is taken to be finite.  A row with an infinity gives NaN in every output up to 64
rows (the kernel takes the difference of two sums of x), infinities or NaN above;
the rows beside it stand.

New ops (the reference's layers are nn.Linear in the model's dtype,
modules/feed_forward.py:4-11).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels import int4 as _k
from ..kernels.common import in_forward_mode
from ..kernels.int4 import MAX_MATRICES, MAX_ROWS
from ..utils import check_ndim, check_shape


def _pad(t: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    return F.pad(t, (0, -t.shape[1] % cols, 0, -t.shape[0] % rows))


def pack_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
              group_size: int = 128):
    """
    Args:
        codes: (out_features, in_features) integers 0..15
        scales: (out_features, ceil(in_features / group_size)); kept as bfloat16
        zeros: as scales, the codes that stand for 0, or None (8 everywhere)
    Returns:
        (packed, scales, zeros) as int4_linear takes them: packed (ceil(N / 16),
        ceil(K / 128), 64, 16) uint8 in the kernel's order, scales and zeros
        (ceil(N / 16), groups, 16) bfloat16
    """
    check_ndim(codes, 2, name="codes")
    N, K = codes.shape
    if group_size not in _k.GROUPS:
        raise ValueError(f"group_size {group_size} must be one of {_k.GROUPS}")
    if N == 0 or K == 0:
        raise ValueError("pack_int4: empty weight")
    if codes.is_floating_point() or codes.dtype == torch.bool:
        raise TypeError(f"pack_int4: codes must be integers, got {codes.dtype}")
    if bool((codes < 0).any() | (codes > 15).any()):
        raise ValueError("pack_int4: codes must be 0..15")
    groups = (K + group_size - 1) // group_size
    check_shape(scales, (N, groups), name="scales")
    check_shape(zeros, (N, groups), name="zeros", optional=True)
    c = _pad(codes.to(torch.uint8), 16, 128)
    nt, kb = c.shape[0] // 16, c.shape[1] // 128
    # (tile, row c, block, j, g, i, half) -> (tile, block, g, c, j, i, half)
    c = c.view(nt, 16, kb, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
    packed = (c[..., 0] | (c[..., 1] << 4)).reshape(nt, kb, 64, 16).contiguous()
    each = 128 // group_size

    def lay(t):
        t = _pad(t.to(torch.bfloat16), 16, each)
        return F.pad(t, (0, kb * each - t.shape[1])).view(nt, 16, kb * each).transpose(1, 2).contiguous()
    return packed, lay(scales), None if zeros is None else lay(zeros)


def quantize_int4(weight: torch.Tensor, group_size: int = 128, symmetric: bool = True):
    """weight (out_features, in_features) -> (packed, scales, zeros or None), each
    group rounded to the nearest code: symmetric, scale = max|w| / 7 around
    code 8; else scale = (max - min) / 15 over the group's range with 0 in it and
    zero points.  The codes are chosen for the scale as bfloat16 keeps it; a group
    of zeros has the scale 0 and so adds exactly nothing."""
    check_ndim(weight, 2, name="weight")
    if group_size not in _k.GROUPS:
        raise ValueError(f"group_size {group_size} must be one of {_k.GROUPS}")
    N, K = weight.shape
    if N == 0 or K == 0:
        raise ValueError("quantize_int4: empty weight")
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("quantize_int4: the weight holds infinities or NaN")
    w = F.pad(weight.detach().float(), (0, -K % group_size)).view(N, -1, group_size)
    if symmetric:
        s, zero = w.abs().amax(2) / 7.0, None
    else:
        lo, hi = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
        s = (hi - lo) / 15.0
    s = s.to(torch.bfloat16)
    by = torch.where(s > 0, s, torch.ones_like(s)).float()
    if not symmetric:
        zero = torch.round(-lo / by).clamp(0, 15)
    q = torch.round(w / by[..., None]) + (8.0 if zero is None else zero[..., None])
    codes = q.clamp(0, 15).to(torch.uint8).reshape(N, -1)[:, :K]
    return pack_int4(codes, s, zero, group_size)


def dequantize_int4(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                    out_features: int | None = None, in_features: int | None = None) -> torch.Tensor:
    """(out_features, in_features) bfloat16: the weights that the codes stand for,
    rounded; without sizes, with the padding."""
    G = _k.group_size(packed, scales, zeros)
    N, K = _sizes(packed, out_features, in_features)
    return _k.dequantize_int4(packed, scales, zeros, N, K, G)


def _sizes(packed, N, K):
    nt, kb = packed.shape[:2]
    N, K = 16 * nt if N is None else int(N), 128 * kb if K is None else int(K)
    if (N + 15) // 16 != nt or (K + 127) // 128 != kb:
        raise ValueError(f"int4: packed {tuple(packed.shape)} holds {16 * nt} rows and {128 * kb} "
                         f"columns (padded), not {N} and {K}")
    return N, K


def int4_linear_multi(x: torch.Tensor, weights, biases, sizes,
                      xscale: torch.Tensor | None = None) -> list:
    """[x W_i^T + bias_i] of 1..4 weights (packed, scales, zeros or None) with one
    group size, all with or all without zero points; sizes: their out_features.
    x (..., in_features) bfloat16; with xscale (x's shape) the input is
    bfloat16(x * xscale).  Returns bfloat16 (..., out_features) tensors."""
    n = len(weights)
    if not 1 <= n <= MAX_MATRICES or len(biases) != n or len(sizes) != n:
        raise ValueError(f"int4_linear_multi: 1..{MAX_MATRICES} weights with as many biases and sizes, "
                         f"got {n}, {len(biases)}, {len(sizes)}")
    if x.dim() == 0:
        raise ValueError("int4_linear: x must have at least one dimension")
    if x.dtype != torch.bfloat16:
        raise TypeError(f"int4_linear: x must be bfloat16, got {x.dtype}")
    if xscale is not None and (xscale.shape != x.shape or xscale.dtype != torch.bfloat16):
        raise ValueError("int4_linear: xscale must be bfloat16 of x's shape")
    K = x.shape[-1]
    if K == 0:
        raise ValueError("int4_linear: x has no features")
    G, zeros = 0, weights[0][2] is None
    for w, b, N in zip(weights, biases, sizes):
        g = _k.group_size(*w)
        if (G and g != G) or (w[2] is None) != zeros:
            raise ValueError("int4_linear_multi: the weights differ in group size or zero points")
        G = g
        _sizes(w[0], N, K)
        if b is not None:
            check_shape(b, (N,), name="bias")
            if b.dtype != torch.bfloat16:
                raise TypeError(f"int4_linear: bias must be bfloat16, got {b.dtype}")
    grad = torch.is_grad_enabled() and (
        x.requires_grad or (xscale is not None and xscale.requires_grad)
        or any(b is not None and b.requires_grad for b in biases)) or in_forward_mode()
    rows = x.numel() // K
    if rows == 0:
        return [x.new_empty(*x.shape[:-1], N) for N in sizes]
    if grad or rows > MAX_ROWS:
        xs = x if xscale is None else x * xscale
        return [F.linear(xs, _k.dequantize_int4(*w, N, K, G), b)
                for w, b, N in zip(weights, biases, sizes)]
    return _k.int4_linear_multi(x, weights, biases, sizes, G, xscale)


def int4_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
                zeros: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                out_features: int | None = None, xscale: torch.Tensor | None = None) -> torch.Tensor:
    """x (..., in_features) bfloat16 -> (..., out_features) bfloat16 (16 times the
    tiles when out_features is None); packed, scales, zeros as pack_int4 lays
    them out.  See int4_linear_multi."""
    if packed.dim() != 4:
        raise ValueError(f"int4: packed must be (tiles, blocks, 64, 16) uint8, got {tuple(packed.shape)}")
    N = 16 * packed.shape[0] if out_features is None else int(out_features)
    return int4_linear_multi(x, [(packed, scales, zeros)], [bias], [N], xscale)[0]
