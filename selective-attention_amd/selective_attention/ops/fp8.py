"""Linear layers in 8 bits with block scales, and the rows that enter them.

    y[m, n] = sum_b s_x[m, b] s_w[n // 128, b] sum_{k in block b} c_x[m, k] c_w[n, k] + bias[n]

c e4m3 codes, b blocks of 128 columns, s powers of two: one for each block of a
row, one for each 128 by 128 of a weight, the smallest s with max|x| <= 448 s (1
for a block of zeros).  A scale is an e8m0 number; torch holds both types.

The rows are rounded by the op before the layer, in the pass that makes them:
rms_norm_fp8 (with the residual's addition), silu_mul_fp8 (SwiGLU's product) or
quantize_rows_fp8 (as they are, or times a gate); each code is the nearest to the
op's own value, not to that value rounded to bfloat16 first.  Infinities and NaN
become NaN codes, which make their row's outputs NaN and no other's; a value beyond
float32's range counts as infinite, one of 2^-150 and less as 0.  fp8_linear
takes such Fp8Rows, or a bfloat16 tensor that it rounds itself; a row's outputs do
not depend on the rows beside it, but for the order of fp32 sums.  It is
differentiable in x (a tensor) and bias: the gradient passes the rounding as it
is, dx = dy W with W the weights that the codes stand for, in bfloat16 (x times xscale
is then rounded to bfloat16 before its codes).

New ops (the reference's layers are nn.Linear in the model's dtype,
modules/feed_forward.py:4-11, behind modules/rms_norm.py:4-44).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from ..kernels import fp8 as _k
from ..kernels.common import in_forward_mode, needs_torch_ops
from ..kernels.fp8 import CODES, MAX_MATRICES, SCALES
from ..utils import check_ndim, check_shape

_BYTES = (SCALES, torch.uint8)


class Fp8Rows:
    """Rows in 8 bits: codes (..., 128 blocks) float8_e4m3fn, zeros behind the last
    feature, and scales (..., 4 ceil(blocks / 4)) float8_e8m0fnu (or its bytes, uint8),
    of which those behind the last block are not used.  shape is that of the tensor
    that the rows stand for, dtype bfloat16, that of the layers."""

    __slots__ = ("codes", "scales", "features")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, features: int | None = None):
        self.codes, self.scales = codes, scales
        self.features = codes.shape[-1] if features is None else features

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.features))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    @property
    def dtype(self) -> torch.dtype:
        return torch.bfloat16

    requires_grad = False

    def dequantize(self) -> torch.Tensor:
        """(..., features) float32: codes times scales."""
        kb = self.codes.shape[-1] // 128
        s = self.scales.view(SCALES)[..., :kb].float().repeat_interleave(128, -1)
        return (self.codes.float() * s)[..., :self.features]

    def __repr__(self) -> str:
        return f"Fp8Rows(shape={tuple(self.shape)}, device={self.device})"


def _check_rows(who: str, x: torch.Tensor, other: torch.Tensor | None, name: str) -> int:
    """The features of x, and of `other`, which has its shape and dtype."""
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{who}: x must have features, got shape {tuple(shape)}")
    if other is not None and (other.shape != shape or other.dtype != x.dtype):
        raise ValueError(f"{who}: {name} must be {tuple(shape)} {x.dtype}, got {tuple(other.shape)} {other.dtype}")
    return shape[-1]


def _no_gradient(who: str, x: torch.Tensor, *others):
    wanted = False
    if torch.is_grad_enabled():
        wanted = x.requires_grad
        for t in others:
            wanted = wanted or (t is not None and t.requires_grad)
    if wanted or in_forward_mode():
        raise RuntimeError(f"{who}: codes have no gradient; pass fp8_linear the rows in bfloat16 instead, "
                           "or call it under torch.no_grad()")


def quantize_rows_fp8(x: torch.Tensor, xscale: torch.Tensor | None = None) -> Fp8Rows:
    """x (..., features) float32 or bfloat16, or x * xscale (of x's shape and dtype), in 8 bits."""
    dim = _check_rows("quantize_rows_fp8", x, xscale, "xscale")
    _no_gradient("quantize_rows_fp8", x, xscale)
    codes, scales = _k.quantize_rows(x, xscale)
    return Fp8Rows(codes, scales, dim)


def silu_mul_fp8(a: torch.Tensor, c: torch.Tensor) -> Fp8Rows:
    """a * silu(c) of bfloat16 tensors of one shape (..., features), in 8 bits."""
    dim = _check_rows("silu_mul_fp8", a, c, "c")
    if a.dtype != torch.bfloat16:
        raise TypeError(f"silu_mul_fp8: a and c must be bfloat16, got {a.dtype}")
    _no_gradient("silu_mul_fp8", a, c)
    codes, scales = _k.quantize_rows(a, c, True)
    return Fp8Rows(codes, scales, dim)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 residual: torch.Tensor | None = None):
    """t rsqrt(mean(t^2) + eps) (1 + weight) in 8 bits, t = x, or x + residual in x's
    dtype: Fp8Rows, with a residual (t, Fp8Rows).  x, residual (..., features) float32
    or bfloat16, weight (features,)."""
    dim = _check_rows("rms_norm_fp8", x, residual, "residual")
    if weight.shape != (dim,):
        check_shape(weight, (dim,), name="weight")
    if dim > _k.MAX_NORM_DIM:
        raise ValueError(f"rms_norm_fp8: {dim} features, at most {_k.MAX_NORM_DIM}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"rms_norm_fp8: eps {eps} must not be negative")
    _no_gradient("rms_norm_fp8", x, weight, residual)
    if weight.dtype != torch.float32:
        weight = weight.float()
    t, codes, scales = _k.rms_norm(x, residual, weight, eps)
    rows = Fp8Rows(codes, scales, dim)
    return rows if residual is None else (t, rows)


def _exponents(top: torch.Tensor):
    """The scale of blocks with the largest magnitude top, as float32 and as e8m0."""
    part, power = torch.frexp(top)
    power = torch.where(top > 0, (power - 9 + (part > 0.875)).clamp(min=-126), 0)
    return torch.ldexp(torch.ones_like(top), power), (power + 127).to(torch.uint8)


def pack_fp8(codes: torch.Tensor, scales: torch.Tensor):
    """
    Args:
        codes: (out_features, in_features) float8_e4m3fn, no NaN
        scales: (ceil(out_features / 128), ceil(in_features / 128)), powers of two from
            2^-126 to 2^127: float8_e8m0fnu, its bytes (uint8), or a float type
    Returns:
        (packed, scales) as fp8_linear takes them: packed (ceil(N / 16), ceil(K / 128), 8,
        16, 16) uint8, tiles of 16 rows and 128 columns with 16 columns of their rows
        after each other; scales (ceil(N / 128), 4 ceil(K / 512)) float8_e8m0fnu
    """
    check_ndim(codes, 2, name="codes")
    N, K = codes.shape
    if N == 0 or K == 0:
        raise ValueError("pack_fp8: empty weight")
    if codes.dtype != CODES:
        raise TypeError(f"pack_fp8: codes must be {CODES}, got {codes.dtype}")
    nb, kb = _k.blocks_of(N), _k.blocks_of(K)
    check_shape(scales, (nb, kb), name="scales")
    if bool(((codes.view(torch.uint8) & 127) == 127).any()):
        raise ValueError("pack_fp8: the codes hold NaN")
    if scales.dtype in _BYTES:
        byte = scales.view(torch.uint8)
        if bool(((byte == 0) | (byte == 255)).any()):
            raise ValueError("pack_fp8: scales must be 2^-126 to 2^127")
    elif scales.is_floating_point():
        part, power = torch.frexp(scales.double())
        if not bool(((part == 0.5) & (power >= -125) & (power <= 128)).all()):
            raise ValueError("pack_fp8: scales must be powers of two from 2^-126 to 2^127 (others: quantize_fp8 the "
                             "weight that they stand for)")
        byte = (power + 126).to(torch.uint8)
    else:
        raise TypeError(f"pack_fp8: scales must be floating or e8m0 bytes, got {scales.dtype}")
    c = F.pad(codes.view(torch.uint8), (0, -K % 128, 0, -N % 16))
    packed = c.view(-1, 16, kb, 8, 16).permute(0, 2, 3, 1, 4).contiguous()
    return packed, F.pad(byte, (0, -kb % 4), value=127).contiguous().view(SCALES)


def quantize_fp8(weight: torch.Tensor):
    """weight (out_features, in_features) -> (packed, scales) as fp8_linear takes them,
    each 128 by 128 block rounded to the nearest codes of its scale."""
    check_ndim(weight, 2, name="weight")
    N, K = weight.shape
    if N == 0 or K == 0:
        raise ValueError("quantize_fp8: empty weight")
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("quantize_fp8: the weight holds infinities or NaN")
    nb, kb = _k.blocks_of(N), _k.blocks_of(K)
    w = F.pad(weight.detach().float(), (0, -K % 128, 0, -N % 128)).view(nb, 128, kb, 128)
    s, byte = _exponents(w.abs().amax((1, 3)))
    codes = (w / s[:, None, :, None]).to(CODES).view(nb * 128, kb * 128)
    return pack_fp8(codes.view(torch.uint8)[:N, :K].contiguous().view(CODES), byte)


def _weight(packed: torch.Tensor, scales: torch.Tensor, N: int, K: int):
    """Checks a packed weight against its sizes."""
    tiles, blocks = (N + 15) >> 4, (K + 127) >> 7
    if packed.shape != (tiles, blocks, 8, 16, 16) or packed.dtype != torch.uint8 or not tiles:
        raise ValueError(f"fp8: packed must be (tiles, blocks, 8, 16, 16) uint8, {(tiles, blocks, 8, 16, 16)} for {N} "
                         f"out_features and {K} in_features, got {tuple(packed.shape)} {packed.dtype}")
    if scales.shape != ((N + 127) >> 7, (blocks + 3) >> 2 << 2):
        raise ValueError(f"fp8: scales must be {((N + 127) >> 7, (blocks + 3) >> 2 << 2)}, got {tuple(scales.shape)}")
    if scales.dtype not in _BYTES:
        raise TypeError(f"fp8: scales must be {SCALES} or its bytes, got {scales.dtype}")
    if not (packed.is_contiguous() and scales.is_contiguous()) or packed.data_ptr() & 15 or scales.data_ptr() & 3:
        raise ValueError("fp8: packed and scales must be contiguous on 16- and 4-byte boundaries")


def dequantize_fp8(packed: torch.Tensor, scales: torch.Tensor, out_features: int | None = None,
                   in_features: int | None = None) -> torch.Tensor:
    """(out_features, in_features) bfloat16: the weights that the codes stand for (exact
    for scales from 2^-117 on); without sizes, with the padding."""
    if packed.dim() != 5:
        raise ValueError(f"fp8: packed must be (tiles, blocks, 8, 16, 16) uint8, got {tuple(packed.shape)}")
    N = 16 * packed.shape[0] if out_features is None else int(out_features)
    K = 128 * packed.shape[1] if in_features is None else int(in_features)
    _weight(packed, scales, N, K)
    return _k.dequantize(packed, scales, N, K)


def _rows(x: Fp8Rows):
    """(features, codes, scales) of rows, checked; slices are copied."""
    K, codes, scales = x.features, x.codes, x.scales
    shape, s = codes.shape, scales.shape
    Kp = (K + 127) >> 7 << 7
    if codes.dtype is not CODES or not Kp or not shape or shape[-1] != Kp:
        raise ValueError(f"fp8_linear: codes must be (..., {Kp}) {CODES}, got {tuple(shape)} {codes.dtype}")
    beside = len(s) == len(shape) and (s[0] == shape[0] if len(s) == 2 else s[:-1] == shape[:-1])
    if not beside or s[-1] != (Kp + 511) >> 9 << 2 or scales.dtype not in _BYTES:
        raise ValueError(f"fp8_linear: scales must be (..., {(Kp + 511) >> 9 << 2}) {SCALES} beside codes "
                         f"{tuple(shape)}, got {tuple(s)} {scales.dtype}")
    if not codes.is_contiguous() or codes.data_ptr() & 15:
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not scales.is_contiguous() or scales.data_ptr() & 3:
        scales = scales.clone(memory_format=torch.contiguous_format)
    return K, codes, scales


class _ColumnSumsFn(torch.autograd.Function):
    """The sums over the rows of (..., N), differentiable any number of times."""

    @staticmethod
    def forward(ctx, dy):
        ctx.shape = dy.shape
        return _k.column_sums(dy)

    @staticmethod
    def backward(ctx, g):
        return g.expand(ctx.shape)


class _Fp8LinearFn(torch.autograd.Function):
    """x W^T + bias; the gradient passes the rows' rounding as it is."""

    @staticmethod
    def forward(ctx, x, rows, bias, packed, scales, N):
        ctx.save_for_backward(packed, scales)
        ctx.N, ctx.K = N, None if x is None else x.shape[-1]
        if rows is None:
            return _k.linear_multi_bf16(x, None, [(packed, scales)], [bias], [N])[0]
        return _k.linear_multi(*rows, [(packed, scales)], [bias], [N])[0]

    @staticmethod
    def backward(ctx, dy):
        dx = db = None
        if ctx.needs_input_grad[0]:
            w = _k.dequantize(*ctx.saved_tensors, ctx.N, ctx.K)
            dx = (dy.reshape(-1, ctx.N) @ w).view(*dy.shape[:-1], ctx.K)
        if ctx.needs_input_grad[2]:
            if needs_torch_ops(dy):
                db = dy.reshape(-1, ctx.N).sum(0)
            else:   # (a launch of its own leaves no history)
                db = _ColumnSumsFn.apply(dy) if torch.is_grad_enabled() else _k.column_sums(dy)
        return dx, None, db, None, None, None


def fp8_linear_multi(x, weights, biases, sizes, xscale: torch.Tensor | None = None) -> list:
    """[x W_i^T + bias_i] of 1..4 weights (packed, scales) in one launch; sizes: their
    out_features.  x: Fp8Rows, or (..., in_features) bfloat16, which is rounded to 8
    bits first, times xscale (x's shape, bfloat16) where that is given.  Returns
    bfloat16 (..., out_features) tensors."""
    n = len(weights)
    if not 1 <= n <= MAX_MATRICES or len(biases) != n or len(sizes) != n:
        raise ValueError(f"fp8_linear_multi: 1..{MAX_MATRICES} weights with as many biases and sizes, "
                         f"got {n}, {len(biases)}, {len(sizes)}")
    is_rows = type(x) is Fp8Rows
    if is_rows:
        if xscale is not None:
            raise ValueError("fp8_linear: xscale goes with x as a tensor, not with rows in 8 bits")
        K, codes, scales = _rows(x)
        grad = False
    else:
        K = _check_rows("fp8_linear", x, xscale, "xscale")
        if x.dtype != torch.bfloat16:
            raise TypeError(f"fp8_linear: x must be bfloat16 or Fp8Rows, got {x.dtype}")
        grad = x.requires_grad or (xscale is not None and xscale.requires_grad)
    for (packed, ws), b, N in zip(weights, biases, sizes):
        _weight(packed, ws, N, K)
        if b is not None:
            if b.shape != (N,):
                check_shape(b, (N,), name="bias")
            if b.dtype != torch.bfloat16:
                raise TypeError(f"fp8_linear: bias must be bfloat16, got {b.dtype}")
            grad = grad or b.requires_grad
    if (grad and torch.is_grad_enabled()) or in_forward_mode():
        if not is_rows and xscale is not None:
            x = x * xscale
        rows = (codes, scales) if is_rows else None
        return [_Fp8LinearFn.apply(None if is_rows else x, rows, b, *w, N)
                for w, b, N in zip(weights, biases, sizes)]
    if is_rows:
        return _k.linear_multi(codes, scales, weights, biases, sizes)
    return _k.linear_multi_bf16(x, xscale, weights, biases, sizes)


def fp8_linear(x, packed: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
               out_features: int | None = None, xscale: torch.Tensor | None = None) -> torch.Tensor:
    """x Fp8Rows or (..., in_features) bfloat16 -> (..., out_features) bfloat16 (16 times
    the tiles when out_features is None); packed, scales as quantize_fp8 gives them.
    See fp8_linear_multi."""
    if packed.dim() != 5:
        raise ValueError(f"fp8: packed must be (tiles, blocks, 8, 16, 16) uint8, got {tuple(packed.shape)}")
    N = 16 * packed.shape[0] if out_features is None else int(out_features)
    return fp8_linear_multi(x, [(packed, scales)], [bias], [N], xscale)[0]
