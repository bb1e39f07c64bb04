"""Launchers of the 8-bit linear layers and of the rows that enter them
(csrc/fp8_rows.hip, csrc/fp8_linear.hip; the reference's layers are nn.Linear in
the model's dtype)."""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .common import act_dtype_code, call_on, require_device, require_one_device

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
MAX_MATRICES = 4
MAX_NORM_DIM = 65536
MAX_ROWS = 1 << 24


def blocks_of(n: int) -> int:
    return (n + 127) // 128


def words_of(n: int) -> int:
    """Bytes of a row of scales: one a block of 128, whole words of four."""
    return (n + 511) // 512 * 4


def _strided(t: torch.Tensor, dim: int) -> torch.Tensor:
    """t (..., dim) as rows of one stride, those of a longer row as they lie."""
    if t.is_contiguous():
        return t
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    return t if t.stride(1) == 1 and t.stride(0) >= dim else t.contiguous()


def _outputs(lead, dim: int, device):
    kb = blocks_of(dim)
    return (torch.empty((*lead, 128 * kb), dtype=CODES, device=device),
            torch.empty((*lead, (kb + 3) // 4 * 4), dtype=SCALES, device=device))


def quantize_rows(x: torch.Tensor, gate: torch.Tensor | None, silu: bool = False):
    """x, gate (..., dim) of one dtype -> (codes, scales) of x, x * gate or x * silu(gate)."""
    require_one_device(x, gate)
    dim = x.shape[-1]
    codes, scales = _outputs(x.shape[:-1], dim, x.device)
    rows = x.numel() // dim
    if rows == 0:
        return codes, scales
    xr, gr = _strided(x, dim), None if gate is None else _strided(gate, dim)
    ldx = dim if xr.is_contiguous() else xr.stride(0)
    ldg = dim if gr is None or gr.is_contiguous() else gr.stride(0)
    call_on(x, "sa_rows_fp8", act_dtype_code(x.dtype), xr.data_ptr(), _lib.ptr(gr), int(silu), rows, dim, ldx, ldg,
            codes.data_ptr(), scales.data_ptr(), _lib.stream_of(x))
    return codes, scales


def rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float):
    """x, residual (..., dim) of one dtype, weight (dim,) float32 -> (sum or None, codes, scales)."""
    require_one_device(x, residual, weight)
    dim = x.shape[-1]
    codes, scales = _outputs(x.shape[:-1], dim, x.device)
    total = None if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows = x.numel() // dim
    if rows == 0:
        return total, codes, scales
    xr = _strided(x, dim)
    res = None if residual is None else residual.contiguous()
    w = weight.contiguous()
    call_on(x, "sa_rms_norm_fp8", act_dtype_code(x.dtype), xr.data_ptr(), _lib.ptr(res), w.data_ptr(), rows, dim,
            dim if xr.is_contiguous() else xr.stride(0), eps, _lib.ptr(total), codes.data_ptr(), scales.data_ptr(),
            _lib.stream_of(x))
    return total, codes, scales


def linear_multi(codes, scales, lead, K: int, weights, biases, sizes):
    """codes, scales of rows with the leading sizes `lead`; weights [(packed, scales)], biases
    [(N_i,) bf16 or None], sizes [N_i] -> [(*lead, N_i) bf16], one launch."""
    require_one_device(codes, scales, *(t for w in weights for t in w), *biases)
    rows = codes.numel() // codes.shape[-1]
    ys, words, kept = [], [], []
    for (packed, ws), b, N in zip(weights, biases, sizes):
        y = torch.empty((*lead, N), dtype=torch.bfloat16, device=codes.device)
        if b is not None and not b.is_contiguous():
            b = b.contiguous()
            kept.append(b)
        words += (packed.data_ptr(), ws.data_ptr(), 0 if b is None else b.data_ptr(), y.data_ptr(), N)
        ys.append(y)
    if rows:
        call_on(codes, "sa_fp8_linear", codes.data_ptr(), scales.data_ptr(), rows, K, len(ys),
                (ctypes.c_int64 * len(words))(*words), _lib.stream_of(codes))
    return ys


def dequantize(packed, scales, N: int, K: int):
    """(N, K) bf16: what the packed weights stand for."""
    require_device(packed, scales)
    out = torch.empty(N, K, dtype=torch.bfloat16, device=packed.device)
    call_on(packed, "sa_fp8_dequant_bf16", packed.data_ptr(), scales.data_ptr(), N, K, out.data_ptr(),
            _lib.stream_of(packed))
    return out
