"""Launchers of the 8-bit linear layers and of the rows that enter them
(csrc/fp8_rows.hip, csrc/fp8_linear.hip; the reference's layers are nn.Linear in
the model's dtype)."""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from .common import act_dtype_code, require_device

CODES, SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu
MAX_MATRICES = 4
MAX_NORM_DIM = 65536
FEW_ROWS = 16     # bfloat16 rows that the product itself rounds


def blocks_of(n: int) -> int:
    return (n + 127) // 128


def _strided(t: torch.Tensor, dim: int):
    """(rows, stride) of t (..., dim): rows of one stride, those of a longer row as they lie."""
    if t.is_contiguous():
        return t, dim
    if t.dim() != 2:
        t = t.reshape(-1, dim)
    if t.stride(1) != 1 or t.stride(0) < dim:
        return t.contiguous(), dim
    return t, t.stride(0)


# (a decode step's calls are bound by host time, and looking these up is a part of it)
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _one_device(x: torch.Tensor, *others) -> int:
    """The index of the tensors' device: require_device without device objects where all is well."""
    d = x.get_device()
    if d < 0:
        require_device(x)
    for t in others:
        if t is not None and t.get_device() != d:
            require_device(x, t)
    return d


def _launch(d: int, name: str, *args) -> None:
    """_lib.call with device d current, on its current stream, the last argument."""
    if _device() == d:
        return _lib.call(name, *args, _stream(d))
    with torch.cuda.device(d):
        return _lib.call(name, *args, _stream(d))


def _last(shape, n: int) -> tuple:
    """shape with n as its last size."""
    return (shape[0], n) if len(shape) == 2 else (*shape[:-1], n)


def _outputs(x: torch.Tensor, dim: int):
    kb, shape = (dim + 127) >> 7, x.shape
    return (x.new_empty(_last(shape, kb << 7), dtype=CODES),
            x.new_empty(_last(shape, (kb + 3) >> 2 << 2), dtype=SCALES))


def quantize_rows(x: torch.Tensor, gate: torch.Tensor | None, silu: bool = False):
    """x, gate (..., dim) of one dtype -> (codes, scales) of x, x * gate or x * silu(gate)."""
    d = _one_device(x, gate)
    dtype, dim = act_dtype_code(x.dtype), x.shape[-1]
    codes, scales = _outputs(x, dim)
    rows = x.numel() // dim
    if rows:
        xr, ldx = _strided(x, dim)
        gr, ldg = (None, dim) if gate is None else _strided(gate, dim)
        _launch(d, "sa_rows_fp8", dtype, xr.data_ptr(), None if gr is None else gr.data_ptr(), silu, rows, dim, ldx,
                ldg, codes.data_ptr(), scales.data_ptr())
    return codes, scales


def rms_norm(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float):
    """x, residual (..., dim) of one dtype, weight (dim,) float32 -> (sum or None, codes, scales)."""
    d = _one_device(x, residual, weight)
    dtype, dim = act_dtype_code(x.dtype), x.shape[-1]
    codes, scales = _outputs(x, dim)
    total = None if residual is None else x.new_empty(x.shape)
    rows = x.numel() // dim
    if rows:
        xr, ldx = _strided(x, dim)
        res = None if residual is None else residual.contiguous()
        w = weight.contiguous()
        _launch(d, "sa_rms_norm_fp8", dtype, xr.data_ptr(), None if res is None else res.data_ptr(), w.data_ptr(),
                rows, dim, ldx, eps, None if total is None else total.data_ptr(), codes.data_ptr(),
                scales.data_ptr())
    return total, codes, scales


_WORDS = [ctypes.c_int64 * (5 * n) for n in range(MAX_MATRICES + 1)]


def _matrices(x, d, weights, biases, sizes):
    """([y_i] for the rows of x on device d, the words of the call, what it keeps alive)."""
    ys, words, kept = [], [], []
    shape, dtype = x.shape, torch.bfloat16
    for (packed, ws), b, N in zip(weights, biases, sizes):
        if packed.get_device() != d or ws.get_device() != d or (b is not None and b.get_device() != d):
            require_device(x, packed, ws, b)
        y = x.new_empty(_last(shape, N), dtype=dtype)
        if b is not None and not b.is_contiguous():
            b = b.contiguous()
            kept.append(b)
        words += (packed.data_ptr(), ws.data_ptr(), 0 if b is None else b.data_ptr(), y.data_ptr(), N)
        ys.append(y)
    return ys, _WORDS[len(ys)](*words), kept


def linear_multi(codes, scales, weights, biases, sizes):
    """codes, scales of rows (..., 128 blocks); weights [(packed, scales)], biases [(N_i,)
    bf16 or None], sizes [N_i] -> [(..., N_i) bf16], one launch."""
    d = _one_device(codes, scales)
    Kp = codes.shape[-1]
    ys, words, _kept = _matrices(codes, d, weights, biases, sizes)
    rows = codes.numel() // Kp
    if rows:
        _launch(d, "sa_fp8_linear", codes.data_ptr(), scales.data_ptr(), rows, Kp, len(ys), words)
    return ys


def linear_multi_bf16(x, xscale, weights, biases, sizes):
    """The same of x, or x * xscale, (..., K) bf16: up to 16 rows in one launch, more
    through their codes."""
    K = x.shape[-1]
    rows = x.numel() // K
    if not 0 < rows <= FEW_ROWS:
        return linear_multi(*quantize_rows(x, xscale), weights, biases, sizes)
    d = _one_device(x, xscale)
    ys, words, _kept = _matrices(x, d, weights, biases, sizes)
    xr, ldx = _strided(x, K)
    gr, ldg = (None, K) if xscale is None else _strided(xscale, K)
    _launch(d, "sa_fp8_linear_bf16", xr.data_ptr(), None if gr is None else gr.data_ptr(), rows, K, ldx, ldg, len(ys),
            words)
    return ys


def dequantize(packed, scales, N: int, K: int):
    """(N, K) bf16: what the packed weights stand for."""
    d = _one_device(packed, scales)
    out = torch.empty(N, K, dtype=torch.bfloat16, device=packed.device)
    _launch(d, "sa_fp8_dequant_bf16", packed.data_ptr(), scales.data_ptr(), N, K, out.data_ptr())
    return out


def column_sums(x: torch.Tensor):
    """(N,) bf16: the sums over all rows of x (..., N) bf16, in fp32."""
    d = _one_device(x)
    N = x.shape[-1]
    x = x.contiguous()
    M = x.numel() // N
    if not M:
        return x.new_zeros(N)
    out = x.new_empty(N)
    need = _lib.load().sa_colsum_bf16_workspace_size(M, N)
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    _launch(d, "sa_colsum_bf16", x.data_ptr(), M, N, out.data_ptr(), _lib.ptr(ws), need)
    return out
