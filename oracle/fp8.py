"""Oracle of the 8-bit linear layers, in float64 on the CPU."""
from __future__ import annotations

import torch


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number of |y| <= 448, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def half_step(y: torch.Tensor) -> torch.Tensor:
    """Half the distance of e4m3 numbers around y: the largest error of a rounding."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 4)


def scale_of(top: torch.Tensor) -> torch.Tensor:
    """The smallest 2^e, e >= -126, with top <= 448 2^e; 1 where top is 0."""
    e = torch.arange(-126, 128, dtype=torch.float64)
    at = torch.searchsorted(448.0 * torch.exp2(e), top.double().contiguous())
    return torch.where(top > 0, torch.exp2(e[at]), 1.0)


def rows(v: torch.Tensor):
    """v (rows, dim) -> (codes (rows, 128 kb), scales (rows, 4 ceil(kb / 4))), what the
    bytes stand for; infinities and NaN as NaN."""
    v = v.double()
    M, D = v.shape
    kb = (D + 127) // 128
    v = torch.nn.functional.pad(v, (0, 128 * kb - D)).view(M, kb, 128)
    fine = torch.isfinite(v)
    s = scale_of(torch.where(fine, v.abs(), 0.0).amax(2))
    codes = torch.where(fine, e4m3(torch.where(fine, v, 0.0) / s[..., None]), torch.nan)
    return codes.view(M, -1), torch.nn.functional.pad(s, (0, -kb % 4), value=1.0)


def rms_norm(x, weight, eps, residual=None):
    """(t, v): the summed rows in x's dtype, and their norm in float64."""
    t = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = t.double()
    return t, d / torch.sqrt(d.pow(2).mean(-1, keepdim=True) + eps) * (1.0 + weight.double())


def unpack(packed: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """Codes (N, K) as numbers, piece by piece: piece j of tile (t, b) holds columns
    128 b + 16 j .. + 15 of rows 16 t .. + 15."""
    nt, kb = packed.shape[:2]
    out = torch.zeros(nt * 16, kb * 128, dtype=torch.float64)
    v = packed.cpu().view(torch.float8_e4m3fn).double()
    for t in range(nt):
        for b in range(kb):
            for j in range(8):
                out[16 * t:16 * t + 16, 128 * b + 16 * j:128 * b + 16 * j + 16] = v[t, b, j]
    return out[:N, :K]


def weight(packed, scales, N: int, K: int) -> torch.Tensor:
    """(N, K) float64: code times scale."""
    s = torch.exp2(scales.cpu().view(torch.uint8).double() - 127)
    return unpack(packed, N, K) * s[torch.arange(N) // 128][:, torch.arange(K) // 128]


def values(codes, scales, K: int) -> torch.Tensor:
    """(rows, K) float64 of rows in 8 bits."""
    s = torch.exp2(scales.cpu().view(torch.uint8).double() - 127)
    return codes.cpu().double()[:, :K] * s[:, torch.arange(K) // 128]


def linear(x, w, bias=None):
    """(y, A): x w^T + bias in float64 and the sum of the magnitudes of its terms."""
    y, A = x @ w.t(), x.abs() @ w.abs().t()
    return (y, A) if bias is None else (y + bias.double(), A + bias.double().abs())
