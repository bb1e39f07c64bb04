"""Oracle of the 4-bit linear layers, in float64 on the CPU."""
from __future__ import annotations

import torch


def unpack(packed: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """Codes (N, K), byte by byte: byte 4 j + i of lane 16 g + c of tile (t, b)
    holds columns 128 b + 32 j + 8 g + 2 i (low half) and + 1 of row 16 t + c."""
    nt, kb = packed.shape[:2]
    out = torch.zeros(nt * 16, kb * 128, dtype=torch.int64)
    p = packed.to(torch.int64)
    for g in range(4):
        for c in range(16):
            for j in range(4):
                for i in range(4):
                    byte = p[:, :, 16 * g + c, 4 * j + i]
                    rows = torch.arange(nt) * 16 + c
                    cols = torch.arange(kb) * 128 + 32 * j + 8 * g + 2 * i
                    out[rows[:, None], cols[None]] = byte & 15
                    out[rows[:, None], cols[None] + 1] = byte >> 4
    return out[:N, :K]


def weight(packed, scales, zeros, N: int, K: int) -> torch.Tensor:
    """(N, K) float64: scale (code - zero)."""
    code = unpack(packed, N, K).double()
    G = 128 * packed.shape[1] // scales.shape[1]
    of = torch.arange(K) // G

    def each(t):   # (tiles, groups, 16) -> (N, K)
        return t.double().transpose(1, 2).reshape(-1, t.shape[1])[:N][:, of]
    return each(scales) * (code - (8.0 if zeros is None else each(zeros)))


def linear(x, w, bias=None, xscale=None):
    """(y, A): x w^T + bias in float64 and the sum of the magnitudes of its terms."""
    x = x.double() if xscale is None else (x * xscale).double()
    y, A = x @ w.t(), x.abs() @ w.abs().t()
    return (y, A) if bias is None else (y + bias.double(), A + bias.double().abs())
