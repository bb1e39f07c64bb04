"""Oracle of the paged KV cache held in 8 bits, in float64 on the CPU.

One block (a page of one kv head) at a time: the e4m3 rounding and the block's
scale from their definitions, the cache's state after a prompt and after single
tokens, and the decode attention over what the cache stands for.
"""
from __future__ import annotations

import math

import torch


def e4m3(y: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 number of |y| <= 448 (3 mantissa bits, exponents -6..8,
    steps of 2^-9 below 2^-6), ties to even; NaN for what is no finite number."""
    y = y.double()
    fin = torch.isfinite(y)
    a = torch.where(fin, y, 0.0).abs()
    e = torch.frexp(a.clamp(min=2.0 ** -6))[1].double() - 1.0
    step = torch.exp2(e - 3.0)
    out = torch.copysign(torch.round(a / step) * step, y)
    return torch.where(fin, out, math.nan)


def block(x: torch.Tensor, keep: torch.Tensor | None = None):
    """x (tokens, dim) -> (codes as float64, scale): s = 2^e, the smallest with
    max|x| <= 448 s over the finite values of the tokens in keep (e >= -126; 1
    when that is 0); tokens outside keep are 0."""
    x = x.double()
    if keep is not None:
        x = torch.where(keep[:, None], x, 0.0)
    fin = torch.where(torch.isfinite(x), x, 0.0).abs()
    top = float(fin.max()) if fin.numel() else 0.0
    scale = 1.0
    if top > 0.0:
        e = -126
        while top > 448.0 * 2.0 ** e:
            e += 1
        scale = 2.0 ** e
    return e4m3(x / scale), scale


class CacheRef:
    """One row and kv head: tokens in order, each (k, v, log_gate)."""

    def __init__(self, page_size: int, gated: bool):
        self.ps, self.gated = page_size, gated
        self.k, self.v, self.g = [], [], []

    def append(self, k, v, g=0.0):
        self.k.append(k.double())
        self.v.append(v.double())
        self.g.append(float(g))

    def blocks(self):
        """[(k codes, k scale, v codes, v scale)] of the full blocks."""
        out = []
        for p in range(len(self.k) // self.ps):
            at = slice(p * self.ps, (p + 1) * self.ps)
            keep = None
            if self.gated:
                keep = torch.tensor([g > -math.inf for g in self.g[at]])
                keep[-1] = True
            kc, ks = block(torch.stack(self.k[at]), keep)
            vc, vs = block(torch.stack(self.v[at]), keep)
            out.append((kc, ks, vc, vs))
        return out

    def keys_values(self):
        """(tokens, dim) keys and values as the cache stands for them."""
        full = self.blocks()
        done = len(full) * self.ps
        k = [kc * ks for kc, ks, _, _ in full] + [t[None] for t in self.k[done:]]
        v = [vc * vs for _, _, vc, vs in full] + [t[None] for t in self.v[done:]]
        return torch.cat(k), torch.cat(v)


def attend(q, k, v, gates=None, scale=None):
    """q (dim,), k, v (tokens, dim), gates (tokens,) or None -> (dim,), float64:
    softmax of scale q.k + gate, the newest key without its gate, over the keys
    whose gate is not -inf."""
    n, D = k.shape
    if n == 0:
        return torch.zeros(v.shape[1], dtype=torch.float64)
    on = torch.ones(n, dtype=torch.bool)
    bias = torch.zeros(n, dtype=torch.float64)
    if gates is not None:
        bias = gates.double().clone()
        on = bias != -math.inf
        bias[-1], on[-1] = 0.0, True
    s = (k[on] @ q.double()) * (D ** -0.5 if scale is None else scale) + bias[on]
    return torch.softmax(s, 0) @ v[on]
