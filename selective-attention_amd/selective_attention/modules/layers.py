"""Library layers of the LMs, as the reference defines them: RMSNorm
(modules/rms_norm.py:4-44), RoPE (modules/rope.py:9-64), SwiGLU
(modules/feed_forward.py:4-11).  In inference RMSNorm and the rotation of q
and k run as single fused kernels (kernels/lm_ops.py); with autograd (the
SSM blocks can train) RMSNorm keeps its torch composite."""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..kernels.int4 import MAX_MATRICES
from ..kernels.lm_ops import (add_rms_norm, add_rms_norm_supported, gemv, gemv_multi,
                              gemv_supported, rms_norm, rope_qk, silu_mul)
from ..ops.int4 import int4_linear, int4_linear_multi, quantize_int4


def _gemv_ok(x: torch.Tensor, lin: nn.Linear) -> bool:
    return (gemv_supported(x, lin.weight)
            and (lin.bias is None or lin.bias.dtype == torch.bfloat16)
            and not (torch.is_grad_enabled() and (x.requires_grad or lin.weight.requires_grad)))


class Linear(nn.Linear):
    """nn.Linear (same parameters and state-dict names) whose inference
    forward on at most 8 bf16 rows, the decode steps' shape, runs the
    small-batch GEMV kernel instead of a GEMM."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if _gemv_ok(x, self):
            return gemv(x, self.weight, self.bias)
        return super().forward(x)

    def split_forward(self, x: torch.Tensor, sizes) -> list:
        """torch.split(self(x), sizes, dim=-1).  On the decode shape the
        weight's row blocks go to one multi-GEMV launch that writes each
        piece as its own contiguous tensor (no copies of split views)."""
        bs = [None] * len(sizes) if self.bias is None else torch.split(self.bias, sizes)
        if _gemv_ok(x, self) and len(sizes) <= 4:
            return gemv_multi(x, torch.split(self.weight, sizes), bs)
        if x.is_cuda and not torch.is_grad_enabled():
            # one GEMM per row block: contiguous pieces, no copies of split views later
            return [F.linear(x, w, bb) for w, bb in zip(torch.split(self.weight, sizes), bs)]
        return list(torch.split(self(x), sizes, dim=-1))


class Int4Linear(nn.Module):
    """A linear layer whose weight is kept as 4-bit codes with a scale for each
    group of input features (ops/int4.py), for inference: bfloat16 rows, no
    weight gradient.  Buffers: packed, scales, zeros (None: symmetric), bias, in
    bfloat16 whatever the module is cast to."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 group_size: int = 128, symmetric: bool = True, device=None):
        super().__init__()
        self.in_features, self.out_features = in_features, out_features
        self.group_size, self.symmetric = group_size, symmetric
        nt, kb = (out_features + 15) // 16, (in_features + 127) // 128
        f = (nt, kb * 128 // group_size, 16)

        def make(shape):
            return torch.zeros(shape, dtype=torch.bfloat16, device=device)
        self.register_buffer("packed", torch.zeros(nt, kb, 64, 16, dtype=torch.uint8, device=device))
        self.register_buffer("scales", make(f))
        self.register_buffer("zeros", None if symmetric else make(f))
        self.register_buffer("bias", make(out_features) if bias else None)

    @classmethod
    def from_linear(cls, lin: nn.Linear, group_size: int = 128, symmetric: bool = True) -> "Int4Linear":
        """lin's weight rounded to its nearest codes (quantize_int4)."""
        q = cls(lin.in_features, lin.out_features, lin.bias is not None, group_size, symmetric,
                lin.weight.device)
        q.packed, q.scales, q.zeros = quantize_int4(lin.weight, group_size, symmetric)
        if lin.bias is not None:
            q.bias = lin.bias.detach().to(torch.bfloat16)
        return q

    def _apply(self, fn, *args, **kwargs):
        kept = {n: getattr(self, n) for n in ("scales", "zeros", "bias")}
        super()._apply(fn, *args, **kwargs)
        for n, t in kept.items():   # moved, not cast
            new = getattr(self, n)
            if t is not None and new.dtype != torch.bfloat16:
                setattr(self, n, t.to(new.device))
        return self

    def weights(self):
        return self.packed, self.scales, self.zeros

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return int4_linear(x, self.packed, self.scales, self.zeros, self.bias, self.out_features)

    def split_forward(self, x: torch.Tensor, sizes) -> list:
        """torch.split(self(x), sizes, dim=-1), each piece a contiguous tensor; one
        launch of several matrices where the pieces are whole tiles."""
        if len(sizes) <= MAX_MATRICES and min(sizes) > 0 and all(n % 16 == 0 for n in sizes[:-1]):
            tiles = [(n + 15) // 16 for n in sizes]
            cut = [[None] * len(sizes) if t is None else torch.split(t, tiles) for t in self.weights()]
            bs = [None] * len(sizes) if self.bias is None else torch.split(self.bias, sizes)
            return int4_linear_multi(x, list(zip(*cut)), bs, sizes)
        return [p.contiguous() for p in torch.split(self(x), sizes, dim=-1)]

    def extra_repr(self) -> str:
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, group_size={self.group_size}, symmetric={self.symmetric}")


def quantize_linears(module: nn.Module, group_size: int = 128, symmetric: bool = True) -> nn.Module:
    """Replace every linear layer inside `module` by its Int4Linear, in place."""
    for name, child in module.named_children():
        if isinstance(child, nn.Linear):
            setattr(module, name, Int4Linear.from_linear(child, group_size, symmetric))
        else:
            quantize_linears(child, group_size, symmetric)
    return module


def project(x: torch.Tensor, linears, xscale: torch.Tensor | None = None) -> list:
    """[lin(x * xscale if xscale is given else x) for lin in linears]: one
    multi-GEMV launch on the decode shape (at most 4 layers), where the
    product x * xscale is taken in bf16 as torch does; 4-bit layers of one kind
    likewise."""
    if all(isinstance(lin, Int4Linear) for lin in linears):
        if len(linears) <= MAX_MATRICES and len({(lin.group_size, lin.symmetric) for lin in linears}) == 1:
            return int4_linear_multi(x, [lin.weights() for lin in linears],
                                     [lin.bias for lin in linears],
                                     [lin.out_features for lin in linears], xscale)
    elif len(linears) <= 4 and all(isinstance(lin, nn.Linear) and _gemv_ok(x, lin) for lin in linears):
        return gemv_multi(x, [lin.weight for lin in linears], [lin.bias for lin in linears], xscale)
    xs = x if xscale is None else x * xscale
    return [lin(xs) for lin in linears]


class RMSNorm(nn.Module):
    """x * rsqrt(mean(x^2) + eps) * (1 + weight), computed in fp32 and
    returned in the dtype of x; the weight starts at 0 (modules/rms_norm.py)."""

    def __init__(self, dim: int, num_groups: int | None = None, eps: float = 1e-6,
                 elementwise_affine: bool = True):
        super().__init__()
        self.eps = eps
        self.num_groups = num_groups
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            shape = (dim,) if num_groups is None else (num_groups, dim)
            self.weight = nn.Parameter(torch.zeros(shape))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if (self.elementwise_affine and x.is_cuda and x.is_contiguous()
                and x.dtype in (torch.float32, torch.bfloat16)
                and not (torch.is_grad_enabled() and (x.requires_grad or self.weight.requires_grad))):
            return rms_norm(x, self.weight, self.eps)     # one fused kernel (inference)
        xf = x.float()
        out = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        if self.elementwise_affine:
            out = out * (1.0 + self.weight.float())
        return out.type_as(x)

    def add_forward(self, x: torch.Tensor, y: torch.Tensor):
        """(x + y, self(x + y)): a pre-norm block's residual add and its next
        norm, in one kernel in inference for bf16 rows of 512k <= 4096 elements."""
        if (self.elementwise_affine and add_rms_norm_supported(x, self.weight)
                and not (torch.is_grad_enabled()
                         and (x.requires_grad or y.requires_grad or self.weight.requires_grad))):
            return add_rms_norm(x, y, self.weight, self.eps)
        s = x + y
        return s, self(s)


def _rotate_half(x: torch.Tensor) -> torch.Tensor:
    h = x.shape[-1] // 2
    return torch.cat((-x[..., h:], x[..., :h]), dim=-1)


class RoPE(nn.Module):
    """Rotary embedding with inverse frequencies base^(-i / (dim/2)) and the
    angle table [theta, theta] over the head dimension (modules/rope.py)."""

    def __init__(self, dim: int, base: float = 10000):
        super().__init__()
        assert dim % 2 == 0
        self.dim, self.base = dim, base
        half = dim // 2
        inv_freq = 1.0 / (base ** (torch.arange(0, half, dtype=torch.float32) / half))
        self.register_buffer("inv_freq", inv_freq, persistent=False)
        # fp32 copy kept outside Module.to(): casting the model to bf16 casts
        # the buffer too, and bf16 frequencies put the angle off by radians at
        # positions in the thousands
        self._inv_fp32 = {}

    def freqs(self, device) -> torch.Tensor:
        """The inverse frequencies in fp32 on `device` (computed once per device)."""
        key = str(device)
        if key not in self._inv_fp32:
            half = self.dim // 2
            f = 1.0 / (self.base ** (torch.arange(0, half, dtype=torch.float32) / half))
            self._inv_fp32[key] = f.to(device)
        return self._inv_fp32[key]

    def cos_sin(self, positions: torch.Tensor):
        ang = positions.to(torch.float32).unsqueeze(-1) * self.freqs(positions.device).unsqueeze(0)
        ang = torch.cat([ang, ang], dim=-1)
        return torch.cos(ang), torch.sin(ang)

    def forward(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, mode: str = "seq"):
        """mode "seq": q, k (batch, heads, seq_len, head_dim), positions (seq_len,);
        mode "pos": q, k (batch, heads, head_dim), positions (batch,)."""
        cos, sin = self.cos_sin(positions)
        if mode == "seq":
            cos, sin = cos[None, None], sin[None, None]
        else:
            cos, sin = cos[:, None], sin[:, None]
        return q * cos + _rotate_half(q) * sin, k * cos + _rotate_half(k) * sin

    def rotate_qk(self, q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor | None,
                  period: int):
        """q, k (..., heads, head_dim) on the GPU, rotated in one fused kernel
        and returned in bf16; row r of the leading dimensions at
        positions[r % period], or at r % period when positions is None."""
        return rope_qk(q, k, self.freqs(q.device), positions, period)


class SwiGLU(nn.Module):
    """out(w1(x) * silu(w2(x))) (modules/feed_forward.py)."""

    def __init__(self, dim: int, hidden_dim: int):
        super().__init__()
        self.w1 = Linear(dim, hidden_dim)
        self.w2 = Linear(dim, hidden_dim)
        self.out = Linear(hidden_dim, dim)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        a, c = project(x, [self.w1, self.w2])
        if (a.is_cuda and a.dtype == torch.bfloat16 and c.dtype == torch.bfloat16
                and a.numel() % 8 == 0
                and not (torch.is_grad_enabled() and (a.requires_grad or c.requires_grad))):
            return self.out(silu_mul(a, c))          # one fused kernel (inference)
        return self.out(a * F.silu(c))
