"""The paged KV cache held in 8 bits: the decode attention that reads it and the
two writes that fill it (see kernels/kv_fp8.py for the layout).

New ops (the reference's caches keep the model's dtype,
inference/selective_attn_cache.py:3-42).  Shape and dtype errors raise before
any launch.
"""
from __future__ import annotations

import math

import torch

from ..kernels import kv_fp8 as _k
from ..utils import check_ndim, check_shape


def paged_decode_attn_fp8(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                          k_scale: torch.Tensor, v_scale: torch.Tensor, k_tail: torch.Tensor,
                          v_tail: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
                          softmax_scale: float | None = None,
                          key_bias: torch.Tensor | None = None) -> torch.Tensor:
    if q.dim() != 3 or k_pages.dim() != 4:
        check_ndim(q, 3, name="q")
        check_ndim(k_pages, 4, name="k_pages")
    b, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    if k_pages.shape[3] != D:
        raise ValueError(f"[k_pages] Shape mismatch: expected head_dim {D}, got {k_pages.shape[3]}")
    if Hkv == 0 or Hq % Hkv or Hq // Hkv > 16:
        raise ValueError(f"num_q_heads {Hq} must be a multiple of num_kv_heads {Hkv}, at most 16 times it")
    check_shape(seq_lens, (b,), name="seq_lens")
    if softmax_scale is not None and not 0.0 < softmax_scale < math.inf:
        raise ValueError(f"softmax_scale must be positive and finite, got {softmax_scale}")
    return _k.paged_decode_attn_fp8(q, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail,
                                    page_table, seq_lens, softmax_scale, key_bias)


def paged_kv_append_fp8(k: torch.Tensor, v: torch.Tensor, log_gate: torch.Tensor | None,
                        page_table: torch.Tensor, seq_lens: torch.Tensor, k_pages: torch.Tensor,
                        v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                        k_tail: torch.Tensor, v_tail: torch.Tensor,
                        gate_pages: torch.Tensor | None) -> None:
    ks, ps = k.shape, k_pages.shape
    if not (len(ks) == 3 and len(ps) == 4 and ks[1] == ps[1] and ks[2] == ps[3] and v.shape == ks
            and (log_gate is None or log_gate.shape == ks[:2])):
        check_ndim(k, 3, name="k")
        check_ndim(k_pages, 4, name="k_pages")
        check_shape(k, (ks[0], ps[1], ps[3]), name="k")
        check_shape(v, tuple(ks), name="v")
        check_shape(log_gate, tuple(ks[:2]), name="log_gate", optional=True)
    if (log_gate is None) != (gate_pages is None):
        raise ValueError("log_gate and gate_pages go together: give both or neither")
    _k.paged_kv_append_fp8(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale,
                           v_scale, k_tail, v_tail, gate_pages)


def paged_kv_build_fp8(k: torch.Tensor, v: torch.Tensor, log_gate: torch.Tensor | None,
                       page_table: torch.Tensor, seq_lens: torch.Tensor, k_pages: torch.Tensor,
                       v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                       k_tail: torch.Tensor, v_tail: torch.Tensor,
                       gate_pages: torch.Tensor | None) -> None:
    check_ndim(k, 4, name="k")
    check_ndim(k_pages, 4, name="k_pages")
    b, _, L, _ = k.shape
    check_shape(k, (b, k_pages.shape[1], L, k_pages.shape[3]), name="k")
    check_shape(v, tuple(k.shape), name="v")
    check_shape(log_gate, tuple(k.shape[:3]), name="log_gate", optional=True)
    if (log_gate is None) != (gate_pages is None):
        raise ValueError("log_gate and gate_pages go together: give both or neither")
    _k.paged_kv_build_fp8(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale, v_scale,
                          k_tail, v_tail, gate_pages)
