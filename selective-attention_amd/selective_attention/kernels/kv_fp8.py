"""Launchers of the paged KV cache held in 8 bits (csrc/kv_fp8.hip,
csrc/attention_fp8.hip; no counterpart in the reference, whose caches keep the
model's dtype, inference/selective_attn_cache.py:3-42).

A block is one page of one kv head.  Full blocks are e4m3 codes with one
power-of-two scale a block; a row's open block (the seq_len % page_size tokens
behind its last full page) stays in bfloat16 until it is full.
"""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .attention import _i32, _rows16
from .common import call_on, require_one_device

FP8 = torch.float8_e4m3fn
PAGE_SIZES = (64, 128)
HEAD_DIMS = (64, 128)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(b, Hq, Hkv, D, ps, max_pages):
    return _lib.load().sa_paged_decode_fp8_workspace_size(b, Hq, Hkv, D, ps, max_pages)


def _check_cache(who, batch, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail, page_table,
                 gate_pages, written):
    """Shapes and dtypes of the cache's tensors; `written`: the call writes them,
    so none may be copied on the way."""
    if k_pages.dim() != 4:
        raise ValueError(f"{who}: k_pages must be (num_pages, kv_heads, page_size, head_dim)")
    n, H, ps, D = k_pages.shape
    if ps not in PAGE_SIZES or D not in HEAD_DIMS:
        raise ValueError(f"{who}: page_size {ps} must be one of {PAGE_SIZES} and head_dim {D} one "
                         f"of {HEAD_DIMS}")
    if n == 0 or H == 0:
        raise ValueError(f"{who}: empty page pool")
    # (one plain chain where all is well: a loop over names costs more than a launch)
    sh, f32 = (n, H), torch.float32
    gates_ok = gate_pages is None or (gate_pages.shape == (n, H, ps) and gate_pages.dtype == f32
                                      and gate_pages.is_contiguous() and not gate_pages.data_ptr() % 16)
    if not (gates_ok and v_pages.shape == (n, H, D, ps) and k_scale.shape == sh == v_scale.shape
            and k_tail.shape == (batch, H, ps, D) and v_tail.shape == (batch, H, D, ps)
            and k_pages.dtype == FP8 == v_pages.dtype and k_scale.dtype == f32 == v_scale.dtype
            and k_tail.dtype == torch.bfloat16 == v_tail.dtype
            and k_pages.is_contiguous() and v_pages.is_contiguous() and k_scale.is_contiguous()
            and v_scale.is_contiguous() and k_tail.is_contiguous() and v_tail.is_contiguous()
            and not (k_pages.data_ptr() | v_pages.data_ptr() | k_scale.data_ptr()
                     | v_scale.data_ptr() | k_tail.data_ptr() | v_tail.data_ptr()) % 16):
        want = [("k_pages", k_pages, (n, H, ps, D), FP8), ("v_pages", v_pages, (n, H, D, ps), FP8),
                ("k_scale", k_scale, sh, f32), ("v_scale", v_scale, sh, f32),
                ("k_tail", k_tail, (batch, H, ps, D), torch.bfloat16),
                ("v_tail", v_tail, (batch, H, D, ps), torch.bfloat16)]
        if gate_pages is not None:
            want.append(("gate_pages" if written else "key_bias", gate_pages, (n, H, ps), f32))
        for name, t, shape, dtype in want:
            if t.shape != shape:
                raise ValueError(f"{who}: {name} must be {shape}, got {tuple(t.shape)}")
            if t.dtype != dtype:
                raise TypeError(f"{who}: {name} must be {dtype}, got {t.dtype}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{who}: {name} must be contiguous on a 16-byte boundary")
    if page_table.dim() != 2 or page_table.shape[0] != batch:
        raise ValueError(f"{who}: page_table must be ({batch}, max_pages), got {tuple(page_table.shape)}")
    return n, H, ps, D


def paged_decode_attn_fp8(q, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail, page_table,
                          seq_lens, softmax_scale=None, key_bias=None):
    """
    Args:
        q: (batch, num_q_heads, head_dim) bfloat16; query head h reads kv head
            h // (num_q_heads // num_kv_heads), at most 16 of them one
        k_pages: (num_pages, num_kv_heads, page_size, head_dim) float8_e4m3fn
        v_pages: (num_pages, num_kv_heads, head_dim, page_size) float8_e4m3fn
        k_scale, v_scale: (num_pages, num_kv_heads) float32 powers of two
        k_tail: (batch, num_kv_heads, page_size, head_dim) bfloat16, the rows'
            open blocks; v_tail: (batch, num_kv_heads, head_dim, page_size)
        page_table: (batch, max_pages) int32; invalid ids contribute no keys
        seq_lens: (batch,) int32 cached tokens per row
        softmax_scale: head_dim ** -0.5 when None
        key_bias: (num_pages, num_kv_heads, page_size) float32 or None: added to
            every key's score except the newest (position seq_len - 1); a key at
            -inf takes no part, whatever it holds (nor does one below some -2e38,
            whose score in powers of two passes float32)

    Returns:
        o: (batch, num_q_heads, head_dim) bfloat16; a row without keys gets zeros.
    """
    who = "paged_decode_attn_fp8"
    if q.dtype != torch.bfloat16:
        raise TypeError(f"{who}: q must be bfloat16, got {q.dtype}")
    b, Hq, D = q.shape
    n, Hkv, ps, _ = _check_cache(who, b, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail,
                                 page_table, key_bias, False)
    require_one_device(q, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail, page_table, seq_lens,
                   key_bias)
    q = _rows16(q)
    pt, sl = _i32(page_table), _i32(seq_lens)
    max_pages = pt.shape[1]
    if b == 0 or max_pages == 0:
        return torch.zeros_like(q)   # no row has a key
    nbytes = _workspace_bytes(b, Hq, Hkv, D, ps, max_pages)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=q.device) if nbytes else None
    o = torch.empty_like(q)
    scale = -1.0 if softmax_scale is None else float(softmax_scale)
    call_on(q, "sa_paged_decode_fp8_fwd", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            k_scale.data_ptr(), v_scale.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr(),
            pt.data_ptr(), sl.data_ptr(), _lib.ptr(key_bias), b, Hq, Hkv, D, ps, max_pages, n,
            scale, o.data_ptr(), _lib.ptr(ws), nbytes, _lib.stream_of(q))
    return o


def _dense(t, dtype):
    return t if t.dtype == dtype and t.is_contiguous() else t.to(dtype).contiguous()


def _lens_and_table(who, page_table, seq_lens, batch):
    for t, name in ((page_table, "page_table"), (seq_lens, "seq_lens")):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{who}: {name} must be a contiguous int32 tensor")
    if seq_lens.shape != (batch,):
        raise ValueError(f"{who}: seq_lens must be ({batch},), got {tuple(seq_lens.shape)}")
    if page_table.shape[1] == 0:
        raise ValueError(f"{who}: page_table has no columns")


def paged_kv_append_fp8(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale, v_scale,
                        k_tail, v_tail, gate_pages):
    """One token per row: k, v (batch, kv_heads, head_dim) into the rows' open
    blocks at slot seq_lens[row] % page_size, log_gate (batch, kv_heads) into the
    page's gates (both None for a cache without gates); a block that this fills
    is rounded into its page.  seq_lens (batch,) int32, below 2^27, advances in
    place; a row of length -1 is left as it is.  While the call runs the lengths
    carry marks in their bits 27 to 30: a reader on another stream waits for it."""
    who = "paged_kv_append_fp8"
    b, H, D = k.shape
    n, _, ps, _ = _check_cache(who, b, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail,
                               page_table, gate_pages, True)
    _lens_and_table(who, page_table, seq_lens, b)
    require_one_device(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale, v_scale,
                   k_tail, v_tail, gate_pages)
    if b == 0:
        return
    k, v = _dense(k, torch.bfloat16), _dense(v, torch.bfloat16)
    lg = None if log_gate is None else _dense(log_gate, torch.float32)
    call_on(k, "sa_paged_kv_append_fp8", k.data_ptr(), v.data_ptr(), _lib.ptr(lg),
            page_table.data_ptr(), seq_lens.data_ptr(), b, H, D, ps, page_table.shape[1], n,
            k_pages.data_ptr(), v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
            k_tail.data_ptr(), v_tail.data_ptr(), _lib.ptr(gate_pages), _lib.stream_of(k))


def paged_kv_build_fp8(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale, v_scale,
                       k_tail, v_tail, gate_pages):
    """A prompt's tokens: k, v (batch, kv_heads, seq_len, head_dim) bf16 (any
    strides with head_dim contiguous), log_gate (batch, kv_heads, seq_len) or
    None; tokens t < seq_lens[r] of row r go to its pages, full pages rounded,
    the rest to its open block.  Slots behind a row's tokens are zeros with -inf
    gates; what no token reaches stays as it was.  One launch."""
    who = "paged_kv_build_fp8"
    b, H, L, D = k.shape
    n, _, ps, _ = _check_cache(who, b, k_pages, v_pages, k_scale, v_scale, k_tail, v_tail,
                               page_table, gate_pages, True)
    _lens_and_table(who, page_table, seq_lens, b)
    require_one_device(k, v, log_gate, page_table, seq_lens, k_pages, v_pages, k_scale, v_scale,
                   k_tail, v_tail, gate_pages)
    if b == 0 or L == 0:
        return   # no tokens: no row has a page to write
    k = k.to(torch.bfloat16)
    v = v.to(torch.bfloat16)
    if (k.stride(3) != 1 or v.stride() != k.stride() or any(x % 8 for x in k.stride()[:3])
            or k.data_ptr() % 16 or v.data_ptr() % 16):
        k, v = (t.clone(memory_format=torch.contiguous_format) for t in (k, v))
    lg, gs = None, (0, 0, 0)
    if log_gate is not None:
        lg = log_gate.to(torch.float32)
        gs = lg.stride()
    call_on(k, "sa_paged_kv_build_fp8", _lib.ptr(k), _lib.ptr(v), k.stride(0), k.stride(2),
              k.stride(1), _lib.ptr(lg), gs[0], gs[1], gs[2], _lib.ptr(page_table),
              _lib.ptr(seq_lens), b, L, H, D, ps, page_table.shape[1], n, _lib.ptr(k_pages),
              _lib.ptr(v_pages), _lib.ptr(k_scale), _lib.ptr(v_scale), _lib.ptr(k_tail),
              _lib.ptr(v_tail), _lib.ptr(gate_pages), _lib.stream_of(k))
