"""Launchers of the token log probabilities (csrc/logprobs.hip; the reference
takes softmax and argmax of its logits, models/causal_lm.py:143-221)."""
from __future__ import annotations

import functools

import torch

from .. import _lib
from .common import act_dtype_code, call_on, require_one_device

MAX_TOP = 64
MAX_VOCAB = 1 << 28


def _rows(logits):
    """(rows, vocab) rows of logits whose last dimension is dense, in place where
    one stride leads from row to row."""
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _targets(t):
    if t.dim() == 1 and t.dtype == torch.int64 and t.is_contiguous():
        return t
    return t.reshape(-1).to(torch.int64).contiguous()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(rows, V, top):
    return _lib.load().sa_token_logprobs_workspace_size(rows, V, top)


def token_logprobs_forward(logits, targets, top, ignore_index, with_stats=True):
    """logits (..., vocab) float32 or bfloat16, targets (...) integers -> (logprob
    (...), entropy (...), stats (rows, 2) for the backward or None, top_ids
    (..., top) int64, top_logprobs (..., top) float32)."""
    require_one_device(logits, targets)
    dev = logits.device
    x = _rows(logits)
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()     # overlapping (expanded) rows
    rows, V = x.shape
    tg = _targets(targets)
    shape = logits.shape[:-1]
    f32 = torch.float32
    lp, H = torch.empty(shape, dtype=f32, device=dev), torch.empty(shape, dtype=f32, device=dev)
    stats = torch.empty((rows, 2), dtype=f32, device=dev) if with_stats else None
    ids = torch.empty((*shape, top), dtype=torch.int64, device=dev)
    tl = torch.empty((*shape, top), dtype=f32, device=dev)
    nbytes = _workspace_bytes(rows, V, top)
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev) if nbytes else None
    call_on(x, "sa_token_logprobs_fwd", act_dtype_code(x.dtype), x.data_ptr(), _stride(x),
            tg.data_ptr(), rows, V, top, ignore_index, lp.data_ptr(), H.data_ptr(),
            _lib.ptr(stats), ids.data_ptr(), tl.data_ptr(), _lib.ptr(ws), nbytes, _lib.stream_of(x))
    return lp, H, stats, ids, tl


def token_logprobs_backward(logits, targets, top, ignore_index, entropy, stats, top_ids, g_lp, g_h,
                            g_top):
    """The logits' gradient for the upstream gradients (None: zero)."""
    x = _rows(logits)
    if x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    rows, V = x.shape
    tg = _targets(targets)
    dx = torch.empty((rows, V), dtype=x.dtype, device=x.device)
    g = [None if t is None else t.to(torch.float32).contiguous() for t in (g_lp, g_h, g_top)]
    call_on(x, "sa_token_logprobs_bwd", act_dtype_code(x.dtype), _lib.ptr(x), _stride(x),
            _lib.ptr(tg), rows, V, top, int(ignore_index), _lib.ptr(entropy), _lib.ptr(stats),
            _lib.ptr(top_ids) if top else None, _lib.ptr(g[0]), _lib.ptr(g[1]),
            _lib.ptr(g[2]) if top else None, _lib.ptr(dx), V, _lib.stream_of(x))
    return dx.view(logits.shape)
