"""Log probabilities of given tokens, the entropy of their distribution and its
largest alternatives, with the logits' gradient: what a decode step answers
with, what scoring a text needs, and (with a minus) a language model's loss.

New op (the reference takes softmax and argmax of its logits,
models/causal_lm.py:143-221, and leaves the loss to its caller).
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ..kernels import logprobs as _k
from ..kernels.common import in_forward_mode, needs_torch_ops
from ..utils import check_shape


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # (...) float32: log p of the given tokens
    entropy: torch.Tensor       # (...) float32: -sum p log p
    top_ids: torch.Tensor       # (..., top) int64, most probable first
    top_logprobs: torch.Tensor  # (..., top) float32


class TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, targets, top, ignore_index):
        lp, H, stats, ids, tl = _k.token_logprobs_forward(logits, targets, top, ignore_index)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, targets, H, stats, ids)
        ctx.top, ctx.ignore_index = top, ignore_index
        return lp, H, ids, tl

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_h, _, g_top):
        logits, targets, H, stats, ids = ctx.saved_tensors
        if g_lp is None and g_h is None and g_top is None:
            return None, None, None, None
        if needs_torch_ops(*(g for g in (g_lp, g_h, g_top) if g is not None)):
            raise RuntimeError("token_logprobs: the backward takes plain upstream gradients (no "
                               "batched ones, transforms or forward mode)")
        dx = _k.token_logprobs_backward(logits, targets, ctx.top, ctx.ignore_index, H, stats, ids,
                                        g_lp, g_h, g_top)
        return dx, None, None, None


def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, top: int = 0,
                   ignore_index: int = -100) -> TokenLogprobs:
    """
    Args:
        logits: (..., vocab) float32 or bfloat16 of any finite size; -inf rules a
            token out.  Read in place where the vocabulary is dense and one stride
            leads from row to row; others (logits[:, :-1] of a batch) are copied,
            in the forward and again in the backward: shift the targets and
            ignore the last place instead, as CausalLM.score does
        targets: (...) int32 or int64 token ids.  ignore_index: logprob 0 and no
            gradient from it, whatever the row holds; any other id outside the
            vocabulary: NaN
        top: alternatives a row, 0..64 and at most vocab; equal logits in the
            order of their ids
    Returns:
        TokenLogprobs, in float32; a row of -inf alone, or with NaN or +inf, gives
        NaN.  Differentiable once in logits (logprob, entropy and top_logprobs);
        the gradient has the logits' dtype.
    """
    if logits.dim() < 1 or not 0 < logits.shape[-1] <= _k.MAX_VOCAB:
        raise ValueError(f"token_logprobs: logits need a vocabulary of 1..{_k.MAX_VOCAB}, got "
                         f"{tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"token_logprobs: logits must be float32 or bfloat16, got {logits.dtype}")
    if targets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"token_logprobs: targets must be int32 or int64, got {targets.dtype}")
    check_shape(targets, tuple(logits.shape[:-1]), name="targets")
    if not 0 <= top <= min(_k.MAX_TOP, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top {top} must be 0..{_k.MAX_TOP} and at most the "
                         f"vocabulary {logits.shape[-1]}")
    top, ignore_index = int(top), int(ignore_index)
    if (torch.is_grad_enabled() and logits.requires_grad) or in_forward_mode():
        return TokenLogprobs(*TokenLogprobsFn.apply(logits, targets, top, ignore_index))
    lp, H, _, ids, tl = _k.token_logprobs_forward(logits, targets, top, ignore_index, False)
    return TokenLogprobs(lp, H, ids, tl)
