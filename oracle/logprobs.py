"""Oracle of the token log probabilities, in float64 on the CPU."""
from __future__ import annotations

import torch


def forward(x, targets, top=0, ignore_index=-100):
    """x (rows, V), targets (rows,) -> (logprob, entropy, top_ids, top_logprobs)."""
    x = x.double()
    V = x.shape[1]
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    ok = (targets >= 0) & (targets < V)
    lp = torch.where(ok, logp.gather(1, targets.clamp(0, V - 1)[:, None])[:, 0], float("nan"))
    lp = torch.where(targets == ignore_index, 0.0, lp)
    p = logp.exp()
    H = -torch.where(p == 0, 0.0, p * logp).sum(1)
    # the order of values (both zeros one), ties to the lowest id
    ids = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    return lp, H, ids, logp.gather(1, ids)


def backward(x, targets, g_lp=None, g_h=None, g_top=None, top=0, ignore_index=-100):
    """The gradient from its formula; upstream gradients (rows,), (rows,), (rows, top)."""
    x = x.double()
    rows, V = x.shape
    _, H, ids, _ = forward(x, targets, top, ignore_index)
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = logp.exp()
    a = torch.zeros(rows, V, dtype=torch.float64)
    if g_lp is not None:
        asked = targets != ignore_index
        g = torch.where(asked, g_lp.double(), 0.0)
        g = torch.where(asked & ((targets < 0) | (targets >= V)), float("nan"), g)
        a.scatter_add_(1, targets.clamp(0, V - 1)[:, None], g[:, None])
    if g_top is not None:
        a.scatter_add_(1, ids, g_top.double())
    d = a - p * a.sum(1, keepdim=True)
    if g_h is not None:
        d = d - g_h.double()[:, None] * (torch.where(p == 0, 0.0, p * logp) + p * H[:, None])
    return d
