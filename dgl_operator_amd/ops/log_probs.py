"""Log probabilities of given classes, with entropy and the best alternatives.

``log_probs`` is what a classifier, a link-prediction ranking over entities or a
mixture-of-experts router answers with: the log probability of each row's target
(its negative mean is the cross entropy), the entropy of the row's distribution,
and the log probabilities and indices of its best classes. All three are
differentiable together in one pass. GPU: HIP kernels (csrc/log_probs.hip) that
read the logits once; CPU: plain PyTorch.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import backend


class LogProbs(NamedTuple):
    """log_prob [...] (None without a target), entropy [...],
    top_log_prob [..., top_k] falling, top_index int64 [..., top_k]."""

    log_prob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_log_prob: torch.Tensor
    top_index: torch.Tensor


def _fwd_ref(logits, target, top_k, ignore_index):
    z = logits if logits.dtype == torch.float64 else logits.float()
    m = z.amax(1, keepdim=True)
    none = m == -math.inf
    d = z - torch.where(none, 0.0, m)
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    logs = torch.where(none, 0.0, torch.log(s))
    a = torch.where(e == 0, 0.0, d * e).sum(1, keepdim=True)
    entropy = torch.where(none, 0.0, logs - a / torch.where(none, 1.0, s))
    logp = d - logs
    lp = None
    if target is not None:
        C = z.shape[1]
        inside = (target >= 0) & (target < C)
        t = torch.where(inside, target, 0).unsqueeze(1)
        lp = torch.where(inside, logp.gather(1, t)[:, 0], math.nan)
        lp = torch.where(target == ignore_index, 0.0, lp)
    # a stable sort: of equal logits the lowest index comes first, NaN leads
    index = torch.sort(z, dim=1, descending=True, stable=True).indices
    index = index[:, :top_k].contiguous()
    return lp, entropy[:, 0], logp.gather(1, index), index, logp, none


def _bwd_ref(logits, target, ignore_index, logp, none, entropy, index,
             g_lp, g_ent, g_top):
    p = torch.exp(logp)
    pull = torch.zeros_like(entropy)
    grad = torch.zeros_like(p)
    if g_lp is not None:
        inside = (target >= 0) & (target < p.shape[1])
        g = torch.where(inside, g_lp, math.nan)
        g = torch.where(target == ignore_index, 0.0, g)
        pull = pull + g
        grad.scatter_add_(1, torch.where(inside, target, 0).unsqueeze(1),
                          torch.where(inside, g, 0.0).unsqueeze(1))
    if g_top is not None:
        pull = pull + g_top.sum(1)
        grad.scatter_add_(1, index, g_top)
    rest = pull.unsqueeze(1)
    if g_ent is not None:
        rest = rest + g_ent.unsqueeze(1) * (
            torch.where(p == 0, 0.0, logp) + entropy.unsqueeze(1))
    grad = torch.where(none, 0.0, grad - p * rest)
    return grad.to(logits.dtype)


class _LogProbs(torch.autograd.Function):
    """CPU path; the GPU's is csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, logits, target, top_k, ignore_index):
        ctx.set_materialize_grads(False)
        ctx.ignore_index = ignore_index
        lp, ent, top, index, logp, none = _fwd_ref(
            logits, target, top_k, ignore_index)
        ctx.save_for_backward(logits, target, index, logp, ent, none)
        ctx.mark_non_differentiable(index)
        return lp, ent, top, index

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        logits, target, index, logp, ent, none = ctx.saved_tensors
        dz = _bwd_ref(logits, target, ctx.ignore_index, logp, none, ent, index,
                      g_lp, g_ent, g_top)
        return dz, None, None, None


def log_probs(
    logits: torch.Tensor,
    target: Optional[torch.Tensor] = None,
    top_k: int = 0,
    ignore_index: int = -100,
) -> LogProbs:
    """Log softmax of logits [..., C] at target [...], with the entropy and the
    top_k best classes of each row, all in fp32 (fp64 for fp64 on CPU).

    * target == ignore_index: log_prob 0 and no gradient from it. Any other
      target outside [0, C) gives NaN, in log_prob and in the row's gradient.
    * A logit of -inf takes its class away (a filtered answer): probability 0,
      nothing to the entropy. A row with no class left has log_prob and
      top_log_prob -inf, entropy 0 and gradient 0.
    * NaN or +inf in a row: its numbers are NaN.
    * Alternatives are ordered by logit, NaN first, ties by the lower index.
    * On GPU top_k is at most 32; logits are fp32, bf16 or fp16.

    The gradient has the logits' type; the index has none.
    """
    assert logits.dim() >= 1 and logits.is_floating_point(), \
        "log_probs: floating point logits [..., C] expected"
    C = logits.shape[-1]
    lead = logits.shape[:-1]
    assert C >= 1, "log_probs: at least one class expected"
    assert 0 <= top_k <= C, f"log_probs: top_k must be in [0, {C}]"
    if target is not None:
        assert target.shape == lead, \
            f"log_probs: target must be {tuple(lead)}, got {tuple(target.shape)}"
        assert target.device == logits.device, \
            "log_probs: target and logits are on different devices"
        assert not target.is_floating_point() and target.dtype != torch.bool, \
            "log_probs: integer targets expected"
        target = target.reshape(-1).long().contiguous()
    rows = 1
    for d in lead:
        rows *= d
    flat = logits if logits.dim() == 2 else logits.reshape(rows, C)
    if logits.is_cuda:
        ext = backend.ext_for(logits)
        ent, top, index, *lp = ext.log_probs(flat, target, top_k, ignore_index)
        lp = lp[0] if lp else None
    else:
        lp, ent, top, index = _LogProbs.apply(flat, target, top_k, ignore_index)
    if len(lead) != 1:
        lp = lp.view(lead) if lp is not None else None
        ent = ent.view(lead)
        top = top.view(lead + (top_k,))
        index = index.view(lead + (top_k,))
    return LogProbs(lp, ent, top, index)
