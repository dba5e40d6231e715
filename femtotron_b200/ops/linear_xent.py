"""Softmax cross entropy of a linear head, ``x = h w^T``, without the logits in memory.

    lse_t = log sum_j exp x_tj,   loss_t = lse_t - x_t,label     (0 where the label is ignored)
    d_tj  = g_t (exp(x_tj - lse_t) - [j = label_t]),   dh = d w,   dw = d^T h

The forward keeps one fp32 number per row (``lse``); the backward computes the product again
and works through the vocabulary in pieces, so that ``d`` and the partial sums of dh stay within
``workspace_bytes`` beside one fp32 sum of dh.  CUDA tensors (bf16) run
``csrc/linear_xent.cu``, which keeps the logits in fp32 (the head that stores them rounds them
to bf16); CPU tensors run the same pieces in PyTorch.  Where the bf16 logits of a batch are
smaller than the workspace, a smaller ``workspace_bytes`` keeps the backward below them.
The autograd entry point is ``functional.linear_cross_entropy``.

The reference computes ``F.cross_entropy`` on full-vocab logits gathered over TP
(femtotron/model/llama.py:91-111).
"""
from __future__ import annotations

import torch

from .ext import LAUNCHES, error_flag, native

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
WORKSPACE_BYTES = 256 * 2 ** 20


def _pieces(T: int, V: int, workspace_bytes: int):
    step = max(256, workspace_bytes // (2 * T) // 256 * 256)
    return [(v, min(v + step, V)) for v in range(0, V, step)]


def forward(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, vstart: int, ignore_index: int,
            reduction: str, workspace_bytes: int = WORKSPACE_BYTES, graded: bool = True):
    """(stats [T, 4], lse [T], losses [T], loss, gradient factor); the last two are None for "none".
    Stats: the largest logit and the sum of exponentials over this shard without the label, the
    label's logit in fp32 and as the kernels' accumulator has it (0 and -inf where the label is
    not in this shard).
    ``graded=False``: no backward will use lse, so one or two rows may be computed another way."""
    reduce = REDUCTIONS[reduction]
    if h.is_cuda:
        out = native().linear_xent_fwd(h, w, labels, vstart, ignore_index, reduce, graded, error_flag(h.device))
        LAUNCHES[0] += 2 if reduce else 1  # the proxy counted one
        return (*out, None, None) if reduce == 0 else tuple(out)
    T, V = h.shape[0], w.shape[0]
    m = torch.full((T,), float("-inf"))
    s, tgt = torch.zeros(T), torch.zeros(T)
    local = labels - vstart
    for a, b in _pieces(T, V, workspace_bytes):
        x = h.float() @ w[a:b].float().t()
        rows = torch.nonzero((local >= a) & (local < b))[:, 0]
        tgt[rows] = x[rows, local[rows] - a]
        x[rows, local[rows] - a] = float("-inf")
        nm = torch.maximum(m, x.max(-1).values)
        base = torch.where(nm == float("-inf"), torch.zeros_like(nm), nm)
        s = s * torch.exp(m - base) + torch.exp(x - base[:, None]).sum(-1)
        m = nm
    has = (local >= 0) & (local < V)
    stats = torch.stack([m, s, tgt, torch.where(has, tgt, torch.full_like(tgt, float("-inf")))], 1)
    return stats, *combine(stats, labels, ignore_index, reduction)


def combine(stats: torch.Tensor, labels: torch.Tensor, ignore_index: int, reduction: str):
    """(lse, losses, loss, gradient factor) of whole-vocabulary stats.  A loss is
    log(1 + sum over the other words of exp(x_j - label's logit)), never below 0."""
    top, sums, tgt, at = stats.unbind(1)
    log_s = torch.log(sums)
    lse = torch.logaddexp(top + log_s, at)
    valid = labels != ignore_index
    # a label that no column answers to has no probability: its loss is not a number (nor is an
    # infinite logit's)
    has = ((at != float("-inf")) | (tgt != 0)) & (tgt != float("inf"))
    losses = torch.logaddexp((top - tgt) + log_s, torch.zeros_like(tgt))
    losses = torch.where(has, losses, torch.full_like(lse, float("nan")))
    losses = torch.where(valid, losses, torch.zeros_like(lse))
    if reduction == "none":
        return lse, losses, None, None
    if reduction == "sum":
        return lse, losses, losses.sum(), torch.ones((), device=lse.device)
    n = valid.sum().float()
    return lse, losses, losses.sum() / n, torch.where(n > 0, 1 / n, torch.zeros_like(n))


def merge_shards(stats: torch.Tensor) -> torch.Tensor:
    """Stats of the vocabulary shards [world, T, 4] as those of the whole vocabulary."""
    m = stats[..., 0].max(0).values
    base = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    s = (stats[..., 1] * torch.exp(stats[..., 0] - base)).sum(0)
    return torch.stack([m, s, stats[..., 2].sum(0), stats[..., 3].max(0).values], 1)


def backward(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, lse: torch.Tensor, grad: torch.Tensor,
             factor: torch.Tensor, dh: torch.Tensor | None, dw: torch.Tensor | None, accumulate: bool, vstart: int,
             ignore_index: int, workspace_bytes: int = WORKSPACE_BYTES) -> None:
    """Write dh [T, H] and dw [V, H] (stored, or added where ``accumulate``).  ``grad``: the
    fp32 gradient of the loss (0-d, times ``factor``) or of each row's."""
    if h.is_cuda:
        n = native().linear_xent_bwd(h, w, labels, lse, grad, factor, dh, dw, accumulate, vstart, ignore_index,
                                     workspace_bytes, error_flag(h.device))
        LAUNCHES[0] += n - 1
        return
    g = grad if grad.dim() else grad * factor
    g = torch.where(labels == ignore_index, torch.zeros_like(lse), g.expand_as(lse))
    local = labels - vstart
    acc = torch.zeros(h.shape)
    for a, b in _pieces(h.shape[0], w.shape[0], workspace_bytes):
        wf = w[a:b].float()
        d = torch.exp(h.float() @ wf.t() - lse[:, None])
        rows = torch.nonzero((local >= a) & (local < b))[:, 0]
        d[rows, local[rows] - a] -= 1.0
        d = torch.where(g[:, None] == 0, torch.zeros_like(d), d * g[:, None])
        if dw is not None:
            part = d.t() @ h.float()
            dw[a:b] = (dw[a:b].float() + part if accumulate else part).to(dw.dtype)
        if dh is not None:
            acc += d @ wf
    if dh is not None:
        dh.copy_(acc)
