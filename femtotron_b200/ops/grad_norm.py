"""Global norm over many gradients, and the gradients clipped by it.

    norm = sqrt(sum over all tensors of x^2),    y = x min(1, max_norm / (norm + 1e-6))

``clip_grads`` does both for gradients that one process holds whole; ``sum_of_squares`` and
``scale_grads`` are its halves, for sums that cross process groups in between
(``training.grad_transform.ClipGradNorm``).  fp32, bf16 and fp16 tensors may be mixed, in any number,
shape and strides.  The sums end in fp64, so no square over- or underflows, and their order depends
on the tensors' sizes and 16-byte alignment alone: the same gradients give the same bits.  Nothing comes back to the host.
A norm that is not finite clips as ``torch.nn.utils.clip_grad_norm_`` does: an infinite one by 0, a
NaN by NaN.

CUDA tensors run ``csrc/grad_norm.cu``, CPU tensors PyTorch.  The reference squares and adds tensor by
tensor in fp32 (femtotron/training/grad_transform.py:13-76).
"""
from __future__ import annotations

import math

import torch

from .ext import LAUNCHES, native

TABLE = 1024  # tensors that one launch takes
MAX_SLOTS = 8


def _tables(tensors) -> int:
    return (len(tensors) + TABLE - 1) // TABLE


def _check(op: str, tensors) -> None:
    for t in tensors:
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16) and (t.is_cuda or not t.is_floating_point()):
            raise TypeError(f"{op}: fp32, bf16 or fp16 tensors are required, got {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError(f"{op}: all tensors must be on one device, got {tensors[0].device} and {t.device}")


def _check_out(op: str, tensors, out) -> None:
    if len(out) != len(tensors):
        raise ValueError(f"{op}: {len(tensors)} tensors and {len(out)} outputs")
    for t, o in zip(tensors, out):
        if o.shape != t.shape or o.dtype != t.dtype or o.device != t.device:
            raise ValueError(f"{op}: an output of {o.dtype} {tuple(o.shape)} for {t.dtype} {tuple(t.shape)}")


def sum_of_squares(tensors, slots=None, n_slots: int = 1) -> torch.Tensor:
    """fp64 [n_slots]: the sums of squares of the tensors of each slot (``slots``: one number per tensor,
    by default all 0)."""
    tensors = list(tensors)
    slots = [0] * len(tensors) if slots is None else [int(s) for s in slots]
    if len(slots) != len(tensors):
        raise ValueError(f"sum_of_squares: {len(tensors)} tensors and {len(slots)} slots")
    if not 1 <= n_slots <= MAX_SLOTS or any(not 0 <= s < n_slots for s in slots):
        raise ValueError(f"sum_of_squares: slots must be in [0, {n_slots}), of 1 to {MAX_SLOTS}")
    if not tensors:
        return torch.zeros(n_slots, dtype=torch.float64)
    if tensors[0].is_cuda:  # (the entry points check all of this again, so it is not done twice)
        LAUNCHES[0] += _tables(tensors)  # and one that the proxy counts
        return native().grad_sumsq(tensors, slots, n_slots)
    _check("sum_of_squares", tensors)
    out = torch.zeros(n_slots, dtype=torch.float64)
    for t, s in zip(tensors, slots):
        out[s] += t.detach().double().pow(2).sum()
    return out


def _check_written(tensors) -> None:
    for t in tensors:
        if t.numel() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise RuntimeError("more than one element of a tensor that is written refers to a single memory location")


def _scale_cpu(tensors, coef, out) -> None:
    for t, o in zip(tensors, tensors if out is None else out):
        o.copy_((t.float() * coef).to(t.dtype) if t.dtype != torch.float64 else t * coef)


@torch.no_grad()
def scale_grads(tensors, coef: torch.Tensor, out=None) -> None:
    """The tensors times ``coef`` (one fp32 number on their device), each rounded once: in place, or
    into ``out``.  No two tensors that are written may share memory (nor one that is written and another
    one that is read)."""
    tensors = list(tensors)
    out = None if out is None else list(out)
    coef = coef.detach().reshape(())
    if tensors and tensors[0].is_cuda and (out is None or out):
        LAUNCHES[0] += _tables(tensors) - 1
        native().grad_scale(tensors, coef, out or [])
        return
    if out is not None:
        _check_out("scale_grads", tensors, out)
    _check("scale_grads", tensors)
    _check_written(tensors if out is None else out)
    _scale_cpu(tensors, coef, out)


@torch.no_grad()
def clip_grads(grads, max_norm: float, out=None) -> torch.Tensor:
    """Clip ``grads`` to the global norm ``max_norm``, in place or into ``out``; returns the norm before
    (fp32, on their device)."""
    grads = list(grads)
    out = None if out is None else list(out)
    max_norm = float(max_norm)
    if not max_norm >= 0 or math.isinf(max_norm):
        raise ValueError(f"clip_grads: max_norm must be a number from 0 on, got {max_norm}")
    if grads and grads[0].is_cuda and (out is None or out):
        LAUNCHES[0] += 2 * _tables(grads) - 1
        return native().grad_clip(grads, max_norm, out or [])
    if out is not None:
        _check_out("clip_grads", grads, out)
    if not grads:
        return torch.zeros(())
    _check("clip_grads", grads)
    _check_written(grads if out is None else out)
    norm = sum_of_squares(grads)[0].sqrt().float()
    _scale_cpu(grads, (max_norm / (norm + 1e-6)).clamp(max=1.0), out)
    return norm
