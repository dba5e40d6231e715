"""Rotary positions over all or part of each head, in half or interleaved layout, scaled for
long contexts.

``rotary_qk`` turns pair ``i`` of every head of a token at position ``p`` by the angle
``p * f_i``, from fp32 tables of its cosine and sine::

    a' = a c - b s,   b' = b c + a s          (``inverse``, the backward pass: s -> -s)

The half layout pairs values ``i`` and ``rot/2 + i`` of a head, the interleaved one values
``2i`` and ``2i + 1``; values from ``rot`` on are passed through.  ``rotary_tables`` makes the
tables in 64 bits and rounds them once to fp32, so positions in the hundred thousands keep an
exact angle (bf16 tables, or fp32 angles, do not).

``inv_frequencies`` gives the frequencies ``f_i`` for a Hugging Face style ``rope_scaling``
dict (keys ``rope_type`` or ``type``, ``factor`` and so on):

  default   f_i = theta^(-2i/rot)
  linear    f_i / factor (positions squeezed into the trained range)
  ntk       theta * factor^(rot / (rot - 2)): the lowest frequency is divided by the factor,
            the highest one stays; ``dynamic`` does this with the factor that the context
            length needs, factor * len / trained - (factor - 1), and not below the trained one
  llama3    by wavelength 2 pi / f: above trained / low_freq_factor divided by the factor,
            below trained / high_freq_factor kept, linear in trained / wavelength between
  yarn      linear in the pair index between the pairs that turn ``beta_fast`` and
            ``beta_slow`` times over the trained length: kept above, divided by the factor
            below; the tables are scaled by ``attention_factor``, by default 0.1 ln(factor) + 1

CUDA tensors run ``csrc/rotary.cu``; CPU tensors the same arithmetic in PyTorch.  The
reference has only the unscaled half layout, inside Hugging Face's layer
(femtotron/model/llama_partial_model.py:143-157).
"""
from __future__ import annotations

import math

import torch

from .ext import error_flag, native

SCALINGS = ("default", "linear", "ntk", "dynamic", "llama3", "yarn")


def inv_frequencies(rot: int, theta: float, scaling: dict | None = None, *, trained: int | None = None,
                    length: int | None = None) -> tuple[torch.Tensor, float]:
    """(frequencies [rot/2] in 64 bits, factor of the tables).  ``trained`` is the context
    length of training (the dict's ``original_max_position_embeddings`` wins over it),
    ``length`` the one to serve, for ``dynamic``."""
    if rot < 0 or rot % 2:
        raise ValueError(f"rotary: the rotated part of a head must be even, got {rot}")
    sc = dict(scaling or {})
    kind = sc.get("rope_type") or sc.get("type") or "default"
    if kind not in SCALINGS:
        raise ValueError(f"rotary: unknown rope_type {kind!r}; available: {SCALINGS}")
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    f = theta ** (-i / rot) if rot else i
    if kind == "default" or rot == 0:
        return f, 1.0
    for key in ("factor", "low_freq_factor", "high_freq_factor") if kind == "llama3" else ("factor",):
        if sc.get(key) is None:
            raise ValueError(f"rotary: {kind} scaling needs {key}, got {sc}")
    factor = float(sc["factor"])
    if factor < 1:
        raise ValueError(f"rotary: factor must be at least 1, got {factor}")
    if kind == "linear":
        return f / factor, 1.0
    trained = sc.get("original_max_position_embeddings") or trained
    if kind != "ntk" and not trained:
        raise ValueError(f"rotary: {kind} scaling needs original_max_position_embeddings")
    if kind in ("ntk", "dynamic"):
        if kind == "dynamic":
            factor = factor * max(length or trained, trained) / trained - (factor - 1)
        if rot == 2:
            return f, 1.0
        return (theta * factor ** (rot / (rot - 2))) ** (-i / rot), 1.0
    if kind == "llama3":
        lo, hi = float(sc["low_freq_factor"]), float(sc["high_freq_factor"])
        turns = trained * f / (2 * math.pi)
        kept = ((turns - lo) / (hi - lo)).clamp(0, 1) if hi > lo else (turns >= hi).to(f.dtype)
        return f * (kept + (1 - kept) / factor), 1.0
    fast, slow = float(sc.get("beta_fast") or 32), float(sc.get("beta_slow") or 1)

    def pair(turns: float) -> float:  # the pair that turns so often over the trained length
        return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))
    first, last = pair(fast), pair(slow)
    if sc.get("truncate", True):
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rot - 1)
    if first == last:
        last += 0.001
    kept = 1 - ((i / 2 - first) / (last - first)).clamp(0, 1)
    att = sc.get("attention_factor")
    if att is None:
        def grow(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1 if factor > 1 else 1.0
        ms, ma = sc.get("mscale"), sc.get("mscale_all_dim")
        att = grow(ms) / grow(ma) if ms and ma else grow(1.0)
    return f * (kept + (1 - kept) / factor), float(att)


def rotary_tables(rot: int, positions: int, theta: float = 10000.0, scaling: dict | None = None, *,
                  trained: int | None = None, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 cosine and sine tables [positions, rot/2]."""
    f, att = inv_frequencies(rot, theta, scaling, trained=trained, length=positions)
    angle = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), f.to(device))
    return (angle.cos() * att).float(), (angle.sin() * att).float()


def _check(q, k, cos, sin, pos):
    for name, t in (("q", q), ("k", k)):
        if t.dim() != 4:
            raise ValueError(f"rotary_qk: {name} must be [batch, tokens, heads, d], got {tuple(t.shape)}")
    if q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3] or q.dtype != k.dtype or q.device != k.device:
        raise ValueError("rotary_qk: q and k must agree in batch, tokens, d, dtype and device")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("rotary_qk: cos and sin must be fp32 tables [positions, rot/2] of one shape")
    if 2 * cos.shape[1] > q.shape[3]:
        raise ValueError(f"rotary_qk: {2 * cos.shape[1]} rotated values do not fit a head of {q.shape[3]}")
    if pos is None:
        if q.shape[1] > cos.shape[0]:
            raise ValueError(f"rotary_qk: {q.shape[1]} tokens, tables of {cos.shape[0]} positions")
        return None
    if pos.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"rotary_qk: positions must be int32 or int64, got {pos.dtype}")
    if pos.dim() == 1:
        pos = pos[None]
    if pos.dim() != 2 or pos.shape[1] != q.shape[1] or pos.shape[0] not in (1, q.shape[0]):
        raise ValueError(f"rotary_qk: positions of shape {tuple(pos.shape)} do not match "
                         f"[{q.shape[0]} or 1, {q.shape[1]}]")
    return pos


def _reach(x: torch.Tensor) -> int:
    """Elements from the first to the last one of x, or -1 where, going up the strides, a step does
    not clear what lies below it: then elements share memory."""
    reach = 0
    for st, n in sorted((st, n) for st, n in zip(x.stride(), x.shape) if n > 1):
        if st <= reach:
            return -1
        reach += st * (n - 1)
    return reach


def _written_twice(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q or k overlaps itself, or q and k, laid out alike, have an element in common (as
    written_twice of csrc/rotary.cu)."""
    if q.numel() == 0 or k.numel() == 0:
        return any(x.numel() and _reach(x) < 0 for x in (q, k))
    reach = [_reach(x) for x in (q, k)]
    if min(reach) < 0:
        return True
    apart, part = divmod(k.data_ptr() - q.data_ptr(), q.element_size())
    if apart > reach[0] or apart < -reach[1] or part:
        return False
    dims = []  # (stride, most steps of q, of k)
    for sq, sk, nq, nk in zip(q.stride(), k.stride(), q.shape, k.shape):
        if nq > 1 and nk > 1 and sq != sk:
            return False  # not laid out alike
        if nq > 1 or nk > 1:
            dims.append((sq if nq > 1 else sk, nq - 1, nk - 1))
    dims.sort(reverse=True)

    def meet(i: int, rest: int) -> bool:  # steps of q less steps of k that come to `rest`
        if i == len(dims):
            return rest == 0
        st, up, down = dims[i]
        below = sum(t * max(a, b) for t, a, b in dims[i + 1:])
        return any(meet(i + 1, rest - c * st)
                   for c in range(max(-down, -((below - rest) // st)), min(up, (rest + below) // st) + 1))
    return meet(0, apart)


def rotary_qk(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
              pos: torch.Tensor | None = None, *, interleaved: bool = False, inverse: bool = False,
              inplace: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Turned copies of q [B, S, nq, d] and k [B, S, nkv, d] (any strides with a unit inner
    one, so slices of a packed projection and heads-first tensors are taken as they are), or
    q and k themselves turned in place.  ``pos``: [B, S] or [S], by default 0, 1, ...

    On CUDA a position outside the tables gives NaN and is reported by
    ``check_kernel_errors`` (code 301); on the CPU it raises.  No autograd: ``rotary`` is the
    differentiable form.  In place, every element of q and k has to be one of its own."""
    if inplace and torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        raise ValueError("rotary_qk: in place on a tensor that autograd follows; use rotary()")
    if q.is_cuda:
        return native().rotary_qk(q, k, cos, sin, pos, interleaved, inverse, inplace, error_flag(q.device))
    pos = _check(q, k, cos, sin, pos)
    if inplace and _written_twice(q, k):
        raise RuntimeError("rotary_qk: in place on q and k that name an element more than once")
    if pos is None:
        pos = torch.arange(q.shape[1], device=q.device)[None]
    if pos.numel() and (int(pos.min()) < 0 or int(pos.max()) >= cos.shape[0]):
        raise IndexError(f"rotary_qk: position outside the tables of {cos.shape[0]} positions")
    c, s = cos[pos.long()][:, :, None], sin[pos.long()][:, :, None]
    s = -s if inverse else s
    r = cos.shape[1]
    out = []
    for x in (q, k):
        xf = x.float()
        y = x if inplace else x.clone(memory_format=torch.contiguous_format)
        if interleaved:
            a, b = xf[..., 0:2 * r:2], xf[..., 1:2 * r:2]
            ya, yb = y[..., 0:2 * r:2], y[..., 1:2 * r:2]
        else:
            a, b = xf[..., :r], xf[..., r:2 * r]
            ya, yb = y[..., :r], y[..., r:2 * r]
        na, nb = a * c - b * s, b * c + a * s
        ya.copy_(na)
        yb.copy_(nb)
        out.append(y)
    return out[0], out[1]


class RotaryFn(torch.autograd.Function):
    """Differentiable ``rotary_qk`` (the tables and positions take no gradient)."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, pos, interleaved):
        ctx.save_for_backward(cos, sin, pos if pos is not None else torch.empty(0))
        ctx.meta = (interleaved, pos is not None)
        return rotary_qk(q, k, cos, sin, pos, interleaved=interleaved)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, pos = ctx.saved_tensors
        interleaved, has = ctx.meta
        dq, dk = rotary_qk(dq, dk, cos, sin, pos if has else None, interleaved=interleaved, inverse=True)
        return dq, dk, None, None, None, None


def rotary(q, k, cos, sin, pos=None, *, interleaved=False):
    """Differentiable form of ``rotary_qk``."""
    return RotaryFn.apply(q, k, cos, sin, pos, interleaved)
