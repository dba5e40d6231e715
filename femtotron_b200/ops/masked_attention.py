"""Attention over whole sequences in which each row sees one interval of keys.

    x_ij = scale q_i k_j,  capped: x = softcap tanh(x / softcap),  with slopes: x -= slope_h |i - j|
    o_i  = sum over lo_i <= j < hi_i of softmax(x_i)_j v_j        (0 where the interval is empty)

``attention_mask`` makes the intervals, once for all layers of a step:

  documents  ``docs`` [batch, tokens]: a document is a run of equal numbers and sees itself only;
             rows with a negative number are padding, which sees nothing and is seen by nothing
             (its q, k, v and output gradient may hold anything), and has output and gradients 0
  causal     a row sees no later key, except that
  prefix     [batch, tokens] bool: the leading run of marked tokens of each document (a prompt) sees
             itself in both directions; marks behind an unmarked token of the document count for
             nothing
  window     keys less than ``window`` tokens away

``masked_attention`` is differentiable in q, k and v (``masked_attention_packed`` in one projection that holds
all three).  On CUDA it runs ``csrc/masked_attn*.cu`` on bf16 tensors of any strides with a head size that is
a multiple of 8 up to 128 (one that TMA does not take is copied first); its results and gradients are the same
bits every time, whatever stands in the places that a row does not see.  Only a NaN or an infinity of a token
that is no padding may reach, beside the rows that see it, the rows of the 128-row tiles that it lies in or is
seen from.  Between forward and backward pass it keeps q, k, v, o, what o's rounding to bf16 left out (as large
as o) and 4 bytes per row and head.  CPU tensors run the formulas in PyTorch (fp64 in fp64), where such a NaN may
reach any row of its sequence.

The reference has causal attention only, inside Hugging Face's layer
(femtotron/model/llama_partial_model.py:143-157).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from .ext import LAUNCHES, error_flag, native

TILE = 128
MAX_TOKENS = 262144
_NEVER = 2 ** 31 - 1
_NO_WINDOW = 2 ** 30


@dataclass
class AttentionMask:
    """``rows`` int32 [batch or 1, tokens rounded up to 128, 2]: the interval (lo, hi) of each row,
    (2^31 - 1, 0) where it sees nothing; ``tiles`` int32 [batch or 1, tiles, 4]: least and largest lo,
    least and largest hi of 128 rows each; ``order`` (CUDA) int32 [batch or 1, tiles]: the tiles as keys, the
    one that the most tiles look at first."""
    rows: torch.Tensor
    tiles: torch.Tensor
    seq_len: int
    order: torch.Tensor | None = None

    @property
    def batch(self) -> int:
        return self.rows.shape[0]


def attention_mask(batch: int, seq_len: int, *, causal: bool = True, window: int | None = None,
                   docs: torch.Tensor | None = None, prefix: torch.Tensor | None = None,
                   device=None) -> AttentionMask:
    """The intervals for ``batch`` sequences of ``seq_len`` tokens (see the top of this file).  A mask
    of one sequence serves every batch size."""
    if batch < 1 or not 1 <= seq_len <= MAX_TOKENS:
        raise ValueError(f"attention_mask: needs a batch of sequences of 1 to {MAX_TOKENS} tokens, got {batch} x {seq_len}")
    if window is not None and window < 1:
        raise ValueError(f"attention_mask: window must be at least 1, got {window}")
    if prefix is not None and not causal:
        raise ValueError("attention_mask: a prefix belongs to a causal mask")
    for name, x, types in (("docs", docs, (torch.int32, torch.int64)), ("prefix", prefix, (torch.bool,))):
        if x is None:
            continue
        if x.dtype not in types:
            raise TypeError(f"attention_mask: {name} must be {' or '.join(str(t) for t in types)}, got {x.dtype}")
        if tuple(x.shape) != (batch, seq_len):
            raise ValueError(f"attention_mask: {name} of shape {tuple(x.shape)} for [{batch}, {seq_len}]")
        want = torch.device(device) if device is not None else (docs if docs is not None else prefix).device
        if x.device.type != want.type or (want.index is not None and x.device.index != want.index):
            raise ValueError(f"attention_mask: {name} is on {x.device}, the mask on {want}")
    given = docs if docs is not None else prefix
    device = given.device if given is not None else torch.device(device if device is not None else "cpu")
    if device.type == "cuda":
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        docs, prefix = (x if x is None or x.stride(-1) == 1 else x.contiguous() for x in (docs, prefix))
        rows, tiles, order = native().attn_mask(batch, seq_len, causal, window or 0, docs, prefix, device)
        return AttentionMask(rows, tiles, seq_len, order)
    S = seq_len
    i = torch.arange(S).expand(batch, S)
    new = i == 0
    if docs is not None:
        new = new.clone()
        new[:, 1:] |= docs[:, 1:] != docs[:, :-1]
    first = torch.where(new, i, torch.zeros_like(i)).cummax(1).values
    stops = new
    leads = torch.zeros_like(new)
    if prefix is not None:
        plain = torch.where(prefix, torch.full_like(i, -1), i).cummax(1).values
        leads = plain < first
        stops = new | ~prefix
    after = torch.full((batch, S + 1), S)
    after[:, :S] = torch.where(stops, i, torch.full_like(i, S))
    stop = after.flip(1).cummin(1).values.flip(1)[:, 1:]
    hi = torch.where(leads, stop, i + 1) if causal else stop
    w = min(window or _NO_WINDOW, _NO_WINDOW)
    lo, hi = torch.maximum(first, i - w + 1), torch.minimum(hi, i + w)
    if docs is not None:
        lo, hi = lo.masked_fill(docs < 0, _NEVER), hi.masked_fill(docs < 0, 0)
    nt = (S + TILE - 1) // TILE
    rows = torch.zeros(batch, nt * TILE, 2, dtype=torch.int32)
    rows[..., 0] = _NEVER
    rows[:, :S] = torch.stack([lo, hi], -1).int()
    t = rows.view(batch, nt, TILE, 2)
    tiles = torch.stack([t[..., 0].amin(-1), t[..., 0].amax(-1), t[..., 1].amin(-1), t[..., 1].amax(-1)], -1)
    return AttentionMask(rows, tiles.contiguous(), S)


def document_ids(input_ids: torch.Tensor, separator: int) -> torch.Tensor:
    """Numbers of the documents of packed rows [batch, tokens]: each ends with a ``separator`` token."""
    ends = input_ids == separator
    return (ends.cumsum(-1) - ends.long()).int()


def alibi_slopes(heads: int, device=None) -> torch.Tensor:
    """Slopes 2^(-8 i / n) for i = 1 ... n of the bias of distance, fp32; for a number of heads that is no
    power of two, those of the next lower power and every other one of the next higher.  On CUDA the host waits
    for the stream, except while a graph is captured, which then holds a kernel per head: keep the tensor."""
    n = 2 ** int(math.log2(heads))
    slopes = [2.0 ** (-8.0 * i / n) for i in range(1, n + 1)]
    slopes += [2.0 ** (-4.0 * i / n) for i in range(1, 2 * (heads - n), 2)]
    if device is not None and torch.device(device).type == "cuda" and torch.cuda.is_current_stream_capturing():
        out = torch.empty(heads, dtype=torch.float32, device=device)
        for i, s in enumerate(slopes):
            out[i].fill_(s)
        return out
    return torch.tensor(slopes, dtype=torch.float32, device=device)


def _visible(mask: AttentionMask) -> torch.Tensor:
    """[batch or 1, S, S] bool."""
    S = mask.seq_len
    lo, hi = mask.rows[:, :S, 0, None], mask.rows[:, :S, 1, None]
    j = torch.arange(S)
    return (j >= lo) & (j < hi)


def _forward_cpu(q, k, v, mask, scale, softcap, slopes):
    B, S, nq, d = q.shape
    nkv = k.shape[2]
    vis = _visible(mask)[:, None]
    dead = mask.rows[:, :S, 1] == 0
    wide = torch.promote_types(q.dtype, torch.float32)
    qf, kf, vf = (x.to(wide).masked_fill(dead[:, :, None, None], 0.0).transpose(1, 2) for x in (q, k, v))
    kf, vf = kf.repeat_interleave(nq // nkv, 1), vf.repeat_interleave(nq // nkv, 1)
    x = qf @ kf.transpose(-1, -2) * scale
    keep = None
    if softcap:
        t = torch.tanh(x / softcap)
        x, keep = softcap * t, 1 - t * t
    if slopes is not None:
        i = torch.arange(S)
        x = x - slopes.to(wide).view(1, nq, 1, 1) * (i[:, None] - i).abs()
    x = x.masked_fill(~vis, float("-inf"))
    lse = torch.logsumexp(x, -1)
    p = torch.where(vis, torch.exp(x - lse[..., None]), torch.zeros_like(x))
    return qf, kf, vf, keep, lse, p


def _forward(ctx, q, k, v, mask, scale, softcap, slopes, graded, *kept):
    if q.is_cuda:
        o, lse, low = native().masked_attn_fwd(q, k, v, mask.rows, mask.tiles, mask.order, scale, softcap, slopes,
                                               graded, error_flag(q.device))
    else:
        *_, vf, _, lse, p = _forward_cpu(q, k, v, mask, scale, softcap, slopes)
        o, low = (p @ vf).transpose(1, 2).to(q.dtype).contiguous(), None
    if graded:
        ctx.save_for_backward(*kept, o, low, lse, mask.rows, mask.tiles, mask.order, slopes)
        ctx.meta = (mask.seq_len, scale, softcap)
    return o


class MaskedAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, scale, softcap, slopes, graded):
        return _forward(ctx, q, k, v, mask, scale, softcap, slopes, graded, q, k, v)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, low, lse, rows, tiles, order, slopes = ctx.saved_tensors
        dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
        _backward(q, k, v, o, low, do, lse, rows, tiles, order, slopes, ctx.meta, dq, dk, dv)
        return dq, dk, dv, None, None, None, None, None


def _heads(qkv, nq, nkv):
    return qkv[:, :, :nq], qkv[:, :, nq:nq + nkv], qkv[:, :, nq + nkv:nq + 2 * nkv]


class MaskedAttnPackedFn(torch.autograd.Function):
    """MaskedAttnFn of one packed projection [batch, tokens, q heads | k heads | v heads, d], whose gradient
    comes back in one piece too."""

    @staticmethod
    def forward(ctx, qkv, nq, nkv, mask, scale, softcap, slopes, graded):
        ctx.heads = (nq, nkv)
        return _forward(ctx, *_heads(qkv, nq, nkv), mask, scale, softcap, slopes, graded, qkv)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        qkv, o, low, lse, rows, tiles, order, slopes = ctx.saved_tensors
        d = torch.empty_like(qkv, memory_format=torch.contiguous_format)
        _backward(*_heads(qkv, *ctx.heads), o, low, do, lse, rows, tiles, order, slopes, ctx.meta, *_heads(d, *ctx.heads))
        return d, None, None, None, None, None, None, None


def _backward(q, k, v, o, low, do, lse, rows, tiles, order, slopes, meta, dq, dk, dv):
    seq_len, scale, softcap = meta
    if q.is_cuda:
        n = native().masked_attn_bwd(q, k, v, o, low, do, lse, rows, tiles, order, scale, softcap, slopes, dq, dk, dv,
                                     error_flag(q.device))
        LAUNCHES[0] += n - 1  # the proxy counted one
        return
    mask = AttentionMask(rows, tiles, seq_len)
    B, S, nq, d = q.shape
    nkv = k.shape[2]
    qf, kf, vf, keep, _, p = _forward_cpu(q, k, v, mask, scale, softcap, slopes)
    g = do.to(p.dtype).masked_fill((rows[:, :S, 1] == 0)[:, :, None, None], 0.0).transpose(1, 2)
    dp = g @ vf.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    if keep is not None:
        ds = ds * keep

    def group(x):  # the query heads of a group share a key head
        return x.view(B, nkv, nq // nkv, S, d).sum(2).transpose(1, 2)
    dq.copy_((ds @ kf * scale).transpose(1, 2))
    dk.copy_(group(ds.transpose(-1, -2) @ qf * scale))
    dv.copy_(group(p.transpose(-1, -2) @ g))


def _check(q, k, v, mask, scale, softcap, slopes):
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("masked_attention: q, k, v must be [batch, tokens, heads, d]")
    if k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError(f"masked_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"masked_attention: {q.shape[2]} query heads do not share {k.shape[2]} key heads evenly")
    if not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"masked_attention: q, k, v are {q.dtype}, {k.dtype}, {v.dtype}")
    if not q.is_floating_point() or (q.is_cuda and q.dtype != torch.bfloat16):
        raise TypeError(f"masked_attention: bfloat16 tensors are required on CUDA (floating ones on the CPU), got {q.dtype}")
    if q.is_cuda and (q.shape[3] % 8 or not 8 <= q.shape[3] <= 128):
        raise ValueError(f"masked_attention: the head size must be a multiple of 8 up to 128 on CUDA, got {q.shape[3]}")
    for x in (k, v, mask.rows, mask.tiles, *([mask.order] if mask.order is not None else []), *([slopes] if slopes is not None else [])):
        if x.device != q.device:
            raise ValueError(f"masked_attention: all operands must be on one device, got {q.device} and {x.device}")
    if q.is_cuda and mask.order is None:
        raise ValueError("masked_attention: the mask must come from attention_mask, on CUDA")
    if mask.seq_len != q.shape[1] or mask.batch not in (1, q.shape[0]):
        raise ValueError(f"masked_attention: a mask of {mask.batch} x {mask.seq_len} for {q.shape[0]} x {q.shape[1]} tokens")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"masked_attention: scale must be positive, got {scale}")
    if not (softcap >= 0 and math.isfinite(softcap)) or (softcap and not 1e-30 < scale / softcap < 1e30):
        raise ValueError(f"masked_attention: softcap must be 0 (none) or positive, got {softcap} (and scale {scale})")
    if slopes is not None and (slopes.dtype != torch.float32 or tuple(slopes.shape) != (q.shape[2],)):
        raise ValueError(f"masked_attention: slopes must be one fp32 number per query head, got {slopes.dtype} "
                         f"{tuple(slopes.shape)}")


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: AttentionMask, *,
                     scale: float | None = None, softcap: float = 0.0, slopes: torch.Tensor | None = None) -> torch.Tensor:
    """Attention output [batch, tokens, heads, d] of q [batch, tokens, heads, d] and k, v [batch, tokens,
    key heads, d] (query head h uses key head h // (heads / key heads)).  ``scale``: 1 / sqrt(d) by
    default; ``softcap``: 0 for none; ``slopes``: fp32 [heads] of the bias of distance, not
    negative (they take no gradient).  A backward pass is of first order."""
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    softcap = float(softcap)
    _check(q, k, v, mask, scale, softcap, slopes)
    if q.numel() == 0:
        return torch.zeros_like(q) + 0 * (q.sum() + k.sum() + v.sum())
    graded = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    slopes = slopes.detach().contiguous() if slopes is not None else None
    return MaskedAttnFn.apply(q, k, v, mask, scale, softcap, slopes, graded)


def masked_attention_packed(qkv: torch.Tensor, heads: int, key_heads: int, mask: AttentionMask, *,
                            scale: float | None = None, softcap: float = 0.0,
                            slopes: torch.Tensor | None = None) -> torch.Tensor:
    """``masked_attention`` of a packed projection [batch, tokens, heads + 2 key_heads, d]."""
    if qkv.dim() != 4 or heads < 1 or key_heads < 1 or qkv.shape[2] != heads + 2 * key_heads:
        raise ValueError(f"masked_attention_packed: {tuple(qkv.shape)} does not hold {heads} + 2 x {key_heads} heads")
    scale = 1.0 / math.sqrt(qkv.shape[-1]) if scale is None else float(scale)
    softcap = float(softcap)
    _check(*_heads(qkv, heads, key_heads), mask, scale, softcap, slopes)
    if qkv.numel() == 0:
        return torch.zeros_like(qkv[:, :, :heads]) + 0 * qkv.sum()
    graded = torch.is_grad_enabled() and qkv.requires_grad
    slopes = slopes.detach().contiguous() if slopes is not None else None
    return MaskedAttnPackedFn.apply(qkv, heads, key_heads, mask, scale, softcap, slopes, graded)
