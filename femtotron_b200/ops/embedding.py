"""Embedding lookup with a factor, and its gradient by sorted tokens.

    out_t = scale w[id_t - vstart]  (0 where the id is in another shard),
    dw[v] = scale sum over id_t = vstart + v of dout_t

The gradient's sums run over the tokens in the order of the batch, in fp32, cut where the sorted list
of tokens is cut into pieces of 32: no atomics, the same bits every time.  A word's pieces are summed beside one
another and joined one after the other, so a batch that is mostly one word takes longer (32768 tokens: three times as
long).  CUDA tensors run ``csrc/embedding.cu`` (fp32, bf16 or fp16; ids int32 or int64),
CPU tensors PyTorch (fp64 in fp64).  The autograd entry point is ``functional.embedding``.

The reference looks rows up with ``F.embedding`` and masks the ids of other shards
(femtotron/parallel/tensor_parallel/embedding.py:57-77).
"""
from __future__ import annotations

import torch

from .ext import LAUNCHES, native


def _local(ids: torch.Tensor, words: int, vstart: int):
    local = ids.reshape(-1).long() - vstart
    has = (local >= 0) & (local < words)
    return local, has


def _wide(*types: torch.dtype) -> torch.dtype:
    """What CPU tensors are computed in: fp32 for narrower types."""
    return torch.float64 if torch.float64 in types else torch.float32


def lookup(ids: torch.Tensor, table: torch.Tensor, vstart: int = 0, scale: float = 1.0) -> torch.Tensor:
    """Rows of ``table`` [words, values] times ``scale``, in its type."""
    if table.is_cuda:
        return native().embed_lookup(ids, table, int(vstart), float(scale))
    local, has = _local(ids, table.shape[0], vstart)
    if table.shape[0] == 0:
        return table.new_zeros(*ids.shape, table.shape[1])
    rows = table[local.masked_fill(~has, 0)]  # nothing here depends on the ids' values: tensors without data pass too
    rows = rows if scale == 1.0 else (rows.to(_wide(table.dtype)) * scale).to(table.dtype)
    return rows.masked_fill(~has[:, None], 0).view(*ids.shape, table.shape[1])


def sorted_grad(ids: torch.Tensor, dout: torch.Tensor, dst: torch.Tensor, accumulate: bool, vstart: int = 0,
                scale: float = 1.0) -> None:
    """Store the table's gradient in ``dst`` [words, values], or add it (contiguous fp32, bf16 or fp16: rounded once;
    others by way of an fp32 copy)."""
    dout = dout.reshape(ids.numel(), dst.shape[1])
    if dst.is_cuda:
        direct = dst.is_contiguous() and dst.dtype in (torch.float32, torch.bfloat16, torch.float16)
        to = dst if direct else torch.empty(dst.shape, dtype=torch.float32, device=dst.device)
        n = native().embed_sorted_grad(ids, dout, to, accumulate and direct, int(vstart), float(scale))
        LAUNCHES[0] += n - 1
        if not direct:  # a buffer of other strides or another type
            dst.add_(to) if accumulate else dst.copy_(to)
        return
    local, has = _local(ids, dst.shape[0], vstart)
    g = torch.zeros(dst.shape, dtype=_wide(dst.dtype, dout.dtype))
    g.index_add_(0, local[has], dout[has].to(g.dtype))
    g = g if scale == 1.0 else g * scale
    dst.copy_(dst.to(g.dtype) + g if accumulate else g)
