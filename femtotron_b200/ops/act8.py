"""Activations kept in 8 bits between forward and backward.

A row of ``n`` values is cut into groups of ``group`` (32, 64, 128 or 256; the last one may be
short).  With ``top = max |x|`` of a group::

    q  = rint(x * (127 * (1 / top)))      int8, ties to even   (0 where top < 2^-120)
    x8 = q * (top * (1 / 127))            the value kept, |x8 - x| <= top / 254

and the scale ``top / 127`` is kept in fp32.  A group that holds a NaN or an infinity comes
back as NaN throughout, so a broken activation is not hidden.

``quantize`` keeps any activation; ``rms_norm`` and ``swiglu`` compute their output from the
exact input and keep the input in 8 bits in the same pass, and their backward passes read
the 8-bit copy.  Each backward also returns the operator's output recomputed from that copy
(``y8``, ``h8``): the operand that the weight gradient of the following projection needs, so
it is not kept either.  Everything is computed in fp32 and rounded once on output.

CUDA tensors run ``csrc/act8.cu`` (``quantize``: bf16, fp16, fp32; the fused operators: bf16);
CPU tensors run the same arithmetic in PyTorch.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from .ext import error_flag, native

GROUPS = (32, 64, 128, 256)
_TINY = 2.0 ** -120


@dataclass
class Act8:
    """An activation in 8 bits: ``codes`` int8 [rows, n rounded up to 16], ``scales`` fp32
    [rows, groups], the values per row ``n``, and the shape, dtype and group size that
    ``dequantize`` restores.  For ``swiglu`` the rows alternate gate and up, and ``shape`` is
    that of [gate | up]."""
    codes: torch.Tensor
    scales: torch.Tensor
    n: int
    shape: torch.Size
    dtype: torch.dtype
    group: int

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 4 * self.scales.numel()

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The kept values as a contiguous tensor of the original shape."""
        if self.codes.is_cuda:
            return native().act8_dequantize(self.codes, self.scales, self.shape, self.n, dtype or self.dtype,
                                            self.group)
        return _decode(self.codes, self.scales, self.n, self.group).to(dtype or self.dtype).view(self.shape)


def _check_group(group: int) -> None:
    if group not in GROUPS:
        raise ValueError(f"act8: group must be one of {GROUPS}, got {group}")


def _buffers(rows: int, n: int, group: int, device):
    _check_group(group)
    codes = torch.empty(rows, (n + 15) // 16 * 16, dtype=torch.int8, device=device)
    scales = torch.empty(rows, (n + group - 1) // group, dtype=torch.float32, device=device)
    return codes, scales


def _encode(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, group: int) -> None:
    rows, n = x.shape
    m = scales.shape[1]
    p = torch.zeros(rows, m * group)
    p[:, :n] = x
    p = p.view(rows, m, group)
    top = p.abs().amax(-1, keepdim=True) if p.numel() else p.new_zeros(rows, m, 1)
    fine = top.isfinite()
    keep = fine & (top >= _TINY)
    mul = torch.where(keep, torch.reciprocal(top) * 127.0, torch.zeros_like(top))
    q = torch.where(fine, torch.round(p * mul), torch.zeros_like(p)).clamp(-127, 127)
    codes.zero_()
    codes[:, :n] = q.reshape(rows, m * group)[:, :n].to(torch.int8)
    s = torch.where(keep, top * (1.0 / 127.0), torch.zeros_like(top))
    scales.copy_(torch.where(fine, s, torch.full_like(s, float("nan")))[..., 0])


def _decode(codes: torch.Tensor, scales: torch.Tensor, n: int, group: int) -> torch.Tensor:
    return codes[:, :n].float() * scales.repeat_interleave(group, 1)[:, :n]


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as 2-D rows."""
    return x.detach().reshape(x.shape[:-1].numel(), x.shape[-1])


def quantize(x: torch.Tensor, group: int = 128) -> Act8:
    """Keep ``x`` (groups along its last dimension) in 8 bits."""
    if not x.is_floating_point():
        raise TypeError(f"act8.quantize: a floating tensor is required, got {x.dtype}")
    if x.is_cuda:
        codes, scales = native().act8_quantize(x, group)
        return Act8(codes, scales, x.shape[-1], x.shape, x.dtype, group)
    if x.dim() == 0:
        raise ValueError("act8.quantize: x needs at least one dimension")
    x2 = _rows(x)
    codes, scales = _buffers(x2.shape[0], x2.shape[1], group, x.device)
    _encode(x2.float(), codes, scales, group)
    return Act8(codes, scales, x2.shape[1], x.shape, x.dtype, group)


def dequantize(a: Act8, dtype: torch.dtype | None = None) -> torch.Tensor:
    return a.dequantize(dtype)


# ------------------------------------------------------------------------------ RMSNorm
def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float, group: int = 128):
    """``y = w x r`` with ``r = rsqrt(mean x^2 + eps)`` over the last dimension; returns
    (y, r [rows], x in 8 bits)."""
    if x.is_cuda:
        y, rstd, codes, scales = native().act8_rms_norm(x, w, eps, group)
        return y, rstd, Act8(codes, scales, x.shape[-1], x.shape, x.dtype, group)
    x2 = _rows(x).float()
    T, H = x2.shape
    codes, scales = _buffers(T, H, group, x.device)
    rstd = torch.rsqrt(x2.pow(2).mean(-1) + eps)
    y = (x2 * rstd[:, None] * w.float()).to(x.dtype)
    _encode(x2, codes, scales, group)
    return y.view(x.shape), rstd, Act8(codes, scales, H, x.shape, x.dtype, group)


def rms_norm_bwd(dy: torch.Tensor, a: Act8, w: torch.Tensor, rstd: torch.Tensor):
    """Backward of ``rms_norm`` with ``n = x8 r``: ``dx = r (dy w - n mean(dy w n))``,
    ``dw = sum dy n`` (fp32) and ``y8 = n w``; returns (dx, dw, y8)."""
    if dy.shape != a.shape:
        raise ValueError(f"act8.rms_norm_bwd: dy has shape {tuple(dy.shape)}, the input had {tuple(a.shape)}")
    if dy.is_cuda:
        return native().act8_rms_norm_bwd(dy, a.codes, a.scales, w, rstd, a.group, error_flag(dy.device))
    n = _decode(a.codes, a.scales, a.n, a.group) * rstd[:, None]
    g = _rows(dy).float()
    dn = g * w.float()
    dx = (rstd[:, None] * (dn - n * (dn * n).mean(-1, keepdim=True))).to(a.dtype)
    y8 = (n * w.float()).to(a.dtype)
    return dx.view(a.shape), (g * n).sum(0), y8.view(a.shape)


# ------------------------------------------------------------------------------ SwiGLU
def swiglu(gu: torch.Tensor, group: int = 128):
    """``h = silu(g) u`` of ``gu = [g | u]`` ([..., 2F]); returns (h [..., F], gu in 8 bits)."""
    if gu.shape[-1] % 2:
        raise ValueError("act8.swiglu: the last dimension must hold gate and up halves")
    F = gu.shape[-1] // 2
    if gu.is_cuda:
        h, codes, scales = native().act8_swiglu(gu, group)
        return h, Act8(codes, scales, F, gu.shape, gu.dtype, group)
    gu2 = _rows(gu).float()
    T = gu2.shape[0]
    codes, scales = _buffers(2 * T, F, group, gu.device)
    g, u = gu2[:, :F], gu2[:, F:]
    h = (g * torch.sigmoid(g) * u).to(gu.dtype)
    _encode(gu2.reshape(2 * T, F), codes, scales, group)
    return h.view(*gu.shape[:-1], F), Act8(codes, scales, F, gu.shape, gu.dtype, group)


def swiglu_bwd(dh: torch.Tensor, a: Act8):
    """Backward of ``swiglu`` from the 8-bit gate and up; returns (dgu [..., 2F], h8 [..., F])."""
    if (*dh.shape[:-1], 2 * dh.shape[-1]) != tuple(a.shape):
        raise ValueError(f"act8.swiglu_bwd: dh has shape {tuple(dh.shape)}, gate and up had {tuple(a.shape)}")
    if dh.is_cuda:
        return native().act8_swiglu_bwd(dh, a.codes, a.scales, a.group)
    F = a.n
    d = _rows(dh).float()
    v = _decode(a.codes, a.scales, F, a.group).view(-1, 2, F)
    g, u = v[:, 0], v[:, 1]
    s = torch.sigmoid(g)
    dgu = torch.cat([s * (1 + g * (1 - s)) * u * d, g * s * d], 1).to(a.dtype)
    return dgu.view(a.shape), (g * s * u).to(a.dtype).view(dh.shape)
