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

from .ext import native

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
        x = torch.empty(self.shape, dtype=dtype or self.dtype, device=self.codes.device)
        x2 = x.view(self.codes.shape[0], self.n)
        if x.is_cuda:
            native().act8_dequantize(self.codes, self.scales, x2, self.group)
        else:
            x2.copy_(_decode(self.codes, self.scales, self.n, self.group))
        return x


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
    """x as 2-D rows with a unit inner stride (a view where its strides allow one)."""
    x2 = x.reshape(x.shape[:-1].numel(), x.shape[-1])
    return x2 if x2.shape[1] <= 1 or x2.stride(1) == 1 else x2.contiguous()


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """``_rows`` whose rows start on 16-byte boundaries, as the fused kernels need."""
    x2 = _rows(x)
    if x2.is_cuda and (x2.data_ptr() % 16 or x2.stride(0) * x2.element_size() % 16):
        x2 = x2.clone(memory_format=torch.contiguous_format)
    return x2


def quantize(x: torch.Tensor, group: int = 128) -> Act8:
    """Keep ``x`` (groups along its last dimension) in 8 bits."""
    if x.dim() == 0:
        raise ValueError("act8.quantize: x needs at least one dimension")
    if not x.is_floating_point():
        raise TypeError(f"act8.quantize: a floating tensor is required, got {x.dtype}")
    x2 = _rows(x.detach())
    codes, scales = _buffers(x2.shape[0], x2.shape[1], group, x.device)
    if x.is_cuda:
        native().act8_quantize(x2, codes, scales, group)
    else:
        _encode(x2.float(), codes, scales, group)
    return Act8(codes, scales, x2.shape[1], x.shape, x.dtype, group)


def dequantize(a: Act8, dtype: torch.dtype | None = None) -> torch.Tensor:
    return a.dequantize(dtype)


# ------------------------------------------------------------------------------ RMSNorm
def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float, group: int = 128):
    """``y = w x r`` with ``r = rsqrt(mean x^2 + eps)`` over the last dimension; returns
    (y, r [rows], x in 8 bits)."""
    x2 = _rows16(x.detach())
    T, H = x2.shape
    codes, scales = _buffers(T, H, group, x.device)
    y = torch.empty(T, H, dtype=x.dtype, device=x.device)
    rstd = torch.empty(T, dtype=torch.float32, device=x.device)
    if x.is_cuda:
        native().act8_rms_norm(x2, w, y, rstd, codes, scales, group, float(eps))
    else:
        xf = x2.float()
        rstd.copy_(torch.rsqrt(xf.pow(2).mean(-1) + eps))
        y.copy_(xf * rstd[:, None] * w.float())
        _encode(xf, codes, scales, group)
    return y.view(x.shape), rstd, Act8(codes, scales, H, x.shape, x.dtype, group)


def rms_norm_bwd(dy: torch.Tensor, a: Act8, w: torch.Tensor, rstd: torch.Tensor):
    """Backward of ``rms_norm`` with ``n = x8 r``: ``dx = r (dy w - n mean(dy w n))``,
    ``dw = sum dy n`` (fp32) and ``y8 = n w``; returns (dx, dw, y8)."""
    if dy.shape != a.shape:
        raise ValueError(f"act8.rms_norm_bwd: dy has shape {tuple(dy.shape)}, the input had {tuple(a.shape)}")
    dy2 = _rows16(dy)
    T, H = dy2.shape
    dx = torch.empty(T, H, dtype=a.dtype, device=dy.device)
    y8 = torch.empty(T, H, dtype=a.dtype, device=dy.device)
    dw = torch.empty(H, dtype=torch.float32, device=dy.device)
    if dy.is_cuda:
        m = native()
        with torch.cuda.device(dy.device):
            part = torch.empty(m.act8_norm_walkers(T, H), H, dtype=torch.float32, device=dy.device)
        m.act8_rms_norm_bwd(dy2, a.codes, a.scales, w, rstd, dx, y8, dw, part, a.group)
    else:
        n = _decode(a.codes, a.scales, H, a.group) * rstd[:, None]
        g = dy2.float()
        dn = g * w.float()
        dx.copy_(rstd[:, None] * (dn - n * (dn * n).mean(-1, keepdim=True)))
        dw.copy_((g * n).sum(0))
        y8.copy_(n * w.float())
    return dx.view(a.shape), dw, y8.view(a.shape)


# ------------------------------------------------------------------------------ SwiGLU
def swiglu(gu: torch.Tensor, group: int = 128):
    """``h = silu(g) u`` of ``gu = [g | u]`` ([..., 2F]); returns (h [..., F], gu in 8 bits)."""
    if gu.shape[-1] % 2:
        raise ValueError("act8.swiglu: the last dimension must hold gate and up halves")
    gu2 = _rows16(gu.detach())
    T, F = gu2.shape[0], gu2.shape[1] // 2
    codes, scales = _buffers(2 * T, F, group, gu.device)
    h = torch.empty(T, F, dtype=gu.dtype, device=gu.device)
    if gu.is_cuda:
        native().act8_swiglu(gu2, h, codes, scales, group)
    else:
        g, u = gu2[:, :F].float(), gu2[:, F:].float()
        h.copy_(g * torch.sigmoid(g) * u)
        _encode(gu2.float().reshape(2 * T, F), codes, scales, group)
    return h.view(*gu.shape[:-1], F), Act8(codes, scales, F, gu.shape, gu.dtype, group)


def swiglu_bwd(dh: torch.Tensor, a: Act8):
    """Backward of ``swiglu`` from the 8-bit gate and up; returns (dgu [..., 2F], h8 [..., F])."""
    if (*dh.shape[:-1], 2 * dh.shape[-1]) != tuple(a.shape):
        raise ValueError(f"act8.swiglu_bwd: dh has shape {tuple(dh.shape)}, gate and up had {tuple(a.shape)}")
    dh2 = _rows16(dh)
    T, F = dh2.shape
    dgu = torch.empty(T, 2 * F, dtype=a.dtype, device=dh.device)
    h8 = torch.empty(T, F, dtype=a.dtype, device=dh.device)
    if dh.is_cuda:
        native().act8_swiglu_bwd(dh2, a.codes, a.scales, dgu, h8, a.group)
    else:
        v = _decode(a.codes, a.scales, F, a.group).view(T, 2, F)
        g, u, d = v[:, 0], v[:, 1], dh2.float()
        s = torch.sigmoid(g)
        dgu[:, :F] = (d * u * s * (1 + g * (1 - s))).to(dgu.dtype)
        dgu[:, F:] = (d * g * s).to(dgu.dtype)
        h8.copy_(g * s * u)
    return dgu.view(a.shape), h8.view(dh.shape)
