"""Activations in 8 bits: format, fused operators and their backward passes.

Oracle: the definition in 64 bits from the stored codes and scales, which are themselves
checked bit for bit against a restatement of the format.  Bounds: results are fp32 sums and
products rounded once to bf16, so an output is within half a bf16 step (at most 2^-8 relative, 8 significant bits) of the
oracle plus fp32 rounding, 2^-18 of the magnitudes that were added (a row of up to 2^13 terms
summed pairwise, each term a handful of roundings of 2^-24, and an exponential good to
2^-21 of its argument's size).  A sigmoid below 2^-126 may be flushed to zero: it counts as
2^-126 in those magnitudes (2^-18 * 2^-108).
"""
import pytest
import torch

from femtotron_b200.ops import act8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16 = 2.0 ** -8
F32 = 2.0 ** -18


def fmt(x: torch.Tensor, group: int):
    """Codes and scales of x [rows, n] by the format's definition (numpy fp32)."""
    import numpy as np
    x = x.float().cpu().numpy()
    rows, n = x.shape
    codes = np.zeros((rows, n), dtype=np.int64)
    scales = np.zeros((rows, -(-n // group)), dtype=np.float32)
    for a in range(0, n, group):
        part = x[:, a:a + group]
        top = np.abs(part).max(1).astype(np.float32)
        tiny = top < np.float32(2.0 ** -120)
        with np.errstate(all="ignore"):
            mul = np.where(tiny, np.float32(0), (np.float32(1) / top) * np.float32(127))
            q = np.rint(part * mul[:, None].astype(np.float32))
        bad = ~np.isfinite(top)
        q = np.where(bad[:, None] | np.isnan(q), 0, q)
        codes[:, a:a + group] = np.clip(q, -127, 127).astype(np.int64)
        s = np.where(tiny, np.float32(0), top * np.float32(1.0 / 127.0))
        scales[:, a // group] = np.where(bad, np.float32("nan"), s)
    return torch.from_numpy(codes), torch.from_numpy(scales)


def values(a: act8.Act8) -> torch.Tensor:
    """The kept values in 64 bits, [rows of codes, n]."""
    rep = a.scales.double().repeat_interleave(a.group, 1)[:, :a.n]
    v32 = a.codes[:, :a.n].float() * rep.float()  # the format keeps the fp32 product
    return v32.double()


def act(shape, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    x[..., ::37] *= 30
    return x.to(dtype).to(device)


def close(got, want, scale_terms, half_step=BF16):
    err = (got.double() - want).abs()
    bound = half_step * want.abs() + F32 * scale_terms + 1e-37
    assert bool((err <= bound).all()), float((err / bound).max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("group", act8.GROUPS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 17), (2, 5, 256), (7, 1023), (130, 4096), (5, 136), (1, 40000)])
def test_quantize_codes_scales_and_values(device, dtype, group, shape):
    x = act(shape, dtype, device)
    a = act8.quantize(x, group)
    n = shape[-1]
    codes, scales = fmt(x.reshape(-1, n), group)
    assert torch.equal(a.codes[:, :n].cpu().long(), codes)
    assert torch.equal(a.scales.cpu(), scales)
    got = a.dequantize(torch.float32)
    assert got.shape == x.shape and torch.equal(got.cpu().reshape(-1, n).double(), values(a).cpu())
    # half a code away at most; 2^-16 of a code and 2^-23 of x for the fp32 products
    step = scales.repeat_interleave(group, 1)[:, :n].reshape(shape).double()
    x64 = x.cpu().double()
    assert bool(((got.cpu().double() - x64).abs() <= step * (0.5 + 2.0 ** -16) + 2.0 ** -23 * x64.abs()).all())
    # in its own type: the kept value rounded once
    back = a.dequantize()
    assert back.dtype == dtype and torch.equal(back, got.to(dtype))


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_special_groups(device):
    x = torch.zeros(4, 256)
    x[0, :128] = 2.0 ** -126          # below the smallest kept magnitude: zeros
    x[0, 128:] = 2.0 ** -119          # above it
    x[1, 5] = float("inf")
    x[2, 200] = float("nan")
    x[3, :128] = torch.finfo(torch.float32).max
    x[3, 3] = -x[3, 3]
    y = act8.quantize(x.to(device), 128).dequantize().cpu()
    assert bool((y[0, :128] == 0).all()) and torch.allclose(y[0, 128:], x[0, 128:], rtol=1e-6)
    assert bool(y[1, :128].isnan().all()) and bool((y[1, 128:] == 0).all())
    assert bool(y[2, 128:].isnan().all()) and bool((y[2, :128] == 0).all())
    assert torch.allclose(y[3, :128], x[3, :128], rtol=1e-6)


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_strided_rows_and_empty(device):
    base = act((9, 3, 200), torch.bfloat16, device)
    for x in (base[:, 1], base[:, :, 3:131], base.transpose(0, 1), base[::2, 0, :64], base[..., ::2]):
        a, b = act8.quantize(x, 64), act8.quantize(x.contiguous(), 64)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    for shape in ((0, 64), (4, 0)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=device)
        assert act8.quantize(x).dequantize().shape == x.shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,H,group", [(1, 8, 32), (3, 256, 128), (5, 520, 64), (33, 1000, 128), (4, 2048, 256),
                                          (17, 4096, 128), (3, 5120, 32), (2, 8192, 128), (3, 16384, 256),
                                          (700, 1024, 128), (0, 256, 128)])
def test_rms_norm_and_backward(device, rows, H, group):
    x, dy = act((rows, H), torch.bfloat16, device), act((rows, H), torch.bfloat16, device, 1)
    w = (1 + 0.1 * act((H,), torch.float32, device, 2)).to(torch.bfloat16)
    y, rstd, a = act8.rms_norm(x, w, 1e-5, group)
    r64 = torch.rsqrt(x.double().pow(2).mean(1) + 1e-5)
    assert torch.allclose(rstd.double(), r64, rtol=1e-6, atol=0)
    want = x.double() * r64[:, None] * w.double()
    close(y, want, want.abs())
    codes, scales = fmt(x, group)
    assert torch.equal(a.codes[:, :H].cpu().long(), codes) and torch.equal(a.scales.cpu(), scales)
    dx, dw, y8 = act8.rms_norm_bwd(dy, a, w, rstd)
    r = rstd.double()[:, None]
    n = values(a) * r
    dn = dy.double() * w.double()
    close(y8, n * w.double(), (n * w.double()).abs())
    mean = (dn * n).mean(1, keepdim=True)
    mag = (dn * n).abs().mean(1, keepdim=True)
    close(dx, r * (dn - n * mean), r * (dn.abs() + n.abs() * mag))
    close(dw, (dy.double() * n).sum(0), (dy.double() * n).abs().sum(0), half_step=0.0)
    again = act8.rms_norm_bwd(dy, a, w, rstd)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, y8), again))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("rows,F,group", [(1, 8, 32), (3, 688, 128), (5, 1000, 64), (2, 14336, 256), (257, 512, 32),
                                          (0, 64, 128)])
def test_swiglu_and_backward(device, rows, F, group):
    gu, dh = act((rows, 2 * F), torch.bfloat16, device), act((rows, F), torch.bfloat16, device, 1)
    h, a = act8.swiglu(gu, group)
    g, u = gu[:, :F].double(), gu[:, F:].double()
    s = torch.sigmoid(g)
    close(h, g * s * u, (1 + g.abs()) * (g * u).abs() * s.clamp(min=2.0 ** -108))
    codes, scales = fmt(gu.reshape(2 * rows, F), group)
    assert torch.equal(a.codes[:, :F].cpu().long(), codes) and torch.equal(a.scales.cpu(), scales)
    dgu, h8 = act8.swiglu_bwd(dh, a)
    v = values(a).view(rows, 2, F)
    g, u, d = v[:, 0], v[:, 1], dh.double()
    s = torch.sigmoid(g)
    big, sm = 1 + g.abs(), s.clamp(min=2.0 ** -108)
    close(h8, g * s * u, big * (g * u).abs() * sm)
    close(dgu[:, :F], d * u * s * (1 + g * (1 - s)), big * big * (d * u).abs() * sm)
    close(dgu[:, F:], d * g * s, big * (d * g).abs() * sm)


def test_backward_formulas_against_differences():
    """The backward formulas, in 64 bits, against central differences of the forward ones."""
    g = torch.Generator().manual_seed(0)
    x, w, dy = (torch.randn(3, 8, generator=g, dtype=torch.float64) for _ in range(3))
    w = w[0]
    e = 1e-6

    def norm(x, w):
        return x * torch.rsqrt(x.pow(2).mean(1, keepdim=True) + 1e-5) * w
    r = torch.rsqrt(x.pow(2).mean(1, keepdim=True) + 1e-5)
    n = x * r
    dn = dy * w
    dx = r * (dn - n * (dn * n).mean(1, keepdim=True))
    for i in range(8):
        step = torch.zeros_like(x)
        step[:, i] = e
        num = ((norm(x + step, w) - norm(x - step, w)) * dy).sum(1) / (2 * e)
        assert torch.allclose(num, dx[:, i], atol=1e-7)
        ws = torch.zeros_like(w)
        ws[i] = e
        num = ((norm(x, w + ws) - norm(x, w - ws)) * dy).sum() / (2 * e)
        assert torch.allclose(num, (dy * n).sum(0)[i], atol=1e-7)

    gate, up = x, dy

    def f(gate, up):
        return gate * torch.sigmoid(gate) * up
    s = torch.sigmoid(gate)
    assert torch.allclose((f(gate + e, up) - f(gate - e, up)) / (2 * e), up * s * (1 + gate * (1 - s)), atol=1e-7)
    assert torch.allclose((f(gate, up + e) - f(gate, up - e)) / (2 * e), gate * s, atol=1e-7)


@pytest.mark.gpu
def test_fused_operators_take_unaligned_rows_and_other_streams():
    base = act((64, 1032), torch.bfloat16, "cuda")
    w = torch.ones(1024, dtype=torch.bfloat16, device="cuda")
    x = base[:, 1:1025]
    y, rstd, a = act8.rms_norm(x, w, 1e-5)
    y2, _, a2 = act8.rms_norm(x.contiguous(), w, 1e-5)
    assert torch.equal(y, y2) and torch.equal(a.codes, a2.codes)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        z = act8.quantize(x, 64).dequantize()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(z, act8.quantize(x.contiguous(), 64).dequantize())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError):
        act8.quantize(x, 48)
    with pytest.raises(TypeError):
        act8.quantize(x.long())
    with pytest.raises(ValueError):
        act8.quantize(torch.zeros((), device=device))
    w = torch.ones(64, dtype=torch.bfloat16, device=device)
    _, rstd, a = act8.rms_norm(x, w, 1e-5)
    with pytest.raises(ValueError):
        act8.rms_norm_bwd(x[:, :32], a, w, rstd)
    with pytest.raises(ValueError):
        act8.swiglu(x[:, :63])
    _, b = act8.swiglu(x)
    with pytest.raises(ValueError):
        act8.swiglu_bwd(x, b)


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    x = torch.zeros(4, 60, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        act8.rms_norm(x, torch.ones(60, dtype=torch.bfloat16, device="cuda"), 1e-5)  # H % 8
    with pytest.raises(RuntimeError):
        act8.rms_norm(x[:, :56].float(), torch.ones(56, device="cuda"), 1e-5)        # fp32
    with pytest.raises(RuntimeError):
        act8.rms_norm(x[:, :56], torch.ones(48, dtype=torch.bfloat16, device="cuda"), 1e-5)
    with pytest.raises(RuntimeError):
        act8.quantize(x.double())
