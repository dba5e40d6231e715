"""Global norm and clipping of many tensors against 64 bits, on the CPU and, marked gpu, through the kernels."""
import math

import pytest
import torch

from femtotron_b200.ops import grad_norm as GN

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def some(device, seed=0, scale=1.0):
    """Tensors of all types, sizes around vectors and chunks, odd places in memory, other strides."""
    g = torch.Generator().manual_seed(seed)
    sizes = [1, 3, 4, 7, 8, 255, 8191, 8192, 8193, 20000]
    xs = [torch.randn(n, generator=g).mul(scale).to(t).to(device) for n in sizes for t in HALF]
    base = torch.randn(5000, generator=g).mul(scale).to(device)
    xs += [base[1:1000], base[1003:2048], base[4000:4001]]
    wide = torch.randn(64, 33, generator=g).mul(scale).to(device)
    xs += [wide.t(), torch.randn(40, 50, generator=g).mul(scale).to(device)[:, ::2], torch.empty(0, device=device),
           torch.randn(3, 5, 7, generator=g).mul(scale).to(torch.bfloat16).to(device).permute(2, 0, 1)]
    return xs


def norm64(xs):
    return math.sqrt(sum(x.double().pow(2).sum().item() for x in xs))


# squares of eight values in fp32 (each sum off by at most 8 units of 2^-24 of itself), fp64 beyond, a root
# (which halves the relative error), one rounding to fp32
NORM_TOL = 4 * 2 ** -24 + 2 ** -24 + 1e-12


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("max_norm", [1.0, 1e6])
@pytest.mark.parametrize("inplace", [True, False])
def test_clip(device, max_norm, inplace):
    xs = some(device)
    before = [x.clone() for x in xs]
    out = None if inplace else [torch.full_like(x, 7.0) for x in xs]
    norm = GN.clip_grads(xs, max_norm, out=out)
    assert norm.dtype == torch.float32 and norm.shape == () and norm.device == xs[0].device
    want = norm64(before)
    assert abs(norm.item() - want) <= NORM_TOL * want
    coef = min(1.0, max_norm / (want + 1e-6))
    for x, b, y in zip(xs, before, out if out is not None else xs):
        if not inplace:
            assert torch.equal(x, b)
        # the factor: the norm's error, a sum, a quotient in fp32; then the product and its rounding
        tol = coef * b.double().abs() * (NORM_TOL + 3 * 2 ** -24 + HALF[y.dtype]) + (1e-7 if y.dtype == torch.float16 else 0)
        assert ((y.double() - b.double() * coef).abs() <= tol).all()
        if coef == 1.0:
            assert torch.equal(y, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1e-30, 1e25])
def test_squares_beyond_fp32(device, scale):
    xs = [x for x in some(device, 1) if x.dtype == torch.float32]
    xs = [(x * scale) for x in xs]
    want = norm64(xs)
    assert abs(GN.sum_of_squares(xs)[0].sqrt().item() - want) <= NORM_TOL * want
    assert abs(GN.clip_grads(xs, 1.0, out=[torch.empty_like(x) for x in xs]).item() - want) <= NORM_TOL * want + 1e-45


@pytest.mark.parametrize("device", DEVICES)
def test_slots(device):
    xs = some(device, 2)
    slots = [i % 4 for i in range(len(xs))]
    got = GN.sum_of_squares(xs, slots, 5)
    assert got.dtype == torch.float64 and got.shape == (5,) and got[4] == 0
    for s in range(4):
        want = sum(x.double().pow(2).sum().item() for x, t in zip(xs, slots) if t == s)
        assert abs(got[s].item() - want) <= 2 * NORM_TOL * want


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_not_finite(device, value):
    xs = [torch.ones(100, device=device), torch.ones(9000, device=device, dtype=torch.bfloat16)]
    xs[1][17] = value
    norm = GN.clip_grads(xs, 1.0)
    assert math.isnan(norm.item()) if math.isnan(value) else norm.item() == math.inf
    if math.isinf(value):
        assert not xs[0].any() and torch.isnan(xs[1][17]) and xs[1].isnan().sum() == 1
    else:
        assert xs[0].isnan().all() and xs[1].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
def test_many_and_none(device):
    xs = [torch.full((1 + i % 3,), 0.5, device=device) for i in range(2500)]
    want = 0.5 * math.sqrt(sum(x.numel() for x in xs))
    assert abs(GN.clip_grads(xs, 1.0).item() - want) < 1e-5 * want
    assert abs(norm64(xs) - 1.0) < 1e-5
    assert GN.clip_grads([], 1.0).item() == 0
    assert GN.clip_grads([torch.empty(0, device=device)], 1.0).item() == 0
    zeros = [torch.zeros(10000, device=device)]
    assert GN.clip_grads(zeros, 1.0).item() == 0 and not zeros[0].any()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = torch.ones(8, device=device)
    with pytest.raises(TypeError, match="fp32, bf16 or fp16"):
        GN.clip_grads([x, x.long()], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        GN.clip_grads([x], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        GN.clip_grads([x], math.nan)
    with pytest.raises(ValueError, match="outputs"):
        GN.clip_grads([x], 1.0, out=[])
    with pytest.raises(ValueError, match="an output of"):
        GN.clip_grads([x], 1.0, out=[x.bfloat16()])
    with pytest.raises(ValueError, match="slots"):
        GN.sum_of_squares([x], [1], 1)
    with pytest.raises(ValueError, match="slots"):
        GN.sum_of_squares([x], [0, 0], 1)


@gpu
def test_gpu_shared_memory_is_refused_and_order_is_fixed():
    x = torch.randn(100, device="cuda")
    for xs, out in (([x, x], None), ([x[:60], x[50:]], None), ([x[:50], x[50:]], [x[50:], x[:50]]),
                    ([x[:50]], [x[1:51]])):
        with pytest.raises(RuntimeError, match="share"):
            GN.clip_grads(xs, 1.0, out=out)
    GN.clip_grads([x[:50], x[50:]], 1.0)
    GN.clip_grads([x], 1.0, out=[x])
    xs = some("cuda", 3)
    assert len({GN.sum_of_squares(xs)[0].item() for _ in range(5)}) == 1


@gpu
def test_gpu_in_a_graph_and_on_another_stream():
    g = [torch.randn(n, device="cuda") for n in (70000, 33)]
    src = [x.clone() for x in g]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        GN.clip_grads(g, 1.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            norm = GN.clip_grads(g, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    for k in (1.0, 3.0):
        for x, y in zip(g, src):
            x.copy_(y * k)
        want = norm64(g)
        graph.replay()
        assert abs(norm.item() - want) <= NORM_TOL * want and abs(norm64(g) - 1.0) < 1e-5
