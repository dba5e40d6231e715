"""fp64 tensors on the CPU are computed in fp64: errors of a few times 2^-53 of the terms, and gradients against differences."""
import torch

from femtotron_b200.ops import functional as FN


def test_embedding():
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(-1, 7, (50,), generator=g)
    w = torch.randn(6, 5, generator=g, dtype=torch.float64)
    do = torch.randn(50, 5, generator=g, dtype=torch.float64)
    scale = 1.0 / 3.0
    one = torch.nn.functional.one_hot(ids.clamp(0, 5), 6).double() * ((ids >= 0) & (ids < 6))[:, None]
    p = torch.nn.Parameter(w.clone())
    out = FN.embedding(ids, p, scale=scale)
    assert out.dtype == torch.float64
    assert ((out - one @ w * scale).abs() <= 2 * 2 ** -53 * w.abs().max()).all()
    out.backward(do)
    FN.embedding(ids, p, scale=scale).backward(do)  # added
    want = 2 * scale * one.T @ do
    assert ((p.grad - want).abs() <= 120 * 2 ** -53 * (2 * scale * one.T @ do.abs())).all()
    assert torch.autograd.gradcheck(lambda x: FN.embedding(ids, x * 1.0, scale=scale), w.clone().requires_grad_())
