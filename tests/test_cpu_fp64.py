"""fp64 tensors on the CPU are computed in fp64: errors of a few times 2^-53 of the terms, and gradients against differences."""
import math

import pytest
import torch

from femtotron_b200.ops import functional as FN
from femtotron_b200.ops import masked_attention as MA
from test_masked_attention import make, mask_parts, reference, run


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


@pytest.mark.parametrize("softcap,bias", [(0.0, False), (2.0, True)])
def test_masked_attention(softcap, bias):
    B, S, nq, nkv, d = 2, 23, 4, 2, 6
    q, k, v, do = make(B, S, nq, nkv, d, 1, "cpu", torch.float64)
    parts = mask_parts("all", B, S, 5)
    mask = MA.attention_mask(B, S, **parts)
    kw = dict(softcap=softcap, slopes=MA.alibi_slopes(nq) if bias else None)
    want, size = reference(q, k, v, do, MA._visible(mask).expand(B, S, S), 1 / math.sqrt(d), softcap, kw["slopes"])
    for x, y, z in zip(run(q, k, v, do, mask, **kw), want, size):
        # as in fp32: 64 units in the last place of the terms' absolute sum
        assert x.dtype == torch.float64 and ((x - y).abs() <= 64 * torch.finfo(torch.float64).eps * (z + y.abs())).all()
    leaves = [x[:1, :7].clone().requires_grad_() for x in (q, k, v)]
    small = MA.attention_mask(1, 7, window=3)
    assert torch.autograd.gradcheck(lambda *x: MA.masked_attention(*x, small, **kw), leaves)
