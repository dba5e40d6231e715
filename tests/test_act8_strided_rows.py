"""Gradients that arrive in rows off every vector boundary, or strided, in the backward passes from 8
bits: the same bits as from a contiguous copy."""
import pytest
import torch

from femtotron_b200.ops import act8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def rows(T, n, device, lead, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, n + lead + 3, generator=g).to(torch.bfloat16).to(device)[:, lead:lead + n]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [0, 1, 8])
@pytest.mark.parametrize("T,H", [(5, 136), (33, 1024), (9, 2056), (7, 4096), (3, 8200)])
def test_rms_norm_backward(device, lead, T, H):
    x, w = rows(T, H, device, 0, 2).contiguous(), rows(1, H, device, 0, 3).reshape(-1).contiguous()
    _, rstd, a = act8.rms_norm(x, w, 1e-5, 64)
    for dy in (rows(T, H, device, lead), rows(2 * T, H, device, lead)[::2],
               torch.ones(1, 1, dtype=torch.bfloat16, device=device).expand(T, H),
               rows(1, H, device, lead).expand(T, H)):
        got = act8.rms_norm_bwd(dy, a, w, rstd)
        want = act8.rms_norm_bwd(dy.contiguous(), a, w, rstd)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    off = rows(1, H, device, 1, 3).reshape(-1)  # a weight off its boundary
    got = act8.rms_norm_bwd(x, a, off, rstd)
    want = act8.rms_norm_bwd(x, a, off.clone(), rstd)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lead", [0, 1, 8])
@pytest.mark.parametrize("T,F", [(5, 72), (33, 688), (3, 4096)])
def test_swiglu_backward(device, lead, T, F):
    _, a = act8.swiglu(rows(T, 2 * F, device, lead, 2), 64)
    _, b = act8.swiglu(rows(T, 2 * F, device, lead, 2).contiguous(), 64)
    assert torch.equal(a.codes[:, :F], b.codes[:, :F]) and torch.equal(a.scales, b.scales)
    for dh in (rows(T, F, device, lead), rows(2 * T, F, device, lead)[::2],
               torch.ones(1, 1, dtype=torch.bfloat16, device=device).expand(T, F)):
        got, want = act8.swiglu_bwd(dh, a), act8.swiglu_bwd(dh.contiguous(), a)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
