"""Row gradients that are not finite, or that belong to ignored rows, in the backward of the head's
per-row losses.

Oracle: the definition in 64 bits, with the gradient of an ignored row taken as 0.  Bounds: d is
rounded to bf16 (2^-8 of itself), the logits behind it are good to 2^-12 here (hidden size 128),
and the results are rounded to bf16 once more."""
import pytest
import torch

from femtotron_b200.ops import functional as FN

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
IGNORE = -100
INF = float("inf")


def make(T, device, H=128, V=300):
    g = torch.Generator().manual_seed(T)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16).to(device)
    w = (torch.randn(V, H, generator=g) * 0.2).to(torch.bfloat16).to(device)
    lab = torch.randint(0, V, (T,), generator=g)
    return h, w, lab.to(device), torch.randn(T, generator=g).to(device)


def gradients(h, w, lab, g):
    h, w = h.clone().requires_grad_(), w.clone().requires_grad_()
    FN.linear_cross_entropy(h, w, lab, reduction="none").backward(g)
    return h.grad, w.grad


def check(h, w, lab, g, dh, dw=None, rows=slice(None)):
    h, w = h.double(), w.double()
    x = h @ w.t()
    d = torch.softmax(x, 1)
    d.scatter_add_(1, lab.clamp(min=0)[:, None], -torch.ones_like(x[:, :1]))
    d *= torch.where(lab == IGNORE, torch.zeros_like(g), g).double()[:, None]
    for got, a, b, at in ((dh, d, w, rows), (dw, d.t(), h, slice(None))):
        if got is not None:
            want, mag = (a @ b)[at], (a.abs() @ b.abs())[at]
            err = (got[at].double() - want).abs()
            assert bool((err <= (2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -8 * want.abs() + 1e-30).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 5, 200])
def test_nan_from_above_reaches_both_gradients(device, T):
    h, w, lab, g = make(T, device)
    lab[T // 2 + 1:] = IGNORE
    dh, dw = gradients(h, w, lab, g * float("nan"))
    assert bool(dh[:T // 2 + 1].isnan().all()) and bool(dw.isnan().all())
    assert bool((dh[T // 2 + 1:] == 0).all())
    # NaN beside zeros
    g = torch.zeros(T, device=device)
    g[0] = float("nan")
    dh, dw = gradients(h, w, lab, g)
    assert bool(dh[0].isnan().all()) and bool(dw.isnan().all()) and bool((dh[1:] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [float("nan"), INF, -INF])
@pytest.mark.parametrize("T", [5, 200])
def test_one_row_that_is_not_finite_leaves_the_others_hidden_gradients(device, bad, T):
    h, w, lab, g = make(T, device)
    g[2] = bad
    dh, dw = gradients(h, w, lab, g)
    assert not bool(dh[2].isfinite().any()) and not bool(dw.isfinite().any())
    fine = torch.arange(T, device=device) != 2
    check(h, w, lab, torch.where(fine, g, torch.zeros_like(g)), dh, rows=fine)
