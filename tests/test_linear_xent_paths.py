"""The forms that the head's cross entropy takes by its sizes: one or two rows (wide and narrow rows of w,
one step and several of a lane's loop), sums of the hidden gradient split over shares and pieces,
gradient sinks that accumulate where the pair kernel runs, with four and with eight epilogue warps.

Oracle and bounds are those of test_linear_xent.py; a sink that holds bf16 is rounded once more per
addition (2^-8 of what it then holds)."""
import pytest
import torch

from femtotron_b200.ops import functional as FN
from test_linear_xent import DEVICES, IGNORE, close, eps_x, make, oracle


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("H,V,pad", [(4096, 1003, 0), (72, 333, 0), (1000, 501, 0), (4096, 517, 8), (2048, 17, 0),
                                     (16, 700, 0), (8, 5, 0), (12304, 40, 0), (24584, 9, 0)])
def test_few_rows(device, T, H, V, pad):
    """`pad`: rows of w on 16-byte boundaries only."""
    h, w, lab = make(T, H, V, device, ignored=0.0)
    if pad:
        w = torch.cat([w, w.new_zeros(V, pad)], 1)[:, :H]
    with torch.no_grad():
        got = FN.linear_cross_entropy(h, w, lab, reduction="none")
    want = oracle(h, w, lab)
    assert bool(((got.double() - want).abs() <= eps_x(h, w) + 2.0 ** -20 * want).all())
    lab2 = lab.clone()
    lab2[-1] = IGNORE
    with torch.no_grad():
        again = FN.linear_cross_entropy(h, w, lab2, reduction="none")
    assert float(again[-1]) == 0.0 and torch.equal(again[:-1], got[:-1])


# shares of the hidden gradient and pieces of the vocabulary (on 148 multiprocessors)
SPLITS = [(130, 136, 23383, 5996423),   # 22 shares in 2 pieces, pair kernel
          (300, 520, 19887, 5236037),   # 2 shares in 3 pieces, pair kernel
          (130, 64, 26742, 2211853),    # 13 shares in 4 pieces
          (520, 64, 14373, 1275991),    # 2 shares in 15 pieces, the last piece one k-block: 1 share
          (64, 64, 28200, 377283)]      # the same for a short batch


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,H,V,workspace", SPLITS)
def test_shares_and_pieces_of_the_hidden_gradient(device, T, H, V, workspace):
    h, w, lab = make(T, H, V, device)
    a, b = h.clone().requires_grad_(), w.clone().requires_grad_()
    FN.linear_cross_entropy(a, b, lab, reduction="sum", workspace_bytes=workspace).backward()
    _, dh, dw, mh, mw = oracle(h, w, lab, torch.ones(T, device=device))
    ex = 2.0 ** -8 + 2 * eps_x(h, w)
    close(a.grad, dh, mh, ex, 2.0 ** -8)
    close(b.grad, dw, mw, ex, 2.0 ** -8)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,H,V", [(100, 256, 700), (200, 256, 700), (200, 1024, 515), (300, 256, 700), (300, 1024, 515),
                                   (64, 1024, 515)])
@pytest.mark.parametrize("sink", ["fp32", "bf16"])
@pytest.mark.parametrize("workspace", [FN.X.WORKSPACE_BYTES, 1])
def test_sinks_accumulate(device, T, H, V, sink, workspace):
    """fp32: stored first, then added twice; bf16: created by the first backward."""
    h, w, lab = make(T, H, V, device)
    w = torch.nn.Parameter(w)
    if sink == "fp32":
        w.main_grad = torch.full(w.shape, 7.0, device=device)
        w.grad_overwrite = True
    for scale in (1.0, 0.5, 2.0):
        (scale * FN.linear_cross_entropy(h, w, lab, reduction="sum", workspace_bytes=workspace)).backward()
    _, _, dw, _, mw = oracle(h, w.detach(), lab, torch.ones(T, device=device))
    ex = 2.0 ** -8 + 2 * eps_x(h, w.detach())
    if sink == "fp32":
        assert w.grad is None
        close(w.main_grad, 3.5 * dw, 3.5 * mw, ex, 2.0 ** -20)
    else:
        close(w.grad, 3.5 * dw, 3.5 * mw, ex, 3 * 2.0 ** -8)
