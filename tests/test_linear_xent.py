"""Cross entropy of a linear head without its logits.

Oracle: 64-bit logits of the same bf16 operands.  Bounds: u = 2^-24 for fp32, 2^-8 for the
rounding to bf16.  A logit is an fp32 sum of H products: off by at most 2^-22 sqrt(H) of its
root-sum-square (random signs; 4 sigma), written ``eps_x`` below; so are lse and the loss (their
derivative by each logit is at most 1).  The entries of d are within eps_x + 2^-8 of theirs
relatively, except the label's, off by 2^-8 of p at most plus 2^-8 of |p - 1|; dh and dw sum
T or V products of them: bounded by the same share of the summed magnitudes.  The result is
rounded once more."""
import math

import pytest
import torch

from femtotron_b200.ops import functional as FN
from femtotron_b200.ops import linear_xent as X

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
IGNORE = -100


def make(T, H, V, device, dtype=torch.bfloat16, spread=2.5, ignored=0.2, seed=0):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g).to(dtype).to(device)
    w = (torch.randn(V, H, generator=g) * (spread / math.sqrt(H))).to(dtype).to(device)
    lab = torch.randint(0, V, (T,), generator=g)
    lab[torch.rand(T, generator=g) < ignored] = IGNORE
    lab[0] = V - 1
    return h, w, lab.to(device)


def oracle(h, w, lab, g=None):
    """losses, and for row gradients g: dh, dw and the magnitudes that their sums add."""
    h, w = h.double(), w.double()
    x = h @ w.t()
    lse = torch.logsumexp(x, 1)
    valid = lab != IGNORE
    at = lab.clamp(min=0)[:, None]
    losses = torch.where(valid, lse - x.gather(1, at)[:, 0], torch.zeros_like(lse))
    if g is None:
        return losses
    d = torch.exp(x - lse[:, None])
    d.scatter_add_(1, at, -torch.ones_like(lse)[:, None])
    d *= torch.where(valid, g.double(), torch.zeros_like(lse))[:, None]
    return losses, d @ w, d.t() @ h, d.abs() @ w.abs(), d.abs().t() @ h.abs()


def eps_x(h, w):
    return 2.0 ** -22 * math.sqrt(h.shape[1]) * float(h.double().pow(2).mean().sqrt() *
                                                      w.double().pow(2).mean().sqrt() * math.sqrt(h.shape[1])) + 2.0 ** -20


def close(got, want, mag, share, step):
    err = (got.double() - want).abs()
    bound = share * mag + step * want.abs() + 1e-30
    assert bool((err <= bound).all()), float((err / bound).max())


SIZES = [(1, 64, 50), (1, 256, 1000), (3, 72, 257), (128, 128, 512), (129, 256, 2048), (130, 64, 100), (200, 200, 3001),
         (300, 520, 1000), (512, 256, 2048), (1021, 64, 777)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("workspace", [X.WORKSPACE_BYTES, 1])
def test_loss_and_gradients(device, T, H, V, reduction, workspace):
    h, w, lab = make(T, H, V, device)
    h.requires_grad_()
    w.requires_grad_()
    out = FN.linear_cross_entropy(h, w, lab, reduction=reduction, workspace_bytes=workspace)
    valid = (lab != IGNORE)
    if reduction == "none":
        g = torch.randn(T, generator=torch.Generator().manual_seed(5)).to(device)
        g[T // 2] = 0.0 if T > 1 else g[0]
        out.backward(g)
    else:
        out.backward(torch.tensor(0.37, device=device))
        g = torch.full((T,), 0.37, device=device, dtype=torch.float64)
        g = g / valid.sum() if reduction == "mean" else g
    losses, dh, dw, mh, mw = oracle(h.detach(), w.detach(), lab, g)
    ex = eps_x(h.detach(), w.detach())
    want = losses if reduction == "none" else losses.sum() if reduction == "sum" else losses.sum() / valid.sum()
    terms = 1 if reduction != "sum" else T
    assert out.dtype == torch.float32
    assert bool(((out.double() - want).abs() <= terms * ex + 2.0 ** -20 * want.abs()).all())
    # d rounded to bf16 as an operand (not on the CPU, where this only loosens the bound)
    close(h.grad, dh, mh, 2.0 ** -8 + 2 * ex, 2.0 ** -8)
    close(w.grad, dw, mw, 2.0 ** -8 + 2 * ex, 2.0 ** -8)
    # rows that do not count leave no gradient
    assert bool((h.grad[~valid] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
def test_pieces_give_the_same_bits_again(device):
    h, w, lab = make(300, 256, 5000, device)
    got = []
    for _ in range(2):
        hh, ww = h.clone().requires_grad_(), w.clone().requires_grad_()
        FN.linear_cross_entropy(hh, ww, lab, workspace_bytes=1 << 20).backward()
        got.append((hh.grad, ww.grad))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("main", [True, False])
def test_gradient_sinks_accumulate(device, main):
    h, w, lab = make(200, 128, 700, device, ignored=0.0)
    w = torch.nn.Parameter(w)
    if main:
        w.main_grad = torch.full(w.shape, 7.0, device=device)
        w.grad_overwrite = True
    for _ in range(3):
        FN.linear_cross_entropy(h, w, lab, reduction="sum").backward()
    _, _, dw, _, mw = oracle(h, w.detach(), lab, torch.ones(200, device=device))
    ex = eps_x(h, w.detach())
    if main:
        assert w.grad is None
        close(w.main_grad, 3 * dw, 3 * mw, 2.0 ** -8 + 2 * ex, 2.0 ** -20)
    else:
        close(w.grad, 3 * dw, 3 * mw, 2.0 ** -8 + 2 * ex, 3 * 2.0 ** -8)


@pytest.mark.parametrize("device", DEVICES)
def test_only_one_gradient_is_wanted(device):
    h, w, lab = make(140, 64, 300, device)
    g = torch.full((140,), 1.0, device=device) / (lab != IGNORE).sum()
    _, dh, dw, mh, mw = oracle(h, w, lab, g)
    ex = 2.0 ** -8 + 2 * eps_x(h, w)
    a = h.clone().requires_grad_()
    FN.linear_cross_entropy(a, w, lab).backward()
    close(a.grad, dh, mh, ex, 2.0 ** -8)
    b = w.clone().requires_grad_()
    FN.linear_cross_entropy(h, b, lab).backward()
    close(b.grad, dw, mw, ex, 2.0 ** -8)


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_counts_large_logits_and_shapes(device):
    h, w, lab = make(6, 64, 300, device)
    none = torch.full_like(lab, IGNORE)
    hh, ww = h.clone().requires_grad_(), w.clone().requires_grad_()
    loss = FN.linear_cross_entropy(hh, ww, none)
    loss.backward()
    assert bool(loss.isnan()) and bool((hh.grad == 0).all()) and bool((ww.grad == 0).all())
    assert float(FN.linear_cross_entropy(h, w, none, reduction="sum")) == 0.0
    # logits in the thousands: one of them takes all the probability
    big = FN.linear_cross_entropy(h * 64, w * 64, lab, reduction="none")
    want = oracle(h * 64, w * 64, lab)
    assert torch.allclose(big.double(), want, rtol=2.0 ** -18, atol=eps_x(h * 64, w * 64))
    # [B, S, H] input and [B, S] labels; strided rows
    l3 = FN.linear_cross_entropy(h.view(2, 3, 64), w, lab.view(2, 3), reduction="none")
    assert torch.equal(l3, FN.linear_cross_entropy(h, w, lab, reduction="none"))
    wide = torch.zeros(6, 128, dtype=h.dtype, device=device)
    wide[:, 64:] = h
    assert torch.equal(FN.linear_cross_entropy(wide[:, 64:], w, lab, reduction="none"), l3)
    # no rows at all
    e = FN.linear_cross_entropy(h[:0], w, lab[:0], reduction="none")
    assert e.shape == (0,) and float(FN.linear_cross_entropy(h[:0], w, lab[:0], reduction="sum")) == 0.0
    assert bool(FN.linear_cross_entropy(h[:0], w, lab[:0]).isnan())
    # a label that no column answers to
    lab2 = lab.clone()
    lab2[1] = 300
    out = FN.linear_cross_entropy(h, w, lab2, reduction="none")
    assert bool(out[1].isnan()) and int(out.isnan().sum()) == 1
    # an ignored row may hold anything: it stays out of the loss and of every other row's gradient
    h2, lab3 = h.clone(), lab.clone()
    h2[2], lab3[2] = float("nan"), IGNORE
    h2.requires_grad_()
    loss = FN.linear_cross_entropy(h2, w, lab3)
    loss.backward()
    assert bool(loss.isfinite()) and bool(h2.grad.isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("world", [2, 3])
def test_vocabulary_shards_join(device, world):
    """The per-shard numbers of a tensor-parallel head join to the whole vocabulary's."""
    h, w, lab = make(150, 64, 600, device)
    step = 600 // world
    stats = torch.stack([X.forward(h, w[r * step:(r + 1) * step], lab, r * step, IGNORE, "none")[0]
                         for r in range(world)])
    lse, losses, loss, factor = X.combine(X.merge_shards(stats), lab, IGNORE, "mean")
    want = oracle(h, w, lab)
    n = int((lab != IGNORE).sum())
    ex = eps_x(h, w)
    assert bool(((losses.double() - want).abs() <= ex + 2.0 ** -20 * want.abs()).all())
    assert abs(float(loss) - float(want.sum()) / n) <= ex + 1e-5 and abs(float(factor) - 1 / n) < 1e-9
    # each shard's gradient is its rows of the whole one
    grad = torch.ones((), device=device)
    _, dh, dw, mh, mw = oracle(h, w, lab, torch.full((150,), 1 / n, device=device))
    total = torch.zeros_like(dh)
    for r in range(world):
        part, gw = torch.empty_like(h), torch.empty(step, 64, dtype=torch.float32, device=device)
        X.backward(h, w[r * step:(r + 1) * step], lab, lse.contiguous(), grad, factor, part, gw, False, r * step, IGNORE)
        close(gw, dw[r * step:(r + 1) * step], mw[r * step:(r + 1) * step], 2.0 ** -8 + 2 * ex, 2.0 ** -20)
        total += part.double()
    close(total, dh, mh, 2.0 ** -7 + 2 * ex, 2.0 ** -7)


@pytest.mark.parametrize("device", DEVICES)
def test_backward_twice(device):
    """A kept graph gives the same gradient again, added to the first."""
    h, w, lab = make(130, 64, 300, device)
    h.requires_grad_()
    w.requires_grad_()
    loss = FN.linear_cross_entropy(h, w, lab, reduction="sum")
    loss.backward(retain_graph=True)
    one = h.grad.clone(), w.grad.clone()
    loss.backward()
    assert torch.equal(h.grad, 2 * one[0]) and torch.allclose(w.grad, 2 * one[1], rtol=2.0 ** -7, atol=0)


def test_oracle_gradient_matches_differences():
    h, w, lab = make(4, 8, 12, "cpu", torch.float64, ignored=0.0)
    lab[1] = IGNORE
    g = torch.tensor([0.3, 1.0, -2.0, 0.5], dtype=torch.float64)
    _, dh, dw, _, _ = oracle(h, w, lab, g)
    for t, d in ((h, dh), (w, dw)):
        for i in range(0, t.numel(), 3):
            keep = t.view(-1)[i].item()
            t.view(-1)[i] = keep + 1e-5
            up = (oracle(h, w, lab) * g).sum()
            t.view(-1)[i] = keep - 1e-5
            down = (oracle(h, w, lab) * g).sum()
            t.view(-1)[i] = keep
            assert abs(float(up - down) / 2e-5 - float(d.view(-1)[i])) < 1e-7


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    h, w, lab = make(4, 64, 100, device)
    with pytest.raises(ValueError):
        FN.linear_cross_entropy(h, w, lab, reduction="median")
    with pytest.raises(ValueError):
        FN.linear_cross_entropy(h, w[:, :32], lab)
    with pytest.raises(ValueError):
        FN.linear_cross_entropy(h, w, lab[:3])
    with pytest.raises(ValueError):
        FN.linear_cross_entropy(h, w, lab.int())
    with pytest.raises(TypeError):
        FN.linear_cross_entropy(h, w.float(), lab)


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    h, w, lab = make(4, 64, 100, "cuda")
    with pytest.raises(RuntimeError):
        FN.linear_cross_entropy(h.float(), w.float(), lab)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        FN.linear_cross_entropy(h[:, :60].clone(memory_format=torch.contiguous_format).new_zeros(4, 64)[:, :60],
                                w.new_zeros(100, 64)[:, :60], lab)
    with pytest.raises(RuntimeError):
        FN.linear_cross_entropy(h, w, lab.cpu())
