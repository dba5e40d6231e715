"""Rows of the head's cross entropy where a small error shows: words predicted with near
certainty, logits made by a single channel, a vocabulary of one word.

Oracle: 64-bit logits of the same operands.  Bounds.  The loss is (m - x_label) + log s with s the
sum of exp(x - m), so it cannot be negative; where the label's logit is the largest the first
term is exactly 0 and s is 1 plus the other words' share, rounded to fp32 a dozen times at most
(2^-20 in all).  A logit is off by at most 2^-15 of itself (512 steps of an accumulator that
truncates, 2^-24 of the sum each), so with logits below 64 the other words' share, and with it a small
loss, is good to 2^-9 of itself.  In the backward, p of the label is 2^(x unit - lse log2 e): five
roundings of 2^-24 of a number of lse's size (2^-21 |lse|), and an exponential good to 2^-20."""
import math

import pytest
import torch

from femtotron_b200.ops import functional as FN

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def one_channel(T, H, V, channel, label, others, device):
    """Logits `label` and `others`, each a product in one channel."""
    h = torch.zeros(T, H, dtype=torch.bfloat16, device=device)
    w = torch.zeros(V, H, dtype=torch.bfloat16, device=device)
    h[:, channel] = 1
    w[:, channel] = others
    w[V // 2, channel] = label
    return h, w, torch.full((T,), V // 2, device=device)


def certain(T, H, V, device, logit=40.0, seed=0):
    """Each token's label stands `logit` above words spread by about one."""
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(T, H, generator=g)
    w = torch.randn(V, H, generator=g) / math.sqrt(H)
    lab = torch.randperm(V, generator=g)[:T]
    w[lab] += logit * h / h.pow(2).sum(1, keepdim=True)
    return h.to(torch.bfloat16).to(device), w.to(torch.bfloat16).to(device), lab.to(device)


def truth(h, w, lab):
    """Losses in 64 bits, from the other words' share."""
    x = h.double() @ w.double().t()
    t = x.gather(1, lab[:, None])
    return torch.log1p(torch.exp(x - t).scatter(1, lab[:, None], 0.0).sum(1))


def check_losses(h, w, lab):
    got = FN.linear_cross_entropy(h, w, lab, reduction="none")
    want = truth(h, w, lab)
    assert bool((got >= 0).all()), float(got.min())
    assert bool(((got.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -9 * want).all()), float(got.max())
    # the same in the form that keeps what the backward needs
    again = FN.linear_cross_entropy(h.clone().requires_grad_(), w, lab, reduction="none")
    assert bool((again >= 0).all())
    assert bool(((again.double() - want).abs() <= 2.0 ** -20 + 2.0 ** -9 * want).all()), float(again.max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 2, 3, 130, 300])
@pytest.mark.parametrize("label,others", [(-32.0, -64.0), (32.0, -8.0), (9.0, 0.0)])
@pytest.mark.parametrize("channel", [0, 4095])
def test_one_dominating_channel(device, T, label, others, channel):
    check_losses(*one_channel(T, 4096, 600, channel, label, others, device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,H", [(1, 4096), (2, 1000), (3, 8192), (100, 4096), (300, 4096), (130, 8192)])
def test_nearly_certain_words(device, T, H):
    check_losses(*certain(T, H, 700, device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 2, 3, 200])
def test_a_vocabulary_of_one_word_costs_nothing(device, T):
    h, w, _ = certain(T, 4096, 700, device)
    losses = FN.linear_cross_entropy(h, w[:1], torch.zeros(T, dtype=torch.long, device=device), reduction="none")
    assert bool((losses == 0).all()), float(losses.abs().max())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [1, 2, 3, 130, 300])
@pytest.mark.parametrize("label,others", [(-32.0, -64.0), (32.0, -8.0)])
@pytest.mark.parametrize("channel", [0, 4095])
def test_a_certain_word_leaves_no_gradient(device, T, label, others, channel):
    h, w, lab = one_channel(T, 4096, 600, channel, label, others, device)
    h.requires_grad_()
    w.requires_grad_()
    FN.linear_cross_entropy(h, w, lab, reduction="sum").backward()
    eps = 2.0 ** -21 * abs(label) + 2.0 ** -20  # of p at the label; the others' share is below 1e-9
    assert float(h.grad.abs().max()) <= eps * abs(label) + 1e-6
    assert float(w.grad.abs().max()) <= eps * T + 1e-6


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T,H", [(300, 4096), (130, 8192)])
def test_mean_loss_of_wide_hidden_states(device, T, H):
    """The accumulator's truncation comes to 2^-26 of a logit per 16 products, 7.6e-6 at 8192, and the
    mean loss moves with it by the logits' variance, 6.25 here: 4.8e-5 if it were left in.  The
    correction is good to a tenth (5e-6 of the loss), and fp32 gives lse to 2^-21 (5e-6 in all for
    the mean, whose roundings go either way)."""
    g = torch.Generator().manual_seed(3)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16).to(device)
    w = (torch.randn(5000, H, generator=g) * (2.5 / math.sqrt(H))).to(torch.bfloat16).to(device)
    lab = torch.randint(0, 5000, (T,), generator=g).to(device)
    off = FN.linear_cross_entropy(h, w, lab, reduction="none").double() - truth(h, w, lab)
    assert abs(float(off.mean())) <= 1e-5, float(off.mean())
