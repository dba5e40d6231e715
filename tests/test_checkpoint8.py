"""Activation checkpoints in 8 bits behave like the 16-bit ones in everything but the kept values: graphs
that are used twice, gradients asked for by name, further differentiable arguments, outputs that
are not a tensor, hidden states by keyword, dropout.

Oracle: the same module on the dequantised hidden states, differentiated without a checkpoint.  The two
run the same operations on the same values, so they are equal bit for bit, except where torch adds
gradients in another order (1e-6, fp32 sums of a few terms)."""
import pytest
import torch
from torch import nn

from femtotron_b200.ops import act8
from femtotron_b200.training.activation_ckpt import ActivationCheckpointWrapper

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class Block(nn.Module):
    """A layer with a second tensor argument and a choice of outputs."""

    def __init__(self, out="tensor", p=0.0):
        super().__init__()
        self.a, self.b = nn.Linear(64, 96), nn.Linear(96, 64)
        self.out, self.drop = out, nn.Dropout(p)

    def forward(self, hidden_states, residual=None, scale=1.0):
        y = self.drop(self.b(torch.nn.functional.silu(self.a(hidden_states)))) * scale
        y = y if residual is None else y + residual * hidden_states.sum(-1, keepdim=True)
        return {"tensor": y, "tuple": (y, y * 2), "dict": {"y": y, "n": 3}, "list": [y]}[self.out]


def value(out):
    return out["y"] if isinstance(out, dict) else out if torch.is_tensor(out) else sum(out)


def setup(device, **kw):
    torch.manual_seed(0)
    block = Block(**kw).to(device)
    first = nn.Linear(64, 64).to(device)
    x, r, g = (torch.randn(5, 64, device=device) for _ in range(3))
    return block, ActivationCheckpointWrapper(block, bits=8), first, x, r, g


def kept(h):
    return act8.quantize(h.detach()).dequantize().requires_grad_()


@pytest.mark.parametrize("device", DEVICES)
def test_a_kept_graph_serves_two_backward_passes(device):
    block, wrapped, first, x, _, g = setup(device)
    out = wrapped(first(x))
    out.backward(g, retain_graph=True)
    one = [p.grad.clone() for p in block.parameters()]
    out.backward(g)
    assert all(torch.equal(p.grad, 2 * o) for p, o in zip(block.parameters(), one))


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_asked_for_by_name(device):
    block, wrapped, first, x, _, g = setup(device)
    h = first(x)
    got = torch.autograd.grad(wrapped(h), [*block.parameters(), first.weight], g)
    h8 = kept(h)
    want = torch.autograd.grad(block(h8), [*block.parameters(), h8], g)
    assert all(torch.equal(a, b) for a, b in zip(got[:-1], want[:-1]))
    assert torch.allclose(got[-1], want[-1].t() @ x, rtol=1e-5, atol=1e-6)
    assert all(p.grad is None for p in block.parameters())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("by", ["position", "keyword"])
def test_a_second_differentiable_argument(device, by):
    """Its graph is shared with the first one's, as a layer's residual is."""
    block, wrapped, first, x, r, g = setup(device)
    r = r.clone().requires_grad_()
    h = first(x)
    res = h * r
    (wrapped(h, res) if by == "position" else wrapped(h, residual=res)).backward(g)
    got = [p.grad.clone() for p in block.parameters()], r.grad, first.weight.grad
    h8, res8 = kept(h), res.detach().clone().requires_grad_()
    want = torch.autograd.grad(block(h8, res8), [*block.parameters(), h8, res8], g)
    assert all(torch.equal(a, b) for a, b in zip(got[0], want))
    assert torch.allclose(got[1], want[-1] * h.detach(), rtol=1e-5, atol=1e-6)
    dh = want[-2] + want[-1] * r.detach()
    assert torch.allclose(got[2], dh.t() @ x, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("out", ["tensor", "tuple", "dict", "list"])
def test_outputs_of_any_kind(device, out):
    block, wrapped, first, x, _, g = setup(device, out=out)
    h = first(x)
    got = wrapped(h)
    assert type(got) is type(block(h)) and torch.equal(value(got), value(block(h)))  # the forward is exact
    value(got).backward(g)
    h8 = kept(h)
    want = torch.autograd.grad(value(block(h8)), list(block.parameters()), g)
    assert all(torch.equal(p.grad, w) for p, w in zip(block.parameters(), want))


@pytest.mark.parametrize("device", DEVICES)
def test_hidden_states_by_keyword_and_without_a_gradient_are_kept_in_8_bits(device):
    block, wrapped, _, x, _, g = setup(device)
    h8 = kept(x)
    want = torch.autograd.grad(block(h8), list(block.parameters()), g)
    exact = torch.autograd.grad(block(x), list(block.parameters()), g)
    assert not torch.equal(want[0], exact[0])
    for call in (lambda: wrapped(hidden_states=x), lambda: wrapped(x), lambda: wrapped(scale=1.0, hidden_states=x)):
        block.zero_grad()
        call().backward(g)
        assert all(torch.equal(p.grad, w) for p, w in zip(block.parameters(), want))


@pytest.mark.parametrize("device", DEVICES)
def test_dropout_repeats_itself(device):
    block, wrapped, first, x, _, g = setup(device, p=0.5)
    h = first(x)
    torch.manual_seed(7)
    out = wrapped(h)
    torch.rand(11, device=device)  # moves the generator on
    out.backward(g)
    h8 = kept(h)
    torch.manual_seed(7)
    want = torch.autograd.grad(block(h8), list(block.parameters()), g)
    assert all(torch.equal(p.grad, w) for p, w in zip(block.parameters(), want))


@pytest.mark.gpu
def test_memory_between_the_passes_is_that_of_8_bits():
    n = 2 ** 25  # hidden values: 64 MB in bf16, 33 in 8 bits with their scales
    wrapped = ActivationCheckpointWrapper(nn.Linear(1024, 8, device="cuda", dtype=torch.bfloat16), bits=8)
    shift = torch.randn(1024, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    torch.ones(8, 8, device="cuda", dtype=torch.bfloat16) @ torch.ones(8, 8, device="cuda", dtype=torch.bfloat16)
    before = torch.cuda.memory_allocated()
    h = torch.zeros(n // 1024, 1024, device="cuda", dtype=torch.bfloat16) + shift  # a sum keeps nothing
    out = wrapped(h)
    del h
    # beside the codes: 8 values per row, and the allocator's rounding
    assert torch.cuda.memory_allocated() - before <= n * (1 + 4 / 128) + 2 * 8 * n // 1024 + 2 ** 20
    out.sum().backward()


def test_reentrant_checkpoints_are_refused_in_8_bits():
    with pytest.raises(ValueError, match="use_reentrant"):
        ActivationCheckpointWrapper(Block(), bits=8, use_reentrant=True)
