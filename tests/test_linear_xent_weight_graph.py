"""A head weight that is itself computed: its gradient flows on to what it was computed from.  (A
parameter's goes to its gradient sink.)

Bounds: d is rounded to bf16 on the GPU (2^-8), the logits are good to 2^-12 of a unit here (hidden
size 64), and dw is rounded to the weight's type, 2^-8 for bf16; the two orders of summing agree to
that."""
import pytest
import torch

from femtotron_b200.ops import functional as FN

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(device):
    g = torch.Generator().manual_seed(0)
    h = torch.randn(40, 64, generator=g).to(torch.bfloat16).to(device)
    master = (torch.randn(300, 64, generator=g) * 0.2).to(device)
    lab = torch.randint(0, 300, (40,), generator=g)
    lab[3] = -100
    return h, master, lab.to(device)


def want(h, w, lab):
    """dw of the summed loss and the magnitudes that it adds, in 64 bits."""
    x = h.double() @ w.double().t()
    d = torch.softmax(x, 1)
    d.scatter_add_(1, lab.clamp(min=0)[:, None], -torch.ones_like(x[:, :1]))
    d *= (lab >= 0)[:, None]
    return d.t() @ h.double(), d.abs().t() @ h.double().abs()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("needs_h", [False, True])
def test_gradient_flows_through_a_computed_weight(device, needs_h):
    h, master, lab = make(device)
    master.requires_grad_()
    w = (2 * master).to(torch.bfloat16)
    dw, mag = want(h, w, lab)
    FN.linear_cross_entropy(h.clone().requires_grad_(needs_h), w, lab, reduction="sum").backward()
    assert master.grad is not None
    err = (master.grad.double() - 2 * dw).abs()
    assert bool((err <= 2 * ((2.0 ** -8 + 2.0 ** -11) * mag + 2.0 ** -7 * dw.abs()) + 1e-30).all())


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_of_a_computed_weight_by_name_and_hook(device):
    h, master, lab = make(device)
    master.requires_grad_()
    w = (2 * master).to(torch.bfloat16)
    seen = []
    w.register_hook(lambda g: seen.append(g))
    loss = FN.linear_cross_entropy(h, w, lab, reduction="sum")
    by_name, = torch.autograd.grad(loss, master, retain_graph=True)
    assert len(seen) == 1 and seen[0].shape == w.shape and seen[0].dtype == w.dtype
    assert torch.equal(by_name, 2 * seen[0].float()) and master.grad is None
    loss.backward()
    assert torch.equal(master.grad, by_name)
