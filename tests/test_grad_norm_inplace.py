"""Clipping and scaling in place: what autograd saved is known to have changed."""
import pytest
import torch

from femtotron_b200.ops import grad_norm as GN

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]


def coef_of(x):
    return torch.tensor(0.5, device=x.device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("call", [lambda x: GN.clip_grads([x], 1e-3), lambda x: GN.scale_grads([x], coef_of(x)),
                                  lambda x: GN.clip_grads([torch.ones_like(x)], 1e-3, out=[x]),
                                  lambda x: GN.scale_grads([torch.ones_like(x)], coef_of(x), out=[x])])
def test_what_was_saved_for_a_backward_pass_is_known_to_have_changed(device, call):
    w = torch.arange(1.0, 9.0, device=device, requires_grad=True)
    y = w * 2
    out = (y * y).sum()  # keeps y
    call(y.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()
    with torch.inference_mode():  # tensors without a version
        call(torch.ones(4, device=device))
    if device == "cuda":  # what is only read is no other than before
        x = torch.ones(4, device=device)
        GN.sum_of_squares([x])
        GN.clip_grads([x], 1.0, out=[torch.empty_like(x)])
        assert x._version == 0
