"""Clipping and scaling in place: what autograd saved is known to have changed, and a call that is refused changes nothing."""
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


@pytest.mark.parametrize("device", DEVICES)
def test_a_tensor_with_a_value_in_several_places_is_refused_before_anything_is_written(device):
    for wide in (torch.ones(3, 1, device=device).expand(3, 4), torch.ones(1, device=device).expand(5)):
        x = torch.full((7,), 2.0, device=device)
        for call in (lambda: GN.clip_grads([x, wide], 1e-3), lambda: GN.scale_grads([x, wide], coef_of(x)),
                     lambda: GN.clip_grads([x, wide], 1e-3, out=[torch.empty_like(x), wide]),
                     lambda: GN.scale_grads([wide, x], coef_of(x), out=[wide, x])):
            with pytest.raises(RuntimeError, match="single memory location"):
                call()
            assert (x == 2).all() and (wide == 1).all()
        GN.clip_grads([x, wide], 1e-3, out=[torch.empty_like(x), torch.empty(wide.shape, device=device)])  # read, not written


@gpu
def test_gpu_strided_outputs_that_share_memory_are_refused():
    base = torch.ones(8, 6, device="cuda")
    a, b = base[:, ::2], base[:, 1::2]
    GN.clip_grads([a, b], 1.0)  # columns in turn: nothing is shared
    assert abs(base.norm().item() - 1) < 1e-5
    for pair in ([a, a], [a, base[:, :5]], [base, a], [a, base]):
        keep = base.clone()
        with pytest.raises(RuntimeError, match="share"):
            GN.clip_grads(pair, 1e-3)
        with pytest.raises(RuntimeError, match="share"):
            GN.scale_grads([torch.ones_like(x) for x in pair], coef_of(base), out=pair)
        assert torch.equal(base, keep)


@pytest.mark.parametrize("device", DEVICES)
def test_sums_of_squares_of_more_slots_than_a_launch_has(device):
    from femtotron_b200.ops import kernels as K
    out = torch.ones(11, device=device)
    K.sumsq_multi([torch.ones(3, device=device), torch.ones(4, 2, device=device).t(), torch.ones(5, device=device).bfloat16()], [0, 9, 9], out)
    assert out.tolist() == [4, 1, 1, 1, 1, 1, 1, 1, 1, 14, 1]
    assert K.sumsq_multi([], [], out) is out
