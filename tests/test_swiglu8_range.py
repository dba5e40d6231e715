"""SwiGLU on 8-bit activations where a product of two inputs leaves fp32's range and the result does
not: with the gate far below zero the sigmoid is 0 and so are the output and all gradients."""
import pytest
import torch

from femtotron_b200.ops import act8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gate,up", [(-1e20, 1e20), (-1e20, -1e20), (-1e30, 3e38), (-200.0, 3e38)])
def test_output_of_a_closed_gate_is_zero(device, gate, up):
    gu = torch.tensor([gate, up]).to(torch.bfloat16).repeat_interleave(64).repeat(3, 1).to(device)
    h, a = act8.swiglu(gu, 32)
    assert bool((h == 0).all())
    _, h8 = act8.swiglu_bwd(torch.ones_like(h), a)
    assert bool((h8 == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("gate,up,dh", [(-1e20, 1e20, 1e20), (-1e30, -3e38, 1e3), (-200.0, 1e25, -1e25)])
def test_gradients_of_a_closed_gate_are_zero(device, gate, up, dh):
    gu = torch.tensor([gate, up]).to(torch.bfloat16).repeat_interleave(64).repeat(3, 1).to(device)
    _, a = act8.swiglu(gu, 32)
    dgu, _ = act8.swiglu_bwd(torch.full((3, 64), dh, device=device).to(torch.bfloat16), a)
    assert bool((dgu == 0).all())
