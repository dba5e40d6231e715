"""What the upstream gradient of an ignored row holds stays out of every result."""
import pytest
import torch

from test_linear_xent_row_gradients import DEVICES, IGNORE, INF, check, gradients, make


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("held", [float("nan"), INF, -INF, 1e38, 1e30])
@pytest.mark.parametrize("T", [5, 200])
def test_an_ignored_row_sets_nothing(device, held, T):
    h, w, lab, g = make(T, device)
    lab[1], g[1] = IGNORE, held
    dh, dw = gradients(h, w, lab, g)
    assert bool((dh[1] == 0).all())
    check(h, w, lab, g, dh, dw)


@pytest.mark.parametrize("device", DEVICES)
def test_all_rows_ignored(device):
    h, w, lab, g = make(5, device)
    dh, dw = gradients(h, w, torch.full_like(lab, IGNORE), g * INF)
    assert bool((dh == 0).all()) and bool((dw == 0).all())
