"""In-place rotation of memory that is not one value per element: refused, since every element would be
turned once for each name it has (on the GPU by threads that race).  What only lies close together is
taken."""
import pytest
import torch

from femtotron_b200.ops import rotary

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def tables(device):
    return rotary.rotary_tables(8, 16, device=device)


def heads(device, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(0)).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["q", "k"])
@pytest.mark.parametrize("how", ["head", "batch", "token", "window"])
def test_a_tensor_that_overlaps_itself_is_refused(device, which, how):
    x = heads(device, 2, 3, 4, 8)
    y = {"head": lambda: x[:, :, :1].expand(2, 3, 4, 8), "batch": lambda: x[:1].expand(2, 3, 4, 8),
         "token": lambda: x[:, :1].expand(2, 3, 4, 8),
         "window": lambda: x.flatten().as_strided((2, 3, 4, 8), (96, 32, 4, 1))}[how]()
    q, k = (y, heads(device, 2, 3, 2, 8)) if which == "q" else (heads(device, 2, 3, 5, 8), y)
    before = q.clone(), k.clone()
    with pytest.raises(RuntimeError, match="more than once"):
        rotary.rotary_qk(q, k, *tables(device), inplace=True)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    # copies are fine
    oq, ok = rotary.rotary_qk(q, k, *tables(device))
    want = rotary.rotary_qk(q.contiguous(), k.contiguous(), *tables(device))
    assert torch.equal(oq, want[0]) and torch.equal(ok, want[1])


@pytest.mark.parametrize("device", DEVICES)
def test_q_and_k_with_heads_in_common_are_refused(device):
    x = heads(device, 2, 3, 6, 8)
    first = x.transpose(1, 2).contiguous().transpose(1, 2)
    for y in (x, first):
        before = y.clone()
        for q, k in ((y, y), (y[:, :, :4], y[:, :, 3:]), (y[:, :, :4], y[:, :, 2:3]), (y[:, :, 2:3], y[:, :, :4]),
                     (y[..., :8], y[:, :, 5:])):
            with pytest.raises(RuntimeError, match="more than once"):
                rotary.rotary_qk(q, k, *tables(device), inplace=True)
        assert torch.equal(y, before)


@pytest.mark.parametrize("device", DEVICES)
def test_neighbours_in_one_tensor_are_taken(device):
    x = heads(device, 2, 3, 6, 16)
    views = [(x[:, :, :4, :8], x[:, :, 4:, :8]), (x[:, :, 4:, :8], x[:, :, :4, :8]), (x[..., :8], x[..., 8:]),
             (x[:, :, ::2, :8], x[:, :, 1::2, :8]), (x[:1, :, :, :8], x[1:, :, :, :8]),
             (x[:, :, :5, :8], x[:, :, 5:, :8]), (x[:, :, :1, 8:], x[:, :, 1:2, 8:])]
    first = x.transpose(1, 2).contiguous().transpose(1, 2)
    views += [(first[:, :, :4, :8], first[:, :, 4:, :8]), (first[:, :, 3:, 8:], first[:, :, :3, 8:])]
    for q, k in views:
        want = rotary.rotary_qk(q, k, *tables(device))
        keep = q.clone(), k.clone()
        rotary.rotary_qk(q, k, *tables(device), inplace=True)
        assert torch.equal(q, want[0]) and torch.equal(k, want[1])
        q.copy_(keep[0])
        k.copy_(keep[1])
