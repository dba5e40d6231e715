"""The backward of the head's cross entropy holds what its workspace bound says: d and all shares of
the hidden gradient but one within ``workspace_bytes`` (or 256 columns of d, where that is more), and
one fp32 sum of the hidden gradient, whose rows may be rounded up to 256, beside them."""
import pytest
import torch

from femtotron_b200.ops import functional as FN
from femtotron_b200.ops import linear_xent as X

MB = 2 ** 20


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,V,workspace", [(1, 4096, 32000, MB), (1, 4096, 64128, X.WORKSPACE_BYTES), (64, 2048, 32000, 8 * MB),
                                             (300, 4096, 32000, 24 * MB), (300, 4096, 32000, 64 * MB),
                                             (300, 4096, 32000, 1), (1021, 1024, 32003, 80 * MB)])
def test_peak_of_the_backward(T, H, V, workspace):
    g = torch.Generator().manual_seed(0)
    h = torch.randn(T, H, generator=g).to(torch.bfloat16).cuda().requires_grad_()
    w = (torch.randn(V, H, generator=g) * H ** -0.5).to(torch.bfloat16).cuda().requires_grad_()
    lab = torch.randint(0, V, (T,), generator=g).cuda()
    FN.linear_cross_entropy(h, w, lab, workspace_bytes=workspace).backward()  # the sinks exist from here on
    loss = FN.linear_cross_entropy(h, w, lab, workspace_bytes=workspace)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    loss.backward()
    peak = torch.cuda.max_memory_allocated() - held
    d = max(workspace, 2 * T * 256)
    rows = T if T <= 128 else -(-T // 256) * 256
    # the gradient that autograd adds to h.grad, and small vectors
    assert peak <= d + 4 * rows * H + 2 * T * H + MB // 4, (peak, d)
