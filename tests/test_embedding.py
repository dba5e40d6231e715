"""Embedding lookup with a factor and its gradient by sorted tokens, on the CPU and, marked gpu, through the kernels."""
import pytest
import torch

from femtotron_b200.ops import embedding as E
from femtotron_b200.ops import functional as FN

gpu = pytest.mark.gpu
DEVICES = ["cpu", pytest.param("cuda", marks=gpu)]
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def ids_of(kind, T, words, g):
    return {"uniform": torch.randint(0, words, (T,), generator=g), "one": torch.full((T,), words // 2),
            "few": torch.randint(0, 3, (T,), generator=g) * (words // 3),
            "rising": torch.arange(T) % words,
            "outside": torch.randint(-words, 2 * words, (T,), generator=g)}[kind]


def case(device, T, V, H, kind, dtype, seed=0, wide=True):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, H, generator=g).to(dtype).to(device)
    ids = ids_of(kind, T, V, g).to(torch.int64 if wide else torch.int32).to(device)
    dout = torch.randn(T, H, generator=g).to(dtype).to(device)
    return ids, w, dout


def grad64(ids, dout, V, vstart, scale):
    local = ids.long() - vstart
    has = (local >= 0) & (local < V)
    dw = torch.zeros(V, dout.shape[1], dtype=torch.float64, device=dout.device)
    size = torch.zeros_like(dw)
    dw.index_put_((local[has],), dout[has].double() * scale, accumulate=True)
    size.index_put_((local[has],), dout[has].double().abs() * scale, accumulate=True)
    return dw, size


SIZES = [(1, 5, 8), (31, 40, 16), (33, 7, 1), (64, 1000, 130), (700, 1025, 264), (2049, 300, 1023)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["uniform", "one", "few", "rising", "outside"])
@pytest.mark.parametrize("T,V,H", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_lookup_and_gradient(device, kind, T, V, H, dtype):
    ids, w, dout = case(device, T, V, H, kind, dtype, wide=T % 2 == 0)
    vstart, scale = (V // 3, 11.25) if kind == "outside" else (0, 1.0)
    out = E.lookup(ids, w, vstart, scale)
    local = ids.long() - vstart
    has = (local >= 0) & (local < V)
    want = torch.where(has[:, None], w[local.clamp(0, V - 1)].double() * scale, torch.zeros(1, dtype=torch.float64, device=device))
    assert ((out.double() - want).abs() <= HALF[dtype] * want.abs()).all()
    want, size = grad64(ids, dout, V, vstart, scale)
    for to in (torch.float32, torch.bfloat16, torch.float16):
        if to not in (torch.float32, dtype):
            continue
        got = torch.full((V, H), 5.0, dtype=to, device=device)
        E.sorted_grad(ids, dout, got, False, vstart, scale)
        # fp32 sums of at most T terms in pieces of 32, the pieces one after the other; one rounding
        tol = (32 + T / 32 + 2) * 2 ** -24 * size + HALF[to] * want.abs() + (2 ** -25 if to == torch.float16 else 0)
        assert ((got.double() - want).abs() <= tol).all()
        more = got.clone()
        E.sorted_grad(ids, dout, more, True, vstart, scale)
        both = got.double() + want
        tol = (32 + T / 32 + 3) * 2 ** -24 * (size + got.double().abs()) + HALF[to] * both.abs() + (2 ** -25 if to == torch.float16 else 0)
        assert ((more.double() - both).abs() <= tol).all()


@pytest.mark.parametrize("device", DEVICES)
def test_sinks(device):
    ids, w, dout = case(device, 100, 50, 24, "uniform", torch.bfloat16)
    ids, dout = ids.view(4, 25), dout.view(4, 25, 24)
    want, size = grad64(ids.view(-1), dout.view(-1, 24), 50, 0, 4.0)
    # the gradient's own buffer in the weight's type, then added to
    p = torch.nn.Parameter(w.clone())
    FN.embedding(ids, p, scale=4.0).backward(dout)
    assert ((p.grad.double() - want).abs() <= HALF[torch.bfloat16] * want.abs() + 2 ** -18 * size).all()
    first = p.grad.clone()
    FN.embedding(ids, p, scale=4.0).backward(dout)
    assert ((p.grad.double() - first.double() - want).abs() <= HALF[torch.bfloat16] * 2.1 * want.abs() + 2 ** -18 * size).all()
    # an fp32 buffer that is overwritten first
    p = torch.nn.Parameter(w.clone())
    p.main_grad, p.grad_overwrite = torch.full((50, 24), 9.0, device=device), True
    told = []
    p._ft_grad_ready = lambda: told.append(1)
    FN.embedding(ids, p, scale=4.0).backward(dout)
    assert ((p.main_grad.double() - want).abs() <= 2 ** -18 * size).all() and p.grad is None and told == [1]
    FN.embedding(ids, p, scale=4.0).backward(dout)
    assert ((p.main_grad.double() - 2 * want).abs() <= 2 ** -17 * size).all()
    # a weight that was computed: the gradient flows on
    leaf = torch.nn.Parameter(w.clone())
    FN.embedding(ids, leaf * 2, scale=4.0).backward(dout)
    assert ((leaf.grad.double() - 2 * want).abs() <= 3 * HALF[torch.bfloat16] * 2 * want.abs() + 2 ** -17 * size).all()


@pytest.mark.parametrize("device", DEVICES)
def test_empty_and_refusals(device):
    ids, w, dout = case(device, 8, 10, 16, "uniform", torch.float32)
    p = torch.nn.Parameter(w.clone())
    out = FN.embedding(ids[:0], p)
    assert out.shape == (0, 16)
    out.sum().backward()
    assert not p.grad.any()
    with pytest.raises(TypeError, match="int32 or int64"):
        FN.embedding(ids.float(), p)
    with pytest.raises(ValueError, match="contiguous"):
        FN.embedding(ids, w.t())
    with pytest.raises(ValueError, match="contiguous"):
        FN.embedding(ids, w[0])
    if device == "cuda":
        with pytest.raises(ValueError, match="ids are on"):
            FN.embedding(ids.cpu(), p)


@gpu
@pytest.mark.parametrize("T,V", [(9000, 128257), (40000, 1200000), (5000, 1023), (5000, 1024), (8192, 262143), (8193, 262144), (7000, 1200000)])
def test_gpu_large_vocabularies(T, V):
    g = torch.Generator().manual_seed(1)
    ids = (torch.exp(torch.rand(T, generator=g) * 12) - 1).long().clamp_(max=V - 1).cuda()
    ids[::7] = V - 1
    ids[1::50] = V  # of another shard
    dout = torch.randn(T, 8, generator=g).cuda()
    got = torch.empty(V, 8, device="cuda")
    E.sorted_grad(ids, dout, got, False)
    again = torch.empty_like(got)
    E.sorted_grad(ids, dout, again, False)
    want, size = grad64(ids, dout, V, 0, 1.0)
    assert ((got.double() - want).abs() <= (34 + T / 32) * 2 ** -24 * size + 2 ** -24 * want.abs()).all()
    assert torch.equal(got, again)


@gpu
def test_gpu_strides_streams_and_graphs():
    ids, w, dout = case("cuda", 600, 90, 264, "uniform", torch.bfloat16)
    want = torch.empty(90, 264, device="cuda")
    E.sorted_grad(ids, dout, want, False)
    spread = torch.empty(600, 2, dtype=ids.dtype, device="cuda")
    spread[:, 0] = ids
    wide = torch.empty(600, 300, dtype=dout.dtype, device="cuda")
    wide[:, 1:265] = dout
    got = torch.empty_like(want)
    E.sorted_grad(spread[:, 0], wide[:, 1:265], got, False)
    assert torch.equal(got, want)
    odd = torch.empty(600 * 264 + 1, dtype=dout.dtype, device="cuda")[1:].view(600, 264).copy_(dout)
    E.sorted_grad(ids, odd, got, False)
    assert torch.equal(got, want)
    assert torch.equal(E.lookup(spread[:, 0], w), w[ids])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        E.sorted_grad(ids, dout, got, False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            E.sorted_grad(ids, dout, got, False)
    torch.cuda.current_stream().wait_stream(side)
    ids.copy_(ids.flip(0))
    graph.replay()
    E.sorted_grad(ids, dout, want, False)
    assert torch.equal(got, want)


@gpu
def test_more_ids_than_places_are_refused():
    ids = torch.zeros(1, dtype=torch.int32, device="cuda").expand(2 ** 30 + 1)
    w = torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="at most"):
        E.lookup(ids, w)
    with pytest.raises(RuntimeError, match="at most"):
        E.sorted_grad(ids, torch.zeros(1, 8, device="cuda").expand(2 ** 30 + 1, 8), w, False)


@pytest.mark.parametrize("sink", [False, True])
def test_a_retained_graph_runs_again(sink):
    w = torch.nn.Parameter(torch.arange(12.0).view(4, 3))
    if sink:
        w.main_grad = torch.zeros(4, 3)
    out = FN.embedding(torch.tensor([1, 1, 3]), w, scale=2.0)
    out.sum().backward(retain_graph=True)
    out.sum().backward()
    want = torch.tensor([0.0, 8.0, 0.0, 4.0])[:, None].expand(4, 3)
    assert torch.equal(w.main_grad if sink else w.grad, want)
    assert (w.grad is None) == sink


def test_second_derivatives_are_refused():
    base = torch.randn(4, 3, requires_grad=True)
    out = FN.embedding(torch.tensor([1, 2]), base * 2.0)
    (g,) = torch.autograd.grad(out.square().sum(), base, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
