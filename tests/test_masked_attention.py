"""Masked attention (documents, padding, window, prefix; capped scores, bias of distance) against its
formulas in 64 bits, on the CPU and, marked gpu, through the sm_100a kernels."""
import math

import pytest
import torch

from femtotron_b200.ops import check_kernel_errors
from femtotron_b200.ops import masked_attention as MA
from femtotron_b200.ops.matmul import linear_fwd

U16 = torch.finfo(torch.bfloat16).eps / 2  # one rounding to bf16, relative


def visible(S, *, causal=True, window=None, docs=None, prefix=None):
    """[S, S] by the definition, element by element."""
    out = torch.zeros(S, S, dtype=torch.bool)
    first = [0] * S
    for i in range(1, S):
        first[i] = first[i - 1] if docs is None or docs[i] == docs[i - 1] else i
    for i in range(S):
        for j in range(S):
            if first[i] != first[j] or (docs is not None and docs[i] < 0):
                continue
            lead = causal and prefix is not None and all(bool(prefix[t]) for t in range(first[j], j + 1))
            out[i, j] = (not causal or j <= i or lead) and (window is None or abs(i - j) < window)
    return out


def reference(q, k, v, do, vis, scale, softcap, slopes):
    """(o, dq, dk, dv, and the root-sum-square sizes of their terms) in 64 bits."""
    B, S, nq, d = q.shape
    n = nq // k.shape[2]
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, do))
    k, v = k.repeat_interleave(n, 1), v.repeat_interleave(n, 1)
    x = q @ k.transpose(-1, -2) * scale
    keep = torch.ones_like(x)
    if softcap:
        t = torch.tanh(x / softcap)
        x, keep = softcap * t, 1 - t * t
    if slopes is not None:
        i = torch.arange(S, device=q.device)
        x = x - slopes.double().view(1, nq, 1, 1) * (i[:, None] - i).abs()
    vis = vis.to(q.device)[:, None]
    p = torch.nan_to_num(torch.softmax(x.masked_fill(~vis, -math.inf), -1))
    dp = do @ v.transpose(-1, -2)
    o = p @ v
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * keep
    # what a relative rounding of p, ds and of the row sums do o can add up to
    grow = p.abs() * ((do * o).abs().sum(-1, keepdim=True)) * keep + ds.abs()

    def group(x):
        return x.view(B, nq // n, n, S, d).sum(2).transpose(1, 2)
    res = [o.transpose(1, 2), (ds @ k * scale).transpose(1, 2), group(ds.transpose(-1, -2) @ q * scale),
           group(p.transpose(-1, -2) @ do)]
    size = [(p @ v.abs()).transpose(1, 2), (grow @ k.abs() * scale).transpose(1, 2),
            group(grow.transpose(-1, -2) @ q.abs() * scale), group(p.transpose(-1, -2) @ do.abs())]
    return res, size


def make(B, S, nq, nkv, d, seed, device, dtype):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, S, h, d, generator=g).to(dtype).to(device) for h in (nq, nkv, nkv, nq))
    return q, k, v, do


def mask_parts(kind, B, S, seed):
    """Arguments of attention_mask for a kind of mask."""
    g = torch.Generator().manual_seed(seed)
    docs = (torch.rand(B, S, generator=g) < 0.05).cumsum(1).int()
    kept = (S * (0.5 + 0.5 * torch.rand(B, 1, generator=g))).long()
    padded = torch.where(torch.arange(S) < kept, docs, torch.full_like(docs, -1))
    marks = (torch.rand(B, S, generator=g) < 0.9)
    return {"causal": {}, "full": dict(causal=False), "window": dict(window=37),
            "docs": dict(docs=docs), "padded": dict(docs=padded), "prefix": dict(prefix=marks),
            "all": dict(docs=padded.long(), prefix=marks, window=29),
            "docs both ways": dict(docs=padded, causal=False, window=50),
            "nothing": dict(docs=torch.full((B, S), -1, dtype=torch.int32))}[kind]


def run(q, k, v, do, mask, **kw):
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    o = MA.masked_attention(*leaves, mask, **kw)
    o.backward(do)
    return [o.detach(), *[x.grad for x in leaves]]


KINDS = ["causal", "full", "window", "docs", "padded", "prefix", "all", "docs both ways", "nothing"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S", [1, 5, 130])
def test_mask_intervals(kind, S):
    B = 2
    parts = mask_parts(kind, B, S, 3)
    m = MA.attention_mask(B, S, **parts)
    for b in range(B):
        one = {n: x[b] if torch.is_tensor(x) else x for n, x in parts.items()}
        assert torch.equal(MA._visible(m)[min(b, m.batch - 1)], visible(S, **one))
    lo, hi = m.rows.view(m.batch, -1, 128, 2).unbind(-1)
    assert torch.equal(m.tiles, torch.stack([lo.amin(-1), lo.amax(-1), hi.amin(-1), hi.amax(-1)], -1))


# fp32 on the CPU: sums of up to S terms, a few roundings each; 64 units in the last place of the terms'
# absolute sum covers them
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (3.0, False), (0.0, True), (3.0, True)])
def test_cpu_against_64_bits(kind, softcap, bias):
    B, S, nq, nkv, d = 2, 61, 6, 2, 12
    q, k, v, do = make(B, S, nq, nkv, d, 1, "cpu", torch.float32)
    parts = mask_parts(kind, B, S, 5)
    mask = MA.attention_mask(B, S, **parts)
    slopes = MA.alibi_slopes(nq) if bias else None
    got = run(q, k, v, do, mask, softcap=softcap, slopes=slopes)
    vis = MA._visible(mask).expand(B, S, S)
    want, size = reference(q, k, v, do, vis, 1 / math.sqrt(d), softcap, slopes)
    for x, y, z in zip(got, want, size):
        assert ((x.double() - y).abs() <= 64 * torch.finfo(torch.float32).eps * (z + y.abs())).all()


def test_cpu_gradients_against_differences():
    B, S, nq, nkv, d = 1, 7, 2, 1, 4
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(B, S, h, d, generator=g) for h in (nq, nkv, nkv))
    docs = torch.tensor([[0, 0, 0, 1, 1, -1, -1]], dtype=torch.int32)
    mask = MA.attention_mask(B, S, docs=docs)
    do = torch.randn(B, S, nq, d, generator=g)
    got = run(q, k, v, do, mask, softcap=2.0, slopes=MA.alibi_slopes(nq))
    h = 1e-2
    for n, x in enumerate((q, k, v)):
        flat = x.view(-1)
        for e in range(0, flat.numel(), 5):
            keep = flat[e].item()
            ends = []
            for step in (h, -h):
                flat[e] = keep + step
                ends.append((MA.masked_attention(q, k, v, mask, softcap=2.0, slopes=MA.alibi_slopes(nq)) * do).sum().item())
            flat[e] = keep
            # the difference quotient is off by h^2 times third derivatives of order ten, and by fp32 noise / h
            assert abs((ends[0] - ends[1]) / (2 * h) - got[n + 1].view(-1)[e].item()) < 5e-3


def test_padding_may_hold_nan():
    B, S = 1, 9
    q, k, v, do = make(B, S, 2, 1, 4, 0, "cpu", torch.float32)
    docs = torch.tensor([[-1, 0, 0, 0, 1, 1, 1, -2, -2]], dtype=torch.int32)
    mask = MA.attention_mask(B, S, docs=docs)
    clean = run(q, k, v, do, mask)
    dead = docs[0] < 0
    for x in (q, k, v, do):
        x[:, dead] = float("nan")
    for x, y in zip(run(q, k, v, do, mask), clean):
        assert torch.equal(x, y) and not x[:, dead].any()


def test_second_derivatives_are_refused():
    q, k, v, do = make(1, 5, 2, 1, 4, 0, "cpu", torch.float32)
    q.requires_grad_()
    do.requires_grad_()
    g, = torch.autograd.grad(MA.masked_attention(q, k, v, MA.attention_mask(1, 5)), q, do, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_slopes_and_document_ids():
    assert torch.equal(MA.alibi_slopes(8), torch.tensor([2.0 ** -i for i in range(1, 9)]))
    assert MA.alibi_slopes(12).shape == (12,)
    ids = torch.tensor([[5, 2, 7, 7, 2, 2, 1]])
    assert MA.document_ids(ids, 2).tolist() == [[0, 0, 1, 1, 1, 2, 3]]


def test_refusals():
    B, S, nq, nkv, d = 2, 6, 4, 2, 8
    q, k, v, _ = make(B, S, nq, nkv, d, 0, "cpu", torch.float32)
    mask = MA.attention_mask(B, S)
    with pytest.raises(ValueError, match="window"):
        MA.attention_mask(B, S, window=0)
    with pytest.raises(ValueError, match="prefix"):
        MA.attention_mask(B, S, causal=False, prefix=torch.ones(B, S, dtype=torch.bool))
    with pytest.raises(ValueError, match="docs of shape"):
        MA.attention_mask(B, S, docs=torch.zeros(B, S + 1, dtype=torch.int32))
    with pytest.raises(TypeError, match="docs must be"):
        MA.attention_mask(B, S, docs=torch.zeros(B, S))
    with pytest.raises(TypeError, match="prefix must be"):
        MA.attention_mask(B, S, prefix=torch.zeros(B, S, dtype=torch.int32))
    with pytest.raises(ValueError, match="the mask on"):
        MA.attention_mask(B, S, docs=torch.zeros(B, S, dtype=torch.int32), device="cuda")
    with pytest.raises(ValueError, match="the mask on"):
        MA.attention_mask(B, S, docs=torch.zeros(B, S, dtype=torch.int32),
                          prefix=torch.zeros(B, S, dtype=torch.bool, device="meta"))
    with pytest.raises(ValueError, match="tokens"):
        MA.attention_mask(B, 0)
    with pytest.raises(ValueError, match="tokens"):
        MA.attention_mask(B, MA.MAX_TOKENS + 1)
    with pytest.raises(ValueError, match="do not match"):
        MA.masked_attention(q, k[:, :-1], v[:, :-1], mask)
    with pytest.raises(ValueError, match="evenly"):
        MA.masked_attention(q[:, :, :3], k, v, mask)
    with pytest.raises(TypeError, match="q, k, v are"):
        MA.masked_attention(q, k.double(), v, mask)
    with pytest.raises(ValueError, match="a mask of"):
        MA.masked_attention(q[:, :-1], k[:, :-1], v[:, :-1], mask)
    with pytest.raises(ValueError, match="a mask of"):
        MA.masked_attention(*(x.repeat(2, 1, 1, 1) for x in (q, k, v)), MA.attention_mask(3, S, docs=torch.zeros(3, S, dtype=torch.int32)))
    with pytest.raises(ValueError, match="scale"):
        MA.masked_attention(q, k, v, mask, scale=0.0)
    with pytest.raises(ValueError, match="softcap"):
        MA.masked_attention(q, k, v, mask, softcap=-1.0)
    with pytest.raises(ValueError, match="softcap"):
        MA.masked_attention(q, k, v, mask, softcap=1e-40)
    with pytest.raises(ValueError, match="slopes"):
        MA.masked_attention(q, k, v, mask, slopes=torch.ones(nkv))
    with pytest.raises(ValueError, match="does not hold"):
        MA.masked_attention_packed(torch.zeros(B, S, 5, d), 4, 2, mask)


# ------------------------------------------------------------------------------ GPU
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,S", [(1, 1), (2, 130), (3, 5000), (2, 20000)])
def test_gpu_mask_equals_the_cpu_mask(kind, B, S):
    parts = mask_parts(kind, B, S, 3)
    on_gpu = {n: x.cuda() if torch.is_tensor(x) else x for n, x in parts.items()}
    m, w = MA.attention_mask(B, S, device="cuda", **on_gpu), MA.attention_mask(B, S, **parts)
    assert torch.equal(m.rows.cpu(), w.rows) and torch.equal(m.tiles.cpu(), w.tiles)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,S", [(1, 1), (2, 130), (3, 5000), (1, 262144)])
def test_gpu_order_of_the_tiles(kind, B, S):
    mask = MA.attention_mask(B, S, device="cuda", **{k: v.cuda() if torch.is_tensor(v) else v
                                                     for k, v in mask_parts(kind, B, S, 3).items()})
    t = mask.tiles.long()
    n = t.shape[1]
    begin = torch.arange(n, device="cuda") * 128
    seen_by = torch.stack([((u[:, 3, None] > begin) & (u[:, 0, None] < begin + 128)).sum(0) for u in t])
    at = mask.order.long()
    assert torch.equal(at.sort(-1).values, torch.arange(n, device="cuda").expand(mask.batch, n))
    work = seen_by.gather(1, at)
    assert (work.diff(dim=1) <= 0).all() and (at.diff(dim=1)[work.diff(dim=1) == 0] > 0).all()


def check_gpu(B, S, nq, nkv, d, kind, softcap=0.0, bias=False, seed=1, spread=1.0):
    q, k, v, do = make(B, S, nq, nkv, d, seed, "cuda", torch.bfloat16)
    q = q * spread
    parts = mask_parts(kind, B, S, 5)
    mask = MA.attention_mask(B, S, device="cuda", **{n: x.cuda() if torch.is_tensor(x) else x for n, x in parts.items()})
    slopes = MA.alibi_slopes(nq, "cuda") if bias else None
    got = run(q, k, v, do, mask, softcap=softcap, slopes=slopes)
    again = run(q, k, v, do, mask, softcap=softcap, slopes=slopes)
    check_kernel_errors(q.device)
    rows = mask.rows[:, :S].cpu().long()
    j = torch.arange(S)
    vis = ((j >= rows[..., 0, None]) & (j < rows[..., 1, None])).expand(B, S, S)
    want, size = reference(q, k, v, do, vis, 1 / math.sqrt(d), softcap, slopes)
    for x, y, z, a in zip(got, want, size, again):
        assert torch.equal(x, a)
        # the operand that is rounded to bf16 before its product (p or ds) and, for the gradients, o in the
        # row sums: two roundings of the terms; one of the result; 2^-14 for the fp32 arithmetic between
        assert ((x.double() - y).abs() <= (2 * U16 + 2 ** -14) * z + U16 * y.abs() + 1e-30).all()


@gpu
@pytest.mark.parametrize("kind", KINDS)
def test_gpu_masks(kind):
    check_gpu(2, 300, 4, 2, 64, kind)


@gpu
@pytest.mark.parametrize("softcap,bias", [(3.0, False), (0.0, True), (20.0, True)])
@pytest.mark.parametrize("kind", ["causal", "all", "docs both ways"])
def test_gpu_scores(kind, softcap, bias):
    check_gpu(2, 389, 4, 4, 128, kind, softcap=softcap, bias=bias, spread=2.0)


@gpu
@pytest.mark.parametrize("softcap", [1e-7, 1e-3, 0.2, 1e5])
def test_gpu_caps_of_any_size(softcap):
    # tiny caps make every score +-cap (and zero scores, q = 0, stay 0), large ones change nothing
    q, k, v, do = make(1, 150, 2, 1, 64, 3, "cuda", torch.bfloat16)
    q[:, 10:20] = 0
    mask = MA.attention_mask(1, 150, device="cuda")
    got = run(q, k, v, do, mask, softcap=softcap)
    vis = torch.ones(150, 150, dtype=torch.bool).tril()[None]
    want, size = reference(q, k, v, do, vis, 1 / 8, softcap, None)
    for x, y, z in zip(got, want, size):
        # as check_gpu, and what fp32 loses of 1 - tanh^2 next to 1: 2^-22 of the largest terms
        assert ((x.double() - y).abs() <= (2 * U16 + 2 ** -14) * z + U16 * y.abs() + 2 ** -22 * z.max() + 1e-30).all()


@gpu
@pytest.mark.parametrize("S", [1, 2, 127, 128, 129, 256, 1000])
@pytest.mark.parametrize("nq,nkv,d", [(1, 1, 8), (3, 1, 40), (8, 2, 80), (6, 2, 128), (5, 5, 96)])
def test_gpu_sizes(S, nq, nkv, d):
    check_gpu(1, S, nq, nkv, d, "causal")


@gpu
def test_gpu_long():
    check_gpu(1, 5003, 2, 1, 64, "padded")
    check_gpu(1, 5003, 2, 2, 128, "window")


@gpu
def test_gpu_longest_sequence_and_offsets_past_32_bits():
    B, S, nq, nkv, d, w = 1, MA.MAX_TOKENS, 68, 4, 128, 100
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 60e9:
        pytest.skip("needs 60 GB of free GPU memory")
    g = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randn(B, S, nq, d, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    k, v = (torch.randn(B, S, nkv, d, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_() for _ in range(2))
    assert q.numel() > 2 ** 31
    o = MA.masked_attention(q, k, v, MA.attention_mask(1, S, window=w, device="cuda"))
    do = torch.randn(B, S, nq, d, generator=g, device="cuda", dtype=torch.bfloat16)
    grads = torch.autograd.grad(o, [q, k, v], do)
    check_kernel_errors(q.device)
    for end in (S, 130 * 1024 + 77):  # the last 300 rows and some in the middle, with what they see and what sees them
        a = end - 600
        part = [x.detach()[:, a:end] for x in (q, k, v, do)]
        i = torch.arange(end - a)
        vis = ((i[:, None] >= i) & (i[:, None] - i < w))[None]
        want, size = reference(*part, vis, 1 / math.sqrt(d), 0.0, None)
        for n, (x, y, z) in enumerate(zip([o.detach(), *grads], want, size)):
            rows = slice(300, 600 if end == S or n < 2 else 500)  # later keys are seen from behind the piece
            x, y, z = x[:, a:end][:, rows].double(), y[:, rows], z[:, rows]
            assert ((x - y).abs() <= (2 * U16 + 2 ** -14) * z + U16 * y.abs()).all()


@gpu
@pytest.mark.parametrize("S,nq,nkv,d", [(2100, 8, 1, 64), (1500, 6, 1, 40), (700, 12, 2, 128)])
@pytest.mark.parametrize("kind", ["causal", "padded"])
def test_gpu_many_heads_on_few_keys(S, nq, nkv, d, kind):
    check_gpu(1, S, nq, nkv, d, kind)


@gpu
def test_gpu_padding_may_hold_nan():
    B, S, nq, nkv, d = 2, 700, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 2, "cuda", torch.bfloat16)
    docs = (torch.arange(S, device="cuda") // 90).int().repeat(B, 1)
    docs[0, 150:170] = -1
    docs[1, 500:] = -1
    docs[1, :3] = -1
    mask = MA.attention_mask(B, S, docs=docs)
    clean = run(q, k, v, do, mask)
    dead = docs < 0
    for x in (q, k, v, do):
        x[dead] = float("nan")
    for x, y in zip(run(q, k, v, do, mask), clean):
        assert torch.equal(x, y) and not x[dead].any()


@gpu
@pytest.mark.parametrize("softcap,bias", [(3.0, False), (1e-3, False), (0.0, True), (3.0, True)])
def test_gpu_padding_may_hold_nan_with_other_scores(softcap, bias):
    B, S, nq, nkv, d = 1, 400, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 2, "cuda", torch.bfloat16)
    docs = (torch.arange(S, device="cuda") // 90).int().repeat(B, 1)
    docs[0, 150:170] = -1
    docs[0, 390:] = -1
    mask = MA.attention_mask(B, S, docs=docs)
    kw = dict(softcap=softcap, slopes=MA.alibi_slopes(nq, "cuda") if bias else None)
    clean = run(q, k, v, do, mask, **kw)
    dead = docs < 0
    for bad in (float("nan"), float("inf")):
        for x in (q, k, v, do):
            x[dead] = bad
        for x, y in zip(run(q, k, v, do, mask, **kw), clean):
            assert torch.equal(x, y) and not x[dead].any()


@gpu
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (3.0, False), (0.0, True)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_gpu_nan_reaches_the_rows_that_see_it(which, softcap, bias):
    # one key at every place of a run of 64, so that every way an exponential is taken meets it
    S, nq, nkv, d = 512, 2, 1, 64
    docs = (torch.arange(S, device="cuda") // 256).int().repeat(64, 1)
    mask = MA.attention_mask(64, S, docs=docs)
    q, k, v, do = (x.expand(64, -1, -1, -1).contiguous() for x in make(1, S, nq, nkv, d, 2, "cuda", torch.bfloat16))
    kw = dict(softcap=softcap, slopes=MA.alibi_slopes(nq, "cuda") if bias else None)
    clean = run(q, k, v, do, mask, **kw)
    at = torch.arange(64, device="cuda")
    {"k": k, "v": v}[which][at, 100 + at] = float("nan")
    got = run(q, k, v, do, mask, **kw)
    for name, x, y in zip(("o", "dq", "dk", "dv"), got, clean):
        assert torch.equal(x[:, 256:], y[:, 256:]), name
    sees = torch.arange(256, device="cuda") >= 100 + at[:, None]
    for x in got[:2]:
        assert not x[:, :256][sees].isfinite().any()
    assert not got[2][:, :256].isfinite().any()  # each key is seen by a row that is lost


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_gpu_padding_over_many_tiles(d):
    # padding inside and behind documents in every one of nine tiles, and whole tiles of it
    B, S, nq, nkv = 2, 1100, 4, 2
    q, k, v, do = make(B, S, nq, nkv, d, 7, "cuda", torch.bfloat16)
    i = torch.arange(S, device="cuda")
    docs = torch.where(i % 61 < 7, -1, 0).int().repeat(B, 1)
    docs[1] = torch.where((i > 200) & (i < 900), -1, i // 500).int()
    mask = MA.attention_mask(B, S, causal=False, docs=torch.where(docs < 0, docs, 3 * (i // 61).int()))
    clean = run(q, k, v, do, mask)
    dead = docs < 0
    for x in (q, k, v, do):
        x[dead] = float("nan")
    for x, y in zip(run(q, k, v, do, mask), clean):
        assert torch.equal(x, y) and not x[dead].any()
    check_kernel_errors(q.device)


@gpu
def test_gpu_strides_and_packed_views():
    B, S, nq, nkv, d = 2, 257, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 4, "cuda", torch.bfloat16)
    mask = MA.attention_mask(1, S, device="cuda")
    want = run(q, k, v, do, mask)

    def odd(x):  # one value behind a boundary
        return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view_as(x).copy_(x)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v, do)]
    packed = torch.cat([q, k, v], 2)
    views = [packed[:, :, :nq], packed[:, :, nq:nq + nkv], packed[:, :, nq + nkv:], do]
    for xs in (heads_first, views, [odd(x) for x in (q, k, v, do)]):
        leaves = [x.detach().requires_grad_() for x in xs[:3]]
        o = MA.masked_attention(*leaves, mask)
        got = [o.detach(), *torch.autograd.grad(o, leaves, xs[3])]
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    MA.masked_attention(*leaves, mask).sum().backward()  # an expanded gradient, all strides 0
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, run(q, k, v, torch.ones_like(do), mask)[1:]))
    wide = torch.randn(B, S, nkv, 1, device="cuda", dtype=torch.bfloat16).expand(B, S, nkv, d)
    full = run(q, k, wide.contiguous(), do, mask)
    leaves = [x.detach().requires_grad_() for x in (q, k, wide)]
    o = MA.masked_attention(*leaves, mask)
    assert torch.equal(o, full[0])


@gpu
def test_gpu_in_a_graph_and_on_another_stream():
    B, S, nq, nkv, d = 1, 384, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 6, "cuda", torch.bfloat16)
    docs = (torch.arange(S, device="cuda") // 100).int()[None]
    want = run(q, k, v, do, MA.attention_mask(B, S, docs=docs))
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        def step():
            o = MA.masked_attention(*leaves, MA.attention_mask(B, S, docs=docs))
            return [o, *torch.autograd.grad(o, leaves, do)]
        eager = [x.detach().clone() for x in step()]
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = [x.detach() for x in step()]
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(eager, want):
        assert torch.equal(x, y)
    for shift in (0, 30):
        docs.copy_(((torch.arange(S, device="cuda") + shift) // 100).int()[None])
        graph.replay()
        fresh = run(q, k, v, do, MA.attention_mask(B, S, docs=docs))
        assert all(torch.equal(x, y) for x, y in zip(kept, fresh))


@gpu
def test_gpu_beside_other_work_on_two_streams():
    # blocks of two calls and of products share SMs, their tensor memory and their shared memory
    args = [make(1, 900, 8, 2, 128, seed, "cuda", torch.bfloat16) for seed in (1, 2)]
    mask = MA.attention_mask(1, 900, device="cuda")
    want = [run(*a, mask) for a in args]
    a = torch.randn(2048, 2048, device="cuda", dtype=torch.bfloat16)
    product = linear_fwd(a, a)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(run(*x, mask))
        with torch.cuda.stream(streams[2]):
            again = linear_fwd(a, a)
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(g, w))
        assert torch.equal(again, product)
    check_kernel_errors(a.device)


@gpu
def test_gpu_mask_made_on_the_host_is_refused():
    q, k, v, _ = make(1, 200, 2, 2, 64, 1, "cuda", torch.bfloat16)
    m = MA.attention_mask(1, 200)
    with pytest.raises(ValueError, match="attention_mask"):
        MA.masked_attention(q, k, v, MA.AttentionMask(m.rows.cuda(), m.tiles.cuda(), 200))


@gpu
def test_gpu_refusals():
    q, k, v, _ = make(1, 8, 2, 1, 64, 0, "cuda", torch.bfloat16)
    mask = MA.attention_mask(1, 8, device="cuda")
    with pytest.raises(TypeError, match="bfloat16"):
        MA.masked_attention(q.half(), k.half(), v.half(), mask)
    with pytest.raises(ValueError, match="multiple of 8"):
        MA.masked_attention(q[..., :12], k[..., :12], v[..., :12], mask)
    with pytest.raises(ValueError, match="one device"):
        MA.masked_attention(q, k, v, MA.attention_mask(1, 8))
