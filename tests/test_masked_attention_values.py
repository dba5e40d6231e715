"""Masked attention on the GPU: bits of a row that do not depend on what it cannot see, and combinations of heads, scores and
masks against the formulas in 64 bits."""
import math

import pytest
import torch

from femtotron_b200.ops import masked_attention as MA
from test_masked_attention import U16, check_gpu, make, mask_parts, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("softcap", [30.0, 50.0])
@pytest.mark.parametrize("bad", [1e3, 3e38, math.inf, math.nan])
def test_capped_scores_do_not_depend_on_padding(bad, softcap, bias):
    # scores of N(0, 1): all within 0.7 of the cap, those of the padding far beyond it
    B, S, nq, nkv, d = 1, 400, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 2, "cuda", torch.bfloat16)
    docs = (torch.arange(S, device="cuda") // 90).int().repeat(B, 1)
    docs[0, 150:170] = -1
    docs[0, 390:] = -1
    mask = MA.attention_mask(B, S, docs=docs)
    kw = dict(softcap=softcap, slopes=MA.alibi_slopes(nq, "cuda") if bias else None)
    clean = run(q, k, v, do, mask, **kw)
    dead = docs < 0
    for x in (q, k, v, do):
        x[dead] = bad
    for name, x, y in zip(("o", "dq", "dk", "dv"), run(q, k, v, do, mask, **kw), clean):
        assert torch.equal(x, y), name


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_capped_scores_do_not_depend_on_other_documents(d, bias):
    B, S, nq, nkv, cap = 1, 400, 4, 2, 30.0
    q, k, v, do = make(B, S, nq, nkv, d, 3, "cuda", torch.bfloat16)
    docs = (torch.arange(S, device="cuda") // 90).int()[None]
    mask = MA.attention_mask(B, S, docs=docs)
    kw = dict(softcap=cap, slopes=MA.alibi_slopes(nq, "cuda") if bias else None)
    clean = run(q, k, v, do, mask, **kw)
    other = docs[0] == 1
    q[:, other] *= 16
    k[:, other] *= 16
    for name, x, y in zip(("o", "dq", "dk", "dv"), run(q, k, v, do, mask, **kw), clean):
        assert torch.equal(x[:, ~other], y[:, ~other]), name
        assert not torch.equal(x[:, other], y[:, other])


@pytest.mark.parametrize("cut", [1, 40, 200, 250])
def test_capped_scores_do_not_depend_on_later_tokens(cut):
    B, S, nq, nkv, d = 1, 300, 4, 2, 64
    q, k, v, do = make(B, S, nq, nkv, d, 4, "cuda", torch.bfloat16)
    mask = MA.attention_mask(B, S, device="cuda")
    clean = run(q, k, v, do, mask, softcap=30.0)
    q[:, cut:] *= 16
    k[:, cut:] *= 16
    got = run(q, k, v, do, mask, softcap=30.0)
    for n in (0, 1):  # (dk and dv gather from later rows)
        assert torch.equal(got[n][:, :cut], clean[n][:, :cut])


def test_row_sums_of_more_than_two_to_the_30_rows():
    B, S, nq, nkv, d = 1, MA.MAX_TOKENS, 4104, 1, 8
    assert S * nq > 2 ** 30
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 125e9:
        pytest.skip("needs 125 GB of free GPU memory")
    g = torch.Generator(device="cuda").manual_seed(0)

    def some(heads):
        return torch.empty(B, S, heads, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    q, k, v, do = some(nq).requires_grad_(), some(nkv), some(nkv), some(nq)
    docs = (torch.arange(S, device="cuda") // 64).int()[None]
    o = MA.masked_attention(q, k, v, MA.attention_mask(B, S, docs=docs))
    (dq,) = torch.autograd.grad(o, q, do)
    vis = torch.ones(64, 64, dtype=torch.bool).tril()[None]
    for first in range(S // 16 - 64, S, S // 16):  # documents all over the rows, all heads of each
        part = [x.detach()[:, first:first + 64] for x in (q, k, v, do)]
        want, size = reference(*part, vis, 1 / math.sqrt(d), 0.0, None)
        x, y, z = dq[:, first:first + 64].double(), want[1], size[1]
        assert ((x - y).abs() <= (2 * U16 + 2 ** -14) * z + U16 * y.abs()).all(), first
    del q, k, v, do, o, dq
    torch.cuda.empty_cache()


SCORES = [(3.0, False), (0.0, True), (20.0, True)]


@pytest.mark.parametrize("softcap,bias", SCORES)
@pytest.mark.parametrize("kind", ["causal", "all", "docs both ways", "full"])
@pytest.mark.parametrize("nq,nkv,d", [(6, 2, 64), (12, 2, 80), (8, 1, 128)])
def test_scores_of_grouped_heads(nq, nkv, d, kind, softcap, bias):
    check_gpu(2, 333, nq, nkv, d, kind, softcap=softcap, bias=bias, spread=2.0)


@pytest.mark.parametrize("softcap,bias", SCORES)
@pytest.mark.parametrize("kind", ["padded", "window", "docs both ways", "full"])
@pytest.mark.parametrize("S,nq,nkv,d", [(2100, 8, 1, 64), (1500, 6, 1, 40), (700, 12, 2, 128)])
def test_scores_where_blocks_share_a_group(S, nq, nkv, d, kind, softcap, bias):
    # few key tiles: dk and dv of a key head come from several blocks and are joined
    check_gpu(1, S, nq, nkv, d, kind, softcap=softcap, bias=bias)


@pytest.mark.parametrize("softcap,bias", [(0.0, False), *SCORES])
@pytest.mark.parametrize("kind", ["padded", "full"])
@pytest.mark.parametrize("S,nq,nkv,d", [(300, 4, 2, 64), (1500, 6, 1, 40)])
def test_packed_projections_have_the_same_bits(S, nq, nkv, d, kind, softcap, bias):
    B = 2
    q, k, v, do = make(B, S, nq, nkv, d, 8, "cuda", torch.bfloat16)
    mask = MA.attention_mask(B, S, device="cuda", **{n: x.cuda() if torch.is_tensor(x) else x for n, x in mask_parts(kind, B, S, 5).items()})
    kw = dict(softcap=softcap, slopes=MA.alibi_slopes(nq, "cuda") if bias else None)
    want = run(q, k, v, do, mask, **kw)
    qkv = torch.cat([q, k, v], 2).requires_grad_()
    o = MA.masked_attention_packed(qkv, nq, nkv, mask, **kw)
    o.backward(do)
    assert torch.equal(o, want[0]) and torch.equal(qkv.grad, torch.cat(want[1:], 2))
