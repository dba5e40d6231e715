"""Rotary positions: layouts, parts of the head, scaled frequencies, forward and inverse.

Oracle: a complex multiplication in 64 bits with the fp32 tables.  The kernel computes two
products and a sum in fp32 (at most 3 roundings of 2^-24 of |a| + |b|) and rounds once to the
output type (half a step, at most: 2^-8 bf16, 2^-11 fp16, 2^-24 fp32)."""
import math

import pytest
import torch

from femtotron_b200.ops import rotary
from femtotron_b200.ops.ext import KernelTimeoutError, check_kernel_errors

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def turned(x, cos, sin, pos, interleaved, inverse):
    r = cos.shape[1]
    z = torch.complex(cos.double(), sin.double())[pos.long()][:, :, None]
    z = z.conj() if inverse else z
    x = x.double()
    head, rest = x[..., :2 * r], x[..., 2 * r:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :r], head[..., r:])
    y = torch.complex(a.contiguous(), b.contiguous()) * z
    if interleaved:
        y = torch.stack([y.real, y.imag], -1).flatten(-2)
    else:
        y = torch.cat([y.real, y.imag], -1)
    mag = (a.abs() + b.abs())
    mag = mag.repeat_interleave(2, -1) if interleaved else torch.cat([mag, mag], -1)
    return torch.cat([y, rest], -1), torch.cat([mag, 0 * rest], -1)


def check(got, want, mag, dtype):
    err = (got.double() - want).abs()
    # 6e-8: half the subnormal step of fp16
    bound = HALF_STEP[dtype] * want.abs() + 2.0 ** -22 * mag + (6e-8 if dtype == torch.float16 else 1e-37)
    assert bool((err <= bound).all()), float((err / bound).max())


def inputs(B, S, nq, nkv, d, dtype, device, order, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = nq + 2 * nkv
    if order == "heads first":
        qkv = torch.randn(B, n, S, d, generator=g).to(dtype).to(device).transpose(1, 2)
    elif order == "odd offset":  # rows that start off every vector boundary
        qkv = torch.randn(B, S, n * d + 1, generator=g).to(dtype).to(device)[..., 1:].unflatten(-1, (n, d))
    else:
        qkv = torch.randn(B, S, n, d, generator=g).to(dtype).to(device)
    return qkv, qkv[:, :, :nq], qkv[:, :, nq:nq + nkv]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("B,S,nq,nkv,d,rot,order", [
    (1, 1, 1, 1, 2, 2, "packed"), (2, 3, 4, 2, 64, 64, "packed"), (2, 7, 5, 1, 128, 64, "heads first"),
    (1, 33, 3, 3, 36, 18, "packed"), (3, 2, 2, 1, 80, 80, "odd offset"), (1, 5, 9, 2, 33, 20, "packed"),
    (2, 4, 8, 8, 256, 4, "heads first"), (1, 6, 2, 2, 64, 0, "packed"), (2, 100, 32, 8, 128, 128, "packed")])
def test_against_complex_products(device, dtype, interleaved, inverse, B, S, nq, nkv, d, rot, order):
    qkv, q, k = inputs(B, S, nq, nkv, d, dtype, device, order)
    cos, sin = rotary.rotary_tables(rot, 4000, 500000.0, device=device)
    pos = torch.randint(0, 4000, (B, S), generator=torch.Generator().manual_seed(1)).to(device)
    before = qkv.clone()
    oq, ok = rotary.rotary_qk(q, k, cos, sin, pos, interleaved=interleaved, inverse=inverse)
    assert torch.equal(qkv, before) and oq.is_contiguous() and ok.is_contiguous()
    for got, x in ((oq, q), (ok, k)):
        want, mag = turned(x, cos, sin, pos, interleaved, inverse)
        check(got, want, mag, dtype)
        assert torch.equal(got[..., rot:], x[..., rot:])
    # in place: the same values, and nothing else of the packed projection touched
    iq, ik = rotary.rotary_qk(q, k, cos, sin, pos.to(torch.int32), interleaved=interleaved, inverse=inverse,
                              inplace=True)
    assert iq is q and ik is k
    assert torch.equal(q, oq) and torch.equal(k, ok) and torch.equal(qkv[:, :, nq + nkv:], before[:, :, nq + nkv:])
    if device == "cuda":
        check_kernel_errors(q.device)


@pytest.mark.parametrize("device", DEVICES)
def test_positions_default_shared_and_empty(device):
    _, q, k = inputs(2, 5, 4, 2, 32, torch.float32, device, "packed")
    cos, sin = rotary.rotary_tables(32, 16, device=device)
    base = rotary.rotary_qk(q, k, cos, sin)
    for pos in (torch.arange(5, device=device), torch.arange(5, device=device)[None],
                torch.arange(5, device=device, dtype=torch.int32).expand(2, 5)):
        assert all(torch.equal(a, b) for a, b in zip(base, rotary.rotary_qk(q, k, cos, sin, pos)))
    for B, S, nq, nkv in ((0, 5, 4, 2), (2, 0, 4, 2), (2, 5, 0, 2), (2, 5, 4, 0)):
        e = torch.zeros(B, S, nq, 32, device=device), torch.zeros(B, S, nkv, 32, device=device)
        o = rotary.rotary_qk(*e, cos, sin)
        assert o[0].shape == e[0].shape and o[1].shape == e[1].shape


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_is_the_inverse_and_matches_differences(device, interleaved):
    _, q, k = inputs(1, 4, 2, 1, 8, torch.float32, device, "packed")
    cos, sin = rotary.rotary_tables(6, 50, device=device)
    pos = torch.tensor([[3, 40, 7, 0]], device=device)
    q, k = q.clone().requires_grad_(), k.clone().requires_grad_()
    oq, ok = rotary.rotary(q, k, cos, sin, pos, interleaved=interleaved)
    gq, gk = torch.randn_like(oq), torch.randn_like(ok)
    torch.autograd.backward([oq, ok], [gq, gk])
    want, mag = turned(gq, cos, sin, pos, interleaved, True)
    check(q.grad, want, mag, torch.float32)

    def f(x):
        return float((turned(x, cos, sin, pos, interleaved, False)[0] * gq.double()).sum())
    base = q.detach().double()
    for i in range(8):
        step = torch.zeros_like(base)
        step[0, 1, 1, i] = 1e-5
        assert abs((f(base + step) - f(base - step)) / 2e-5 - float(q.grad[0, 1, 1, i])) < 1e-5


def test_tables_are_exact_far_out():
    cos, sin = rotary.rotary_tables(128, 131072, 500000.0)
    f, _ = rotary.inv_frequencies(128, 500000.0)
    for p in (1, 70001, 131071):
        for i in (0, 1, 17, 63):
            assert abs(float(cos[p, i]) - math.cos(p * float(f[i]))) < 2.0 ** -24
            assert abs(float(sin[p, i]) - math.sin(p * float(f[i]))) < 2.0 ** -24


@pytest.mark.parametrize("scaling", [
    None, {"rope_type": "linear", "factor": 4.0}, {"rope_type": "dynamic", "factor": 2.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 2048},
    {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 2048},
    {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 2048, "mscale": 1.0,
     "mscale_all_dim": 0.8, "beta_fast": 32.0, "beta_slow": 1.0}])
def test_scaled_frequencies_match_the_library(scaling):
    """Against transformers' initialisers (fp32: 2^-20 relative)."""
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    kind = (scaling or {}).get("rope_type", "default")
    params = dict(scaling or {"rope_type": "default"}, rope_theta=10000.0)
    cfg = LlamaConfig(hidden_size=512, num_attention_heads=4, num_key_value_heads=4, max_position_embeddings=2048,
                      rope_parameters=params)
    length = 8192
    f, att = rotary.inv_frequencies(128, 10000.0, scaling, trained=2048, length=length)
    if kind == "default":
        want, watt = 1.0 / (10000.0 ** (torch.arange(0, 128, 2).double() / 128)), 1.0
    else:
        want, watt = ROPE_INIT_FUNCTIONS[kind](cfg, torch.device("cpu"), seq_len=length)
    assert torch.allclose(f, want.double(), rtol=2.0 ** -18, atol=0)
    assert abs(att - watt) < 1e-6


def test_ntk_keeps_the_highest_and_divides_the_lowest_frequency():
    f, _ = rotary.inv_frequencies(64, 10000.0)
    g, _ = rotary.inv_frequencies(64, 10000.0, {"rope_type": "ntk", "factor": 4.0})
    assert g[0] == f[0] and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12 and bool((g <= f).all())


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    _, q, k = inputs(2, 3, 4, 2, 32, torch.float32, device, "packed")
    cos, sin = rotary.rotary_tables(32, 16, device=device)
    with pytest.raises(ValueError):
        rotary.rotary_qk(q[0], k[0], cos, sin)
    with pytest.raises(ValueError):
        rotary.rotary_qk(q, k[:1], cos, sin)
    with pytest.raises(ValueError):
        rotary.rotary_qk(q, k.to(torch.bfloat16), cos, sin)
    with pytest.raises(ValueError):
        rotary.rotary_qk(q, k, cos.to(torch.bfloat16), sin.to(torch.bfloat16))
    with pytest.raises(ValueError):
        rotary.rotary_qk(q[..., :16], k[..., :16], cos, sin)
    with pytest.raises(ValueError):
        rotary.rotary_qk(q, k, cos[:2], sin[:2])
    with pytest.raises(ValueError):
        rotary.rotary_qk(q, k, cos, sin, torch.zeros(2, 4, dtype=torch.long, device=device))
    with pytest.raises(TypeError):
        rotary.rotary_qk(q, k, cos, sin, torch.zeros(2, 3, device=device))
    with pytest.raises(ValueError):
        rotary.rotary_qk(q.clone().requires_grad_(), k, cos, sin, inplace=True)
    for bad in ({"rope_type": "unheard-of"}, {"rope_type": "linear", "factor": 0.5}, {"rope_type": "yarn", "factor": 2.0}):
        with pytest.raises(ValueError):
            rotary.inv_frequencies(32, 10000.0, bad)
    with pytest.raises(ValueError):
        rotary.inv_frequencies(31, 10000.0)


def test_position_outside_the_tables_raises_on_the_cpu():
    _, q, k = inputs(1, 2, 1, 1, 8, torch.float32, "cpu", "packed")
    cos, sin = rotary.rotary_tables(8, 4)
    for p in ([[0, 4]], [[-1, 0]]):
        with pytest.raises(IndexError):
            rotary.rotary_qk(q, k, cos, sin, torch.tensor(p))


@pytest.mark.gpu
def test_position_outside_the_tables_is_reported():
    """The kernel checks every position against the tables before it reads them."""
    _, q, k = inputs(1, 3, 2, 1, 8, torch.float32, "cuda", "packed")
    cos, sin = rotary.rotary_tables(8, 4, device="cuda")
    oq, _ = rotary.rotary_qk(q, k, cos, sin, torch.tensor([[0, 4, 2]], device="cuda"))
    assert bool(oq[0, 1].isnan().all()) and bool(oq[0, 0].isfinite().all()) and bool(oq[0, 2].isfinite().all())
    with pytest.raises(KernelTimeoutError):
        check_kernel_errors(q.device)
    check_kernel_errors(q.device)
