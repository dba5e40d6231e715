"""The loss without logits, 8-bit activations and general rotary positions inside the model and
the training command.

Tolerances: fp32 paths that compute the same in another order agree to 1e-5 of the largest value
(sums of up to a few hundred terms, 2^-24 each).  Eight bits keep a value to within half of
1/127 of its group's largest magnitude: about 0.6 % rms of normal values, so gradients stay within a
few per cent of the exact ones (5 % asked)."""
import os
import subprocess
import sys

import pytest
import torch

from common_models import full_state, tiny_config
from femtotron_b200.models import LlamaForTraining
from femtotron_b200.models.layers import LlamaDecoderLayer, LlamaRotaryEmbedding
from femtotron_b200.ops import act8, rotary
from femtotron_b200.ops import functional as FN
from femtotron_b200.training import apply_activation_checkpointing

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def config(**attrs):
    cfg = tiny_config()
    for k, v in attrs.items():
        setattr(cfg, k, v)
    return cfg


def run(cfg, sd, ids, bits=None, dtype=torch.float32, device="cpu"):
    model = LlamaForTraining(cfg, dtype=dtype, device=device)
    model.load_state_dict({k: v.to(dtype) for k, v in sd.items()})
    if bits:
        n = apply_activation_checkpointing(model, lambda m: isinstance(m, LlamaDecoderLayer), bits=bits)
        assert n == cfg.num_hidden_layers
    loss = model(ids, labels=ids)["loss"]
    loss.backward()
    return float(loss.detach()), {k.replace("._checkpoint_wrapped_module", ""): p.grad.float() for k, p in model.named_parameters()}


def rel(a, b):
    return float((a - b).norm() / b.norm())


@pytest.fixture(scope="module")
def base():
    cfg = config()
    sd = full_state(cfg)
    ids = torch.randint(0, cfg.vocab_size, (2, 48), generator=torch.Generator().manual_seed(1))
    return sd, ids, run(cfg, sd, ids)


def test_loss_without_logits_and_general_rotation_change_nothing(base):
    sd, ids, (loss, grads) = base
    for attrs in (dict(loss_keep_logits=False), dict(rotary_spec={}), dict(rotary_spec={"scaling": None, "partial": 1.0})):
        other, og = run(config(**attrs), sd, ids)
        assert abs(other - loss) < 1e-5
        for k in grads:
            assert float((og[k] - grads[k]).abs().max()) <= 1e-5 * float(grads[k].abs().max()) + 1e-9, (attrs, k)


def test_interleaved_layout_is_the_half_layout_with_permuted_rows(base):
    sd, ids, (loss, _) = base
    cfg = config(rotary_spec={"interleaved": True})
    d = cfg.hidden_size // cfg.num_attention_heads
    perm = torch.stack([torch.arange(d // 2), torch.arange(d // 2) + d // 2], 1).reshape(-1)  # 0, r, 1, r + 1, ...
    other = dict(sd)
    for k, v in sd.items():
        if "q_proj" in k or "k_proj" in k:
            other[k] = v.view(-1, d, v.shape[1])[:, perm].reshape(v.shape)
    assert abs(run(cfg, other, ids)[0] - loss) < 1e-5


def test_scaling_and_partial_rotation_reach_the_tables():
    e = LlamaRotaryEmbedding(config(rotary_spec={"scaling": {"rope_type": "linear", "factor": 4.0}, "partial": 0.5}))
    cos, sin = e(torch.zeros(1, 40, 64), seq_len=40)
    want = rotary.rotary_tables(8, 128, e.theta, {"rope_type": "linear", "factor": 4.0})
    assert cos.dtype == torch.float32 and torch.equal(cos, want[0]) and torch.equal(sin, want[1])
    for bad in ({"partial": 0.0}, {"partial": 1.5}, {"scale": 2}):
        with pytest.raises(ValueError):
            LlamaRotaryEmbedding(config(rotary_spec=bad))


def test_checkpoint_in_8_bits_recomputes_from_the_kept_values():
    torch.manual_seed(0)
    inner = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.SiLU(), torch.nn.Linear(96, 64))
    model = torch.nn.Sequential(torch.nn.Linear(64, 64), inner)
    wrapped = torch.nn.Sequential(model[0], inner)
    x = torch.randn(5, 64)
    h = model[0](x)
    exact = inner(h)
    # the gradient that the kept values give
    h8 = act8.quantize(h).dequantize().requires_grad_()
    g = torch.randn(5, 64)
    inner.zero_grad()
    inner(h8).backward(g)
    want = [p.grad.clone() for p in inner.parameters()]
    inner.zero_grad()
    apply_activation_checkpointing(wrapped, lambda m: m is inner, bits=8)
    out = wrapped(x)
    assert torch.equal(out, exact)
    model[0].zero_grad()
    out.backward(g)
    assert all(torch.equal(p.grad, w) for p, w in zip(inner.parameters(), want))
    ref = h8.grad.t() @ x
    assert torch.allclose(model[0].weight.grad, ref, rtol=1e-5, atol=1e-6)
    with pytest.raises(ValueError):
        apply_activation_checkpointing(torch.nn.Sequential(torch.nn.Linear(2, 2)), lambda m: True, bits=4)


def test_norm_mlp_block_matches_its_formula_on_the_kept_values():
    g = torch.Generator().manual_seed(0)
    T, H, F = 7, 64, 96
    x, dout = torch.randn(T, H, generator=g), torch.randn(T, H, generator=g)
    wn = 1 + 0.1 * torch.randn(H, generator=g)
    wg, wu = torch.randn(F, H, generator=g) * 0.1, torch.randn(F, H, generator=g) * 0.1
    wd = torch.randn(H, F, generator=g) * 0.1
    ps = [torch.nn.Parameter(w.clone()) for w in (wn, wg, wu, wd)]
    xx = x.clone().requires_grad_()
    out = FN.NormMLP8Fn.apply(xx, ps[0], 1e-5, 32, *ps[1:])
    out.backward(dout)
    # forward: exact
    n, r, x8 = act8.rms_norm(x, wn, 1e-5, 32)
    gu = torch.cat([n @ wg.t(), n @ wu.t()], 1)
    a, gu8 = act8.swiglu(gu, 32)
    assert torch.allclose(out, x + a @ wd.t(), rtol=1e-5, atol=1e-5)
    # backward: from the kept bytes
    dgu, a8 = act8.swiglu_bwd(dout @ wd, gu8)
    dx, dwn, n8 = act8.rms_norm_bwd(dgu @ torch.cat([wg, wu]), x8, wn, r)
    for got, want in ((xx.grad, dx + dout), (ps[0].grad, dwn), (ps[1].grad, dgu[:, :F].t() @ n8),
                      (ps[2].grad, dgu[:, F:].t() @ n8), (ps[3].grad, dout.t() @ a8)):
        assert rel(got, want) < 1e-5
    # and near the exact gradient
    ex = [p.detach().clone().requires_grad_() for p in (x, wn, wg, wu, wd)]
    nn_ = ex[0] * torch.rsqrt(ex[0].pow(2).mean(1, keepdim=True) + 1e-5) * ex[1]
    y = ex[0] + (torch.nn.functional.silu(nn_ @ ex[2].t()) * (nn_ @ ex[3].t())) @ ex[4].t()
    y.backward(dout)
    for got, want in zip([xx, *ps], ex):
        assert rel(got.grad, want.grad) < 0.05


@pytest.mark.parametrize("bits,mlp", [(8, False), (None, True), (8, True)])
def test_gradients_in_8_bits_stay_near_the_exact_ones(base, bits, mlp):
    sd, ids, (loss, grads) = base
    other, og = run(config(mlp_act8=mlp), sd, ids, bits=bits)
    assert abs(other - loss) < 1e-5  # the forward is exact
    for k in grads:
        assert rel(og[k], grads[k]) < 0.05, k


def test_8_bit_block_is_left_out_without_a_backward(base):
    sd, ids, (loss, _) = base
    model = LlamaForTraining(config(mlp_act8=True), dtype=torch.float32)
    model.load_state_dict(sd)
    with torch.no_grad():
        assert abs(float(model(ids, labels=ids)["loss"]) - loss) < 1e-5


def train(tmp_path, name, *extra):
    """Losses of four steps of the training command on two gloo ranks, and its output."""
    import json
    metrics = tmp_path / f"{name}.jsonl"
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
           "--master-port", "29653", "-m", "femtotron_b200.scripts.train", "--config", "configs/tiny_llama_long.yaml",
           "--seq_len", "64", "--micro_batch_size", "4", "--hidden_size", "64", "--intermediate_size", "160",
           "--vocab_size", "256", "--num_hidden_layers", "2", "--num_samples", "200", "--train_steps", "4",
           "--warmup_steps", "1", "--metrics_path", str(metrics), "--checkpoint_dir", str(tmp_path / name),
           "--checkpoint_interval", "1000", *extra]
    r = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""), capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return [json.loads(line)["loss"] for line in metrics.read_text().splitlines()], r.stdout


@pytest.mark.parametrize("layout", [["--zero_stage", "3"], ["--tp", "2"], ["--tp", "2", "--sequence_parallel", "true"]],
                         ids=["zero3", "tp", "tp-sp"])
def test_training_command_runs_all_of_them(tmp_path, layout):
    """ZeRO-3 gathers and shards each layer around its 8-bit checkpoint; with tensor parallelism the
    vocabulary shards join in the loss and the 8-bit MLP block stands aside.  The losses follow those
    of the plain run."""
    on, said = train(tmp_path, "all", *layout)
    off, plain = train(tmp_path, "plain", *layout, "--ac_bits", "16", "--mlp_act8", "false", "--loss_keep_logits", "true")
    assert "in 8 bits" in said and "in 8 bits" not in plain
    assert len(on) == len(off) == 4
    # bf16 model: a rounding of the loss's inputs apart at most (2^-8 of a logit below 0.5)
    assert all(abs(a - b) < 2e-3 for a, b in zip(on, off))


def test_8_bit_mlp_block_under_zero3_without_checkpointing(tmp_path):
    layout = ["--zero_stage", "3", "--ac_enabled", "false"]
    on, _ = train(tmp_path, "on", *layout)
    off, _ = train(tmp_path, "off", *layout, "--mlp_act8", "false", "--loss_keep_logits", "true")
    assert len(on) == 4 and all(abs(a - b) < 2e-3 for a, b in zip(on, off))


@pytest.mark.gpu
def test_model_on_the_gpu_with_everything_on():
    from femtotron_b200.ops import attention, check_kernel_errors
    cfg = tiny_config(hidden_size=256, intermediate_size=688, vocab_size=2048, max_position_embeddings=512)
    sd = full_state(cfg)
    ids = torch.randint(0, cfg.vocab_size, (2, 256), generator=torch.Generator().manual_seed(1)).cuda()
    sd = {k: v.cuda() for k, v in sd.items()}
    loss, grads = run(cfg, sd, ids, dtype=torch.bfloat16, device="cuda")
    before = attention.SDPA_FALLBACKS[0]
    for k, v in dict(loss_keep_logits=False, mlp_act8=True, rotary_spec={"scaling": {"rope_type": "linear", "factor": 1.0}}).items():
        setattr(cfg, k, v)
    other, og = run(cfg, sd, ids, bits=8, dtype=torch.bfloat16, device="cuda")
    check_kernel_errors()
    assert attention.SDPA_FALLBACKS[0] == before
    assert abs(other - loss) < 2e-2
    for k in grads:
        assert rel(og[k], grads[k]) < 0.08, (k, rel(og[k], grads[k]))
