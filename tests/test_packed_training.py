"""Documents, windows, capped scores, a bias of distance and scaled embeddings in the model and the training
command, and the three operators of a packed step together.

Tolerances: fp32 paths that compute the same in another order agree to 1e-5 of the largest value (sums of up to
a few hundred terms, 2^-24 each); positions shifted by a document's place turn queries and keys by other angles whose
difference is the same, which adds the rounding of the angles (fp32, up to 100 turns: 1e-5)."""
import os

import pytest
import torch

from common_models import full_state, tiny_config
from femtotron_b200.models import LlamaForTraining
from femtotron_b200.models.layers import Attention, LlamaDecoderLayer
from femtotron_b200.ops import functional as FN
from femtotron_b200.ops import grad_norm as GN
from femtotron_b200.ops import masked_attention as MA
from femtotron_b200.scripts import train
from femtotron_b200.training import apply_activation_checkpointing

gpu = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def config(**attrs):
    cfg = tiny_config()
    for k, v in attrs.items():
        setattr(cfg, k, v)
    return cfg


def run(cfg, sd, ids, labels=None, bits=None, **kw):
    model = LlamaForTraining(cfg, dtype=torch.float32)
    model.load_state_dict(sd)
    if bits:
        apply_activation_checkpointing(model, lambda m: isinstance(m, LlamaDecoderLayer), bits=bits)
    out = model(ids, labels=ids if labels is None else labels, materialize_logits=True, **kw)
    out["loss"].backward()
    return float(out["loss"].detach()), out["logits"].detach(), \
        {k.replace("._checkpoint_wrapped_module", ""): p.grad for k, p in model.named_parameters()}


def same(a, b, tol=1e-5):
    assert abs(a[0] - b[0]) < tol * 10
    assert float((a[1] - b[1]).abs().max()) <= tol * float(b[1].abs().max())
    for k in b[2]:
        assert float((a[2][k] - b[2][k]).abs().max()) <= 2 * tol * float(b[2][k].abs().max()) + 1e-9, k


@pytest.fixture(scope="module")
def base():
    cfg = config()
    sd = full_state(cfg)
    ids = torch.randint(1, cfg.vocab_size, (2, 48), generator=torch.Generator().manual_seed(1))
    return sd, ids, run(cfg, sd, ids)


@pytest.mark.parametrize("spec", [dict(), dict(window=48), dict(softcap=1e7), dict(separator=0), dict(window=1000, separator=0)])
def test_nothing_changes_where_nothing_is_masked(base, spec):
    sd, ids, want = base
    # a cap of 1e7 changes scores s by s^3 / 3e14
    same(run(config(attn_spec=spec), sd, ids), want)


def test_a_packed_row_equals_its_documents(base):
    sd, ids, _ = base
    row = ids[:1].clone()
    row[0, 19] = row[0, 40] = 0
    cfg = config(attn_spec={"separator": 0})
    _, logits, _ = run(cfg, sd, row)
    for a, b in ((0, 20), (20, 41), (41, 48)):
        _, alone, _ = run(config(), sd, row[:, a:b])
        assert float((logits[:, a:b] - alone).abs().max()) < 1e-4 * float(alone.abs().max())
    same(run(config(), sd, row, docs=MA.document_ids(row, 0)), run(cfg, sd, row))


@pytest.mark.parametrize("bits", [None, 16])
def test_padding_and_prefix(base, bits):
    sd, ids, _ = base
    docs = torch.zeros(2, 48, dtype=torch.int32)
    docs[0, 30:] = -1
    labels = ids.clone()
    labels[0, 30:] = -100
    prefix = torch.zeros(2, 48, dtype=torch.bool)
    prefix[:, :9] = True
    _, logits, _ = run(config(), sd, ids, labels, bits=bits, docs=docs, prefix=prefix)
    _, alone, _ = run(config(), sd, ids[:1, :30], prefix=prefix[:1, :30])
    assert float((logits[:1, :30] - alone).abs().max()) < 1e-5 * float(alone.abs().max())
    # the first token of the prompt sees its end, not what comes after it
    other = ids.clone()
    other[:, 8] = ids[:, 8] % 255 + 1
    later = ids.clone()
    later[:, 9] = ids[:, 9] % 255 + 1
    first = [run(config(), sd, x, prefix=prefix)[1][:, 0] for x in (ids, other, later)]
    assert (first[0] - first[1]).abs().max() > 1e-4 and torch.equal(first[0], first[2])


def test_window_cap_and_bias_reach_every_layer(base):
    sd, ids, (loss, logits, _) = base
    for spec in (dict(window=5), dict(softcap=0.05), dict(alibi=True)):
        _, other, _ = run(config(attn_spec=spec), sd, ids)
        assert (other - logits).abs().max() > 1e-4
    # two layers of windows of 5 reach 8 tokens back, no further
    a, b = ids.clone(), ids.clone()
    b[:, 10] = a[:, 10] % 255 + 1
    x, y = (run(config(attn_spec=dict(window=5)), sd, z)[1] for z in (a, b))
    assert torch.equal(x[:, 19:], y[:, 19:]) and (x[:, 18] - y[:, 18]).abs().max() > 0


def test_embed_scale(base):
    sd, ids, _ = base
    grown = {k: v * 4 if "embed_tokens" in k else v for k, v in sd.items()}
    a, b = run(config(embed_scale=4.0), sd, ids), run(config(), grown, ids)
    assert abs(a[0] - b[0]) < 1e-5 and torch.allclose(a[1], b[1], rtol=1e-5, atol=1e-5)
    k = next(k for k in sd if "embed_tokens" in k)
    assert torch.allclose(a[2][k], 4 * b[2][k], rtol=1e-4, atol=1e-7)


def test_refusals():
    with pytest.raises(ValueError, match="unknown keys"):
        LlamaForTraining(config(attn_spec={"windows": 3}))
    with pytest.raises(ValueError, match="window"):
        LlamaForTraining(config(attn_spec={"window": 0}))
    with pytest.raises(ValueError, match="softcap"):
        LlamaForTraining(config(attn_spec={"softcap": -1.0}))
    args = train.parse_args(["--config", os.path.join(ROOT, "configs", "tiny_llama_packed.yaml"), "--pp", "2"])
    with pytest.raises(ValueError, match="doc_separator"):
        train.model_config_from(train.load_config(args))


def test_heads_of_a_rank_take_their_own_slopes():
    B, S, nq, nkv, d = 2, 20, 4, 2, 8
    qkv = torch.randn(B * S, (nq + 2 * nkv) * d, generator=torch.Generator().manual_seed(0))
    plan = Attention(MA.attention_mask(1, S), 0.0, MA.alibi_slopes(nq))
    whole = plan(qkv, B, S, nq, nkv, d, 0).view(B * S, nq, d)
    x = qkv.view(B * S, nq + 2 * nkv, d)
    for r in range(2):
        part = torch.cat([x[:, 2 * r:2 * r + 2], x[:, nq + r:nq + r + 1], x[:, nq + nkv + r:nq + nkv + r + 1]], 1)
        assert torch.allclose(plan(part.reshape(B * S, -1), B, S, 2, 1, d, r).view(B * S, 2, d), whole[:, 2 * r:2 * r + 2],
                              rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("tp", ["1", "2"])
def test_command(tmp_path, tp):
    from test_cli import _run
    cfg = os.path.join(ROOT, "configs", "tiny_llama_packed.yaml")
    out = _run(["--config", cfg, "--num_hidden_layers", "2", "--seq_len", "50", "--micro_batch_size", "2", "--attn_alibi",
                "--checkpoint_dir", str(tmp_path / "ck"), "--tp", tp, "--train_steps", "3"], tmp_path, nproc=int(tp))
    assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-3000:]
    assert "step      3/3" in out.stdout


# ------------------------------------------------------------------------------ the operators together
def step(ids, docs, table, wqkv, nq, nkv, d, target):
    """Embedding, one projection, masked attention, a squared loss, all gradients, clipped; returns the lot."""
    p = torch.nn.Parameter(table.clone())
    w = wqkv.detach().clone().requires_grad_()
    x = FN.embedding(ids, p, scale=3.0)
    B, S, H = x.shape
    qkv = (x.reshape(-1, H) @ w).view(B, S, nq + 2 * nkv, d)
    mask = MA.attention_mask(B, S, docs=docs, window=40)
    o = MA.masked_attention_packed(qkv, nq, nkv, mask, softcap=5.0, slopes=MA.alibi_slopes(nq, ids.device))
    ((o.float() - target) ** 2).mean().backward()
    grads = [p.grad, w.grad]
    norm = GN.clip_grads(grads, 1e-3)
    return [o.detach(), norm, *grads]


@gpu
def test_gpu_operators_together():
    g = torch.Generator().manual_seed(3)
    B, S, H, V, nq, nkv, d = 2, 333, 64, 50, 4, 2, 32
    ids = torch.randint(0, V, (B, S), generator=g)
    docs = (torch.rand(B, S, generator=g) < 0.02).cumsum(1).int()
    docs[1, 300:] = -1
    table = torch.randn(V, H, generator=g) * 0.3
    w = torch.randn(H, (nq + 2 * nkv) * d, generator=g) * 0.1
    target = torch.randn(B, S, nq, d, generator=g)
    want = step(ids, docs, table, w, nq, nkv, d, target)
    cast = [x.cuda() for x in (ids, docs, table.bfloat16(), w.bfloat16())]
    got = step(*cast, nq, nkv, d, target.cuda())
    again = step(*cast, nq, nkv, d, target.cuda())
    # a chain of about six bf16 roundings (2^-9 rms each, 2^-8 at most) on either side of the exact chain
    for x, y, z in zip(got, want, again):
        assert float((x.float().cpu() - y).norm() / y.norm()) < 6 * 2 ** -8
        assert torch.equal(x, z)


@gpu
def test_gpu_model_on_packed_rows():
    cfg = config(num_attention_heads=4, num_key_value_heads=2, hidden_size=256, intermediate_size=512, embed_scale=4.0,
                 attn_spec={"separator": 0, "window": 50, "softcap": 20.0})
    sd = full_state(cfg)
    ids = torch.randint(0, 40, (2, 150), generator=torch.Generator().manual_seed(1))
    loss, logits, _ = run(cfg, sd, ids)
    model = LlamaForTraining(cfg, dtype=torch.bfloat16, device="cuda")
    model.load_state_dict({k: v.bfloat16() for k, v in sd.items()})
    for _ in range(2):
        out = model(ids.cuda(), labels=ids.cuda(), materialize_logits=True)
        out["loss"].backward()
        # some thirty roundings of 2^-9 of two layers and the head
        assert abs(float(out["loss"].detach()) - loss) < 0.02 * loss
        assert float((out["logits"].detach().float().cpu() - logits).norm() / logits.norm()) < 30 ** 0.5 * 2 ** -8
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
