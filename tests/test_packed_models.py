"""Models on packed documents: the factor of the embedding wherever the embedding comes from, slopes that are made
once, exported models."""
import json

import pytest
import torch
from safetensors.torch import load_file

from femtotron_b200.models import LlamaForTraining
from femtotron_b200.models.export import export_hf
from femtotron_b200.models.layer_factory import DefaultLayerFactory
from femtotron_b200.models.layers import Attention
from femtotron_b200.models.parallel_plan import ParallelRule
from femtotron_b200.ops import masked_attention as MA
from femtotron_b200.parallel.tensor_parallel import VocabParallelEmbedding
from femtotron_b200.training import apply_activation_checkpointing
from common_models import full_state
from test_packed_training import base, config, run, same  # noqa: F401

gpu = pytest.mark.gpu


def graded(model, ids):
    out = model(ids, labels=ids, materialize_logits=True)
    out["loss"].backward()
    return float(out["loss"].detach()), out["logits"].detach(), \
        {k.replace("._checkpoint_wrapped_module", ""): p.grad for k, p in model.named_parameters()}


class OneRank:
    """A parallel context without groups."""
    tp_size = 1

    def get_group(self, name):
        return None

    def get_size(self, name):
        return 1

    def get_rank(self, name):
        return 0


class OwnEmbedding(torch.nn.Module):
    def __init__(self, plain):
        super().__init__()
        self.weight = plain.weight

    def forward(self, ids):
        return self.weight[ids]


@pytest.mark.parametrize("kind", ["checkpointed", "vocabulary", "vocabulary, checkpointed", "vocabulary, temporary", "factory", "own"])
def test_embed_scale_reaches_every_embedding(base, kind):
    sd, ids, _ = base
    want = run(config(embed_scale=4.0), sd, ids)
    cfg = config(embed_scale=4.0)
    model = LlamaForTraining(cfg, dtype=torch.float32)
    plain = model.model.embed_tokens
    if kind.startswith("vocabulary"):
        if "temporary" in kind:
            model.model.embed_tokens = VocabParallelEmbedding.from_embedding_temp(plain, OneRank())
            assert model.model.embed_tokens.scale == 4.0
        else:
            model.model.embed_tokens = VocabParallelEmbedding.from_embedding(plain, OneRank(), ParallelRule("vocab_embed", {}))
    elif kind == "factory":  # what it makes without tensor parallelism, and with it
        model.model.embed_tokens = DefaultLayerFactory().make_embedding(cfg, None, dtype=torch.float32, device=None)
        model.load_state_dict(sd)
        same(graded(model, ids), want)
        model.zero_grad(set_to_none=True)
        model.model.embed_tokens = VocabParallelEmbedding(cfg.vocab_size, cfg.hidden_size, OneRank(), dtype=torch.float32)
    elif kind == "own":
        model.model.embed_tokens = OwnEmbedding(plain)
    model.load_state_dict(sd)
    if "checkpointed" in kind:
        assert apply_activation_checkpointing(model, lambda m: isinstance(m, (torch.nn.Embedding, VocabParallelEmbedding))) == 1
    same(graded(model, ids), want)


def test_another_factor_of_the_embedding_is_refused(base):
    sd, ids, _ = base
    model = LlamaForTraining(config(embed_scale=4.0), dtype=torch.float32)
    model.model.embed_tokens = VocabParallelEmbedding.from_embedding(model.model.embed_tokens, OneRank(), ParallelRule("vocab_embed", {}))
    model.load_state_dict(sd)
    model.model.embed_tokens.scale = 2.0
    with pytest.raises(ValueError, match="embed_scale"):
        model(ids)


def test_slopes_are_made_once(base, monkeypatch):
    sd, ids, _ = base
    made = []
    slopes = MA.alibi_slopes
    monkeypatch.setattr(MA, "alibi_slopes", lambda *a: made.append(a) or slopes(*a))
    model = LlamaForTraining(config(attn_spec={"alibi": True}), dtype=torch.float32)
    model.load_state_dict(sd)
    with torch.no_grad():
        first = model(ids)["logits"].clone()
    for _ in range(2):  # what a pass without gradients made serves those with gradients
        loss, logits, _ = graded(model, ids)
        assert torch.equal(logits, first)
    assert len(made) == 1 and set(model.state_dict()) == set(sd)


@pytest.mark.parametrize("bits", [8, 16])
def test_layer_checkpoints_keep_the_mask(base, monkeypatch, bits):
    sd, ids, _ = base
    docs = torch.zeros(2, 48, dtype=torch.int32)
    docs[0, 30:] = -1
    docs[1, 20:] = 1
    seen = []
    call = Attention.__call__
    monkeypatch.setattr(Attention, "__call__", lambda self, *a: seen.append(self) or call(self, *a))
    cfg = config(attn_spec={"window": 9, "softcap": 5.0, "alibi": True}, embed_scale=4.0)
    want = run(cfg, sd, ids, docs=docs)
    del seen[:]
    got = run(cfg, sd, ids, bits=bits, docs=docs)
    assert len(seen) == 2 * cfg.num_hidden_layers and len(set(map(id, seen))) == 1  # forward and again for the backward pass
    assert got[0] == want[0] and torch.equal(got[1], want[1])
    for k, g in want[2].items():
        # 8 bits round a value by 2^-8 of its group's largest at most; two layers of six products pass that on
        assert float((got[2][k] - g).norm()) <= (12 * 2 ** -8 if bits == 8 else 1e-6) * float(g.norm()), k


def test_shapes_without_data():
    from femtotron_b200.ops import embedding as E
    with torch.device("meta"):
        emb = VocabParallelEmbedding(10, 4, OneRank(), dtype=torch.float32)
        emb.scale = 3.0
        assert emb(torch.zeros(2, 3, dtype=torch.long)).shape == (2, 3, 4)
    # ids of other shards, a shard without words, and a table whose first row is no number
    w = torch.tensor([[float("nan")], [2.0]])
    assert E.lookup(torch.tensor([5, -1, 8, 6]), w, 5, 2.0)[1:].flatten().tolist() == [0.0, 0.0, 4.0]
    assert E.lookup(torch.tensor([[5], [6]]), torch.empty(0, 7), 0).tolist() == [[[0.0] * 7]] * 2


def test_a_backbone_that_knows_no_documents(base):
    sd, ids, want = base

    class Backbone(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, input_ids):
            return self.inner(input_ids)
    model = LlamaForTraining(config(), dtype=torch.float32)
    model.load_state_dict(sd)
    model.model = Backbone(model.model)
    with torch.no_grad():
        assert torch.equal(model(ids)["logits"], want[1])
        with pytest.raises(TypeError, match="docs"):
            model(ids, docs=torch.zeros_like(ids))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("kind", ["strided", "fp64"])
def test_gradient_buffers_of_any_strides_and_type(device, kind):
    from femtotron_b200.ops.functional import embedding
    g = torch.Generator().manual_seed(0)
    w, ids = torch.randn(9, 16, generator=g).bfloat16().to(device), torch.randint(0, 9, (40,), generator=g).to(device)
    do = torch.randn(40, 16, generator=g).bfloat16().to(device)
    want = torch.zeros(9, 16, dtype=torch.float64, device=device).index_add_(0, ids, do.double())
    p = torch.nn.Parameter(w)
    if kind == "strided":
        p.grad = torch.zeros(16, 9, dtype=torch.bfloat16, device=device).t()
    else:
        p.main_grad = torch.zeros(9, 16, dtype=torch.float64, device=device)
    got = p.grad if kind == "strided" else p.main_grad
    for k in (1, 2):  # one rounding to bf16 of either sum; 2^-18: fp32 sums
        embedding(ids, p).backward(do)
        assert ((got - k * want).abs() <= (2 ** -8 * 2 * k * want.abs() if kind == "strided" else 0) + 2 ** -18 * 40 * 4).all()


def checkpoint(path, model):
    path.mkdir()
    (path / "meta.json").write_text(json.dumps({"tp_size": 1, "dp_size": 1}))
    torch.save({"optimizer": {}, "model": model.state_dict()}, path / "shard_tp0_dp0.pt")
    return str(path)


@pytest.mark.parametrize("attrs", [dict(embed_scale=3.0), dict(embed_scale=3.0, attn_spec={"separator": 0}), dict(embed_scale=1.0), {}])
def test_exported_models_compute_the_same(base, tmp_path, attrs):
    from transformers import AutoConfig, LlamaForCausalLM
    sd, ids, _ = base
    cfg = config(**attrs)
    model = LlamaForTraining(cfg, dtype=torch.float32)
    model.load_state_dict(sd)
    out = export_hf(checkpoint(tmp_path / "ck", model), cfg, str(tmp_path / "hf"), dtype=torch.float32)
    assert {k: getattr(cfg, k) for k in attrs} == attrs
    with torch.no_grad():
        want = model(ids)["logits"]  # (no separator among the ids)
        theirs = LlamaForCausalLM.from_pretrained(out, dtype=torch.float32)(input_ids=ids).logits
        read = AutoConfig.from_pretrained(out)
        again = LlamaForTraining(read, dtype=torch.float32)
        again.load_state_dict(load_file(out + "/model.safetensors"))
        ours = again(ids)["logits"]
    # fp32 in another order, as same()
    assert float((theirs - want).abs().max()) < 1e-5 * float(want.abs().max())
    assert float((ours - want).abs().max()) < 1e-5 * float(want.abs().max())
    assert not hasattr(read, "embed_scale")


@pytest.mark.parametrize("attrs,what", [(dict(attn_spec={"softcap": 5.0}), "softcap=5.0"), (dict(attn_spec={"window": 7}), "window=7"),
                                        (dict(attn_spec={"alibi": True}), "alibi"),
                                        (dict(embed_scale=3.0, tie_word_embeddings=True), "tied")])
def test_what_llama_cannot_express_is_not_exported(base, tmp_path, attrs, what):
    from transformers import AutoConfig
    _, ids, _ = base
    cfg = config(**attrs)
    model = LlamaForTraining(cfg, dtype=torch.float32)
    ck = checkpoint(tmp_path / "ck", model)
    with pytest.raises(ValueError, match=what):
        export_hf(ck, cfg, str(tmp_path / "hf"))
    assert not (tmp_path / "hf").exists()
    out = export_hf(ck, cfg, str(tmp_path / "own"), dtype=torch.float32, keep_attributes=True)
    again = LlamaForTraining(AutoConfig.from_pretrained(out), dtype=torch.float32)
    again.load_state_dict(load_file(out + "/model.safetensors"), strict=not cfg.tie_word_embeddings)
    with torch.no_grad():
        assert torch.equal(again(ids)["logits"], model(ids)["logits"])


@gpu
def test_gpu_slopes_neither_wait_nor_stop_a_graph():
    cfg = config(num_attention_heads=12, num_key_value_heads=6, hidden_size=192, intermediate_size=256,
                 attn_spec={"alibi": True, "window": 50, "softcap": 20.0})
    sd = {k: v.bfloat16() for k, v in full_state(cfg).items()}
    ids = torch.randint(1, 200, (2, 150), generator=torch.Generator().manual_seed(1)).cuda()
    model = LlamaForTraining(cfg, dtype=torch.bfloat16, device="cuda")
    model.load_state_dict(sd)
    with torch.no_grad():
        want = model.model(ids)
        torch.cuda.set_sync_debug_mode("error")
        try:
            got = model.model(ids)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        assert torch.equal(got, want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        for kept in (True, False):  # with slopes at hand, and made in the graph
            if not kept:
                model.model._slopes.clear()
            with torch.cuda.stream(side):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    out = model.model(ids)
            torch.cuda.current_stream().wait_stream(side)
            assert bool(model.model._slopes) == kept
            graph.replay()
            assert torch.equal(out, want)
        assert torch.equal(model.model(ids), want)


@gpu
@pytest.mark.parametrize("spec", [{"alibi": True}, {"alibi": True, "separator": 0, "softcap": 20.0}])
def test_gpu_model_with_a_bias_of_distance(spec):
    cfg = config(num_attention_heads=6, num_key_value_heads=2, hidden_size=384, intermediate_size=512, embed_scale=4.0,
                 attn_spec=spec)
    sd = {k: v.bfloat16().float() for k, v in full_state(cfg).items()}
    ids = torch.randint(0, 40, (2, 150), generator=torch.Generator().manual_seed(1))
    loss, logits, grads = run(cfg, sd, ids)
    model = LlamaForTraining(cfg, dtype=torch.bfloat16, device="cuda")
    model.load_state_dict(sd)
    got = graded(model, ids.cuda())
    # some thirty roundings of 2^-9 of two layers and the head forward, twice as many again backward
    assert abs(got[0] - loss) < 0.02 * loss
    assert float((got[1].float().cpu() - logits).norm() / logits.norm()) < 30 ** 0.5 * 2 ** -8
    for k, g in grads.items():
        assert float((got[2][k].float().cpu() - g).norm() / g.norm()) < 90 ** 0.5 * 2 ** -8, k
