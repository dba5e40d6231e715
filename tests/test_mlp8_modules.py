"""The 8-bit MLP block computes norm and MLP in one function.  It stands aside where something hangs on
either module's call: hooks (a sharding unit gathers its weights in them) or an activation checkpoint."""
import pytest
import torch

from common_models import full_state, tiny_config
from femtotron_b200.models import LlamaForTraining
from femtotron_b200.models.layers import LlamaMLP
from femtotron_b200.training import apply_activation_checkpointing


def model(mlp_act8):
    cfg = tiny_config()
    cfg.mlp_act8 = mlp_act8
    m = LlamaForTraining(cfg, dtype=torch.float32)
    m.load_state_dict(full_state(cfg))
    ids = torch.randint(0, cfg.vocab_size, (2, 24), generator=torch.Generator().manual_seed(1))
    return m, ids


def gradients(m, ids):
    m(ids, labels=ids)["loss"].backward()
    return [p.grad.clone() for p in m.parameters()]


HOOKS = {
    "forward pre": lambda m, f: m.register_forward_pre_hook(lambda *a: f()),
    "forward": lambda m, f: m.register_forward_hook(lambda *a: f()),
    "backward pre": lambda m, f: m.register_full_backward_pre_hook(lambda *a: f()),
    "backward": lambda m, f: m.register_full_backward_hook(lambda *a: f()),
}


@pytest.mark.parametrize("kind", HOOKS)
@pytest.mark.parametrize("name", ["mlp", "post_attention_layernorm"])
def test_hooks_on_either_module_run(name, kind):
    m, ids = model(True)
    calls = []
    HOOKS[kind](getattr(m.model.layers["0"], name), lambda: calls.append(1))
    gradients(m, ids)
    assert calls == [1]


def test_a_checkpointed_mlp_stays_checkpointed():
    m, ids = model(True)
    plain, _ = model(False)
    runs = []
    forward = LlamaMLP.forward
    try:
        LlamaMLP.forward = lambda self, *a, **k: (runs.append(1), forward(self, *a, **k))[1]
        n = apply_activation_checkpointing(m, lambda x: isinstance(x, LlamaMLP))
        got = gradients(m, ids)
    finally:
        LlamaMLP.forward = forward
    assert len(runs) == 2 * n  # once forward, once again in the backward
    for a, b in zip(got, gradients(plain, ids)):
        assert torch.equal(a, b)  # nothing was rounded to 8 bits
