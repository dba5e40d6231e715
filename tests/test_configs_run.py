"""Every configuration that is shipped can be started as it stands: what the training command checks before
its first step holds for it."""
import glob
import os

import pytest

from femtotron_b200.scripts import train

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CONFIGS = sorted(os.path.basename(p) for p in glob.glob(os.path.join(ROOT, "configs", "*.yaml")))


@pytest.mark.parametrize("name", CONFIGS)
def test_configuration(name):
    cfg = train.load_config(train.parse_args(["--config", os.path.join(ROOT, "configs", name)]))
    assert 0 <= cfg["warmup_steps"] <= cfg["train_steps"]
    assert cfg["ac_bits"] in (8, 16) and not (cfg["ac_bits"] == 8 and cfg["ac_use_reentrant"])
    if not cfg.get("model_name"):
        mc = train.model_config_from(cfg)
        if getattr(mc, "rotary_spec", None) is not None:
            from femtotron_b200.models.layers import rotary_spec_of
            from femtotron_b200.ops import rotary
            spec = rotary_spec_of(mc)
            rotary.inv_frequencies(spec["rot"], cfg["rope_theta"], spec["scaling"], trained=cfg["max_position_embeddings"],
                                   length=cfg["seq_len"])
