"""Rotary positions of a checkpoint's configuration that no model can mean, and keys that say what is done anyway.  No GPU."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import checkpoint  # noqa: E402
from georefine_b200.serving import ContextServingError  # noqa: E402

BASE = dict(hidden_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=1024, vocab_size=1000, rope_theta=5000.0,
            max_position_embeddings=8192)


@pytest.mark.parametrize("given", [
    dict(rope_scaling={"type": "linear", "factor": -2.0}), dict(rope_scaling={"type": "linear", "factor": 0}), dict(rope_scaling={"type": "linear", "factor": float("nan")}),
    dict(rope_scaling={"rope_type": "yarn", "factor": 4.0, "beta_fast": 1, "beta_slow": 2}), dict(rope_scaling={"rope_type": "yarn", "factor": 4.0, "attention_factor": -1.0}),
    dict(rope_scaling={"rope_type": "yarn", "factor": 4.0, "attention_factor": "much"}), dict(rope_scaling={"rope_type": "yarn", "factor": 4.0}, rope_theta=1.0),
    dict(rope_scaling={"low_freq_factor": 4.0, "high_freq_factor": 1.0, "factor": 2.0}), dict(partial_rotary_factor=1.5), dict(partial_rotary_factor=0.001), dict(partial_rotary_factor=0.4),
    dict(rope_scaling="linear"), dict(rope_scaling=[1, 2]), dict(rope_parameters={"rope_theta": None, "rope_type": "default"}), dict(rope_parameters={"rope_theta": "large"}),
])
def test_numbers_that_mean_nothing_are_refused_as_the_checkpoint_s(given):
    with pytest.raises(ContextServingError):
        checkpoint.decoder_config({**BASE, **given})


def test_an_override_is_the_caller_s_mistake():
    with pytest.raises(ValueError):
        checkpoint.decoder_config(BASE, tp_world=3)


@pytest.mark.parametrize("truncate", [True, None])
def test_whole_numbers_at_the_ends_of_yarn_s_ramp_may_be_asked_for(truncate):
    """They are what the ramp has anyway; a ramp between broken numbers is another one."""
    plain = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}
    cfg = checkpoint.decoder_config({**BASE, "rope_scaling": {**plain, "truncate": truncate}})
    assert cfg.rope_options == checkpoint.decoder_config({**BASE, "rope_scaling": plain}).rope_options


@pytest.mark.parametrize("scaling", [{"rope_type": "yarn", "factor": 4.0, "truncate": False}, {"rope_type": "linear", "factor": 4.0, "truncate": True}])
def test_other_ends_of_a_ramp_are_refused(scaling):
    with pytest.raises(ContextServingError):
        checkpoint.decoder_config({**BASE, "rope_scaling": scaling})
