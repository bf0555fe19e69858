"""Scalings of rotary positions at the edges of their rules.  No GPU."""
import math

import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import ops  # noqa: E402


@pytest.mark.parametrize("factor,want", [(0.25, 1.0), (0.999, 1.0), (1.0, 1.0), (1.5, 0.1 * math.log(1.5) + 1), (32.0, 0.1 * math.log(32.0) + 1)])
def test_yarn_leaves_components_as_they_are_where_a_context_is_not_extended(factor, want):
    """The factor on both components grows with the extension, from 1 on: a shorter context takes none."""
    scaling = {"kind": "yarn", "factor": factor, "original": 4096}
    assert math.isclose(ops.rope_frequencies(64, 1e4, scaling)[1], want, rel_tol=1e-15)
    assert math.isclose(ops.Rope(64, 1e4, scaling=scaling, device="cpu").factor, want, rel_tol=1e-15)
    assert ops.rope_frequencies(64, 1e4, {**scaling, "attention": 0.75})[1] == 0.75


@pytest.mark.parametrize("scaling", [{"kind": "linear", "factor": None}, {"kind": "ntk", "factor": None}, {"kind": "yarn", "factor": 4.0, "original": None}, {"kind": "yarn", "factor": 4.0, "original": 64, "slow": None},
                                     {"kind": "bands", "factor": 2.0, "original": 64, "low": None, "high": 4.0}])
def test_only_yarn_s_factor_on_components_may_be_left_open(scaling):
    from georefine_b200 import serve

    with pytest.raises(ValueError, match="positive"):
        ops.rope_frequencies(64, 1e4, scaling)
    with pytest.raises(ValueError, match="positive"):
        serve.DecoderConfig(rope_scaling=scaling)


@pytest.mark.parametrize("kw", [dict(scaling={"kind": "linear", "factor": 5e-324}), dict(scaling={"kind": "linear", "factor": 2.0 ** -60}), dict(theta=1e-200), dict(scaling={"kind": "ntk", "factor": 1e-300})])
def test_pairs_that_turn_too_far_a_position_are_refused(kw):
    """Of 2^60 radians and more, 40 digits hold no fraction of a turn to 2^-64."""
    for call in (lambda: ops.rope_frequencies(64, **kw), lambda: ops.Rope(64, device="cpu", **kw)):
        with pytest.raises(ValueError, match="radians"):
            call()
    assert ops.rope_frequencies(2, 1e4, {"kind": "linear", "factor": 2.0 ** -59})[0] == [2.0 ** 59]
