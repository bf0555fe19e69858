"""Temperatures that the verification of drafts refuses, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, sampling  # noqa: E402

P = 1 << 20           # stands for device memory: aligned, never touched


@pytest.mark.parametrize("temperature", [0.0, -1.0, 5e-324, 1e-31, 1e21, float("inf"), float("nan")])
def test_outside_the_range(temperature):
    v = sampling.DraftVerifier(8, 2, 4, "cpu")
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    with pytest.raises(ValueError, match="temperature"):
        v(torch.zeros(6, 10), i32(6), i32(3), torch.zeros(6), torch.zeros(2), temperature=temperature)
    s = _native.VerifyStep()
    for name, value in dict(logits=P, ldl=1000, tokens=P, starts=P, u_keep=P, u_draw=P, stats=P, out_tokens=P, out_rows=P, out_count=P, rows=6, seqs=2, vocab=1000, width=6,
                            temperature=temperature).items():
        setattr(s, name, value)
    assert _native.lib().grb_verify_drafts(s, None) == 1
