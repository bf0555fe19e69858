"""What ``Sampler.verify`` hands to the verifier and refuses, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, ops, sampling  # noqa: E402


def test_sequences_of_more_nodes_than_are_looked_at(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_launch", lambda device, name, *args: calls.append(args))
    s = sampling.Sampler(1.0, device="cpu", seed=1)
    go = lambda *sizes: s.verify(torch.zeros(sum(sizes), 12), [0] * sum(sizes), [p for n in sizes for p in range(-1, n - 1)], [sum(sizes[:i]) for i in range(len(sizes) + 1)])
    tokens, rows, count = go(256, 3)
    step = _native.VerifyStep.from_buffer_copy(calls.pop()[0])
    assert (step.rows, step.seqs, step.width, tokens.shape) == (259, 2, 256, (2, 256))
    for sizes in ((257,), (3, 300)):
        with pytest.raises(ValueError, match="256"):
            go(*sizes)
    assert not calls
