"""What the engine does when an attention reports that it gave up a wait: on the CPU over a stand-in for the decoder, and on a GPU with a
status word that the host sets (no kernel gives up)."""
import types

import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import ops, serve  # noqa: E402
from test_serve_host_logic import VOCAB, greedy  # noqa: E402
from test_serve_trees_host import TreeDecoder  # noqa: E402


class Reporting(TreeDecoder):
    """A decoder whose next check fails when it is told to, once."""
    fail, kept = False, 0

    def check_status(self):
        if self.fail:
            self.fail = False
            raise RuntimeError("attention reported status 16")

    def keep(self, *args):
        self.kept += 1
        super().keep(*args)


def _state(b, slot):
    return list(b.active[slot]["tokens"]), b.active[slot]["pos"]


def test_nothing_of_a_failed_pass_counts_and_the_next_one_goes_on(monkeypatch):
    d = Reporting(monkeypatch, max_rows=16)
    b = serve.Batcher(d)
    prompt = [5, 6, 7]
    want = greedy(prompt, 20)
    d.fail = True
    free = len(d._free)
    with pytest.raises(RuntimeError, match="status"):
        b.admit(prompt)
    assert len(d._free) == free and not b.active
    slot = b.admit(prompt)
    calls = {"step": lambda: b.step(), "verify": lambda: b.verify({slot: want[len(b.active[slot]["tokens"]):][:2]}),
             "trees": lambda: b.verify_trees({slot: ([(want[len(b.active[slot]["tokens"])] + 1) % VOCAB, want[len(b.active[slot]["tokens"])]], [0, 0])})}
    for name, call in calls.items():
        before, kept = _state(b, slot), d.kept
        d.fail = True
        with pytest.raises(RuntimeError, match="status"):
            call()
        assert _state(b, slot) == before and d.kept == kept, name
        got = call()[slot]
        assert b.active[slot]["tokens"] == want[:len(b.active[slot]["tokens"])] and len(b.active[slot]["tokens"]) > len(before[0]), (name, got)
    assert b.step(fetch=False) is None
    d.fail = True
    with pytest.raises(RuntimeError, match="status"):
        b.sync_tokens()
    b.sync_tokens()
    n = len(b.active[slot]["tokens"])
    assert b.active[slot]["tokens"] == want[:n]
    b.retire(slot)


def test_a_sampled_tree_of_a_failed_pass_is_not_kept(monkeypatch):
    d = Reporting(monkeypatch, max_rows=16)
    b = serve.Batcher(d)
    slot = b.admit([5, 6, 7])
    sampler = types.SimpleNamespace(verify=lambda logits, tokens, parents, starts: (torch.tensor([[3, -1]]), torch.tensor([[0, -1]]), torch.tensor([1])))
    before = _state(b, slot)
    d.fail = True
    with pytest.raises(RuntimeError, match="status"):
        b.verify_trees({slot: ([1], [0])}, sampler=sampler)
    assert _state(b, slot) == before and d.kept == 0


def test_the_word_is_read_where_the_pass_left_it_and_cleared():
    d = object.__new__(serve.BatchDecoder)
    d._status_host = None
    d.check_status()                                   # a decoder that has no such attention
    d._status_host, d._tree_attn = torch.zeros(1, dtype=torch.int32), ops.TreeAttention(4, 2, 4, 1, "cpu")
    d.check_status()
    d._tree_attn.status.fill_(16)
    d.check_status()                                   # (no pass has brought it over)
    d._status_host.copy_(d._tree_attn.status)
    with pytest.raises(RuntimeError, match="16"):
        d.check_status()
    d.check_status()
    assert int(d._status_host) == int(d._tree_attn.status) == int(d._tree_attn.scratch[0]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_a_status_that_the_host_sets(fmt):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    cfg = serve.DecoderConfig(hidden=512, layers=1, heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=512)
    d = serve.BatchDecoder(serve.DecoderWeights.synthetic(cfg, "cuda:0", seed=3, max_m=64), max_rows=64, max_slots=2, max_context=512, kv_format=fmt)
    b = serve.Batcher(d)
    slot = b.admit([5, 6, 7])
    tree = {slot: ([1, 2], [0, 1])}
    want = b.verify_trees(tree)[slot]
    b.retire(slot)
    slot = b.admit([5, 6, 7])
    for _ in range(2):                                 # (the second time over a graph that was captured before)
        d._tree_attn.status.fill_(16)
        with pytest.raises(RuntimeError, match="status 16"):
            b.verify_trees({slot: tree[next(iter(tree))]})
    assert b.verify_trees({slot: ([1, 2], [0, 1])})[slot] == want
    d._tree_attn.status.fill_(16)
    if fmt == "e4m3":
        for call in (b.step, lambda: b.verify({slot: [1]}), lambda: b.admit([4, 4])):
            d._tree_attn.status.fill_(16)
            with pytest.raises(RuntimeError, match="status 16"):
                call()
    else:
        b.step()                                       # steps over a BF16 cache do not go through that attention
        with pytest.raises(RuntimeError, match="status 16"):
            b.verify_trees({slot: ([1], [0])})
    b.step()


def test_a_failed_prompt_of_a_sequence_with_a_draft_head(monkeypatch):
    d = Reporting(monkeypatch, max_rows=16)
    d.h = torch.zeros(16, 4)
    absorbed = []
    head = types.SimpleNamespace(absorb=lambda slots, *rest: absorbed.append(slots) or [0] * len(slots), z=torch.zeros(16, 4))
    spec = serve.MTPSpeculator(serve.Batcher(d), head, k=2)
    free = len(d._free)
    d.fail = True
    with pytest.raises(RuntimeError, match="status"):
        spec.admit([5, 6, 7])
    assert len(d._free) == free and not spec.b.active and not spec.first
    slot = spec.admit([5, 6, 7])
    assert spec.b.active[slot]["tokens"] == greedy([5, 6, 7], 1) and slot in spec.first
