"""Host logic of tree speculation on the CPU: rows, masks and rotary positions that go down, the walk over the target's arg-max
rows, what is kept in the cache, refusals - over a stand-in for the decoder whose "model" is a hash of the sequence so far."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import ops, serve  # noqa: E402
from test_serve_host_logic import VOCAB, FakeDecoder, _next, greedy  # noqa: E402


class TreeDecoder(FakeDecoder):
    def __init__(self, monkeypatch, **kw):
        super().__init__(**kw)
        self.page_table = self.pages_of_the_stack = object()
        monkeypatch.setattr(ops, "kv_keep", self.keep)

    def set_tree_rows(self, slots, positions, tokens, base, rope, masks):
        self.set_rows(slots, positions, tokens)
        self.tree = list(zip(slots, positions, tokens, base, rope, masks))
        assert len(masks) == len(slots) and all(len(m) == len(masks[0]) for m in masks)

    def run(self, kind, n, *, graph=True):
        if kind != "tree":
            return super().run(kind, n, graph=graph)
        self.runs.append((kind, n, graph))
        assert n == len(self.tree)
        for slot, pos, token, *_ in self.tree:
            if slot >= 0:
                assert pos <= self.pages[slot]
                self.cache[slot][pos] = token
        for i, (slot, pos, token, base, rope, mask) in enumerate(self.tree):
            if slot < 0:
                continue
            nodes = [j for j in range(64 * len(mask)) if mask[j // 64] >> j % 64 & 1]
            assert base + nodes[-1] == pos and rope == base + len(nodes) - 1
            history = [self.cache[slot][p] for p in range(base)] + [self.cache[slot][base + j] for j in nodes]
            self.next_token[i] = _next(history)

    def keep(self, slots, base, path, count, table, pages):
        assert table is self.page_table
        for s, b, p, c in zip(slots.tolist(), base.tolist(), path.tolist(), count.tolist()):
            old = dict(self.cache[s])
            for j in range(1, c):
                self.cache[s][b + j] = old[b + p[j]]


def test_a_walk_emits_the_target_s_tokens_and_keeps_its_path(monkeypatch):
    d = TreeDecoder(monkeypatch, max_rows=16)
    b = serve.Batcher(d)
    p1, p2 = [5, 6, 7], [9, 9, 9, 9]
    s1, s2 = b.admit(p1), b.admit(p2)
    w1, w2 = greedy(p1, 12), greedy(p2, 12)
    wrong = lambda t: (t + 1) % VOCAB
    # the first: the right token second among three siblings, its child right, the grandchild wrong; the second: nothing right
    out = b.verify_trees({s1: ([wrong(w1[1]), w1[1], 3, w1[2], wrong(w1[3])], [0, 0, 0, 2, 4]), s2: ([wrong(w2[1])] * 2, [0, 1])})
    assert out == {s1: w1[1:4], s2: w2[1:2]}
    assert d.runs[-1] == ("tree", 16, True) and [r[0] for r in d.tree[9:]] == [-1] * 7       # nine nodes in the bucket of 16
    assert b.active[s1]["pos"] == len(p1) + 3 and b.active[s2]["pos"] == len(p2) + 1
    assert b.step() == {s1: w1[4], s2: w2[2]}                    # the kept entries are where plain steps expect them
    out = b.verify_trees({s2: (w2[3:7], [0, 1, 2, 3])})          # a chain, all right
    assert out == {s2: w2[3:8]}
    out = b.verify_trees({s1: ([], [])})                         # no drafts: a plain step
    assert out == {s1: [w1[5]]} and b.verify_trees({}) == {}
    # the same token twice below one node: the first is followed
    out = b.verify_trees({s1: ([w1[6], w1[6], w1[7]], [0, 0, 2])})
    assert out == {s1: w1[6:8]}


def test_refusals(monkeypatch):
    d = TreeDecoder(monkeypatch, max_rows=8)
    b = serve.Batcher(d)
    slot = b.admit([1, 2])
    before = (dict(b.active[slot]), list(d.runs))
    for bad in (([1, 2], [0]), ([1], [-1]), ([1, 2], [0, 2]), ([1] * 8, [0] * 8)):
        with pytest.raises(ValueError):
            b.verify_trees({slot: bad})
    assert (dict(b.active[slot]), list(d.runs)) == before


def test_generate_with_a_tree_drafter(monkeypatch):
    d = TreeDecoder(monkeypatch, max_rows=8)
    session = serve.FastSession(d)
    slot = session.batcher.admit([4, 4])
    st = serve.State(slot, 2, session.batcher.active[slot]["tokens"])
    want = greedy([4, 4], 14)

    def drafter(state):                                          # two right tokens and a wrong one
        n = len(session.batcher.active[state.slot]["tokens"])
        right = greedy([4, 4], n + 2)[n:]
        return [0, right[0], right[1]], [0, 0, 2]

    assert list(session.generate(st, max_tokens=9, tree_drafter=drafter)) == want[:9]
    assert session.batcher.active[slot]["pos"] == 2 + 8
    assert list(session.generate(st, max_tokens=3)) == want[9:12]
