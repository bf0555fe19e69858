"""A tree pass that is refused leaves the decoder as it was: no pages taken, no rows queued (on the CPU, over a stand-in)."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import serve  # noqa: E402
from test_serve_host_logic import greedy  # noqa: E402
from test_serve_trees_host import TreeDecoder  # noqa: E402


def test_no_pages_are_taken_for_a_refused_pass(monkeypatch):
    d = TreeDecoder(monkeypatch, max_rows=8)
    b = serve.Batcher(d)
    one, two = b.admit([1, 2]), b.admit([3])
    pages, runs, rows = dict(d.pages), list(d.runs), d.row_pos.clone()
    for bad in ({one: ([1] * 4, [0] * 4), two: ([1] * 4, [0] * 4)}, {one: ([1] * 9, [0] * 9)}, {one: ([1], [0]), two: ([1, 2], [0])}, {one: ([1], [0]), two: ([1], [1])}):
        with pytest.raises(ValueError):
            b.verify_trees(bad)
        assert d.pages == pages and d.runs == runs and torch.equal(d.row_pos, rows)
    with pytest.raises(KeyError):
        b.verify_trees({one: ([1], [0]), 5: ([1], [0])})
    assert d.pages == pages


def test_passes_between_the_largest_bucket_and_the_decoder_s_rows(monkeypatch):
    """A decoder of 12 rows has buckets of up to 8: passes of 9 to 12 nodes run as they are."""
    d = TreeDecoder(monkeypatch, max_rows=12)
    b = serve.Batcher(d)
    slot = b.admit([1, 2, 3])
    want = greedy([1, 2, 3], 30)
    for drafts in (7, 8, 11):
        n = len(b.active[slot]["tokens"])
        assert b.verify_trees({slot: (want[n:n + drafts], list(range(drafts)))}) == {slot: want[n:n + drafts + 1]}
        assert d.runs[-1] == ("tree", drafts + 1, True)
    pages = dict(d.pages)
    with pytest.raises(ValueError, match="larger"):
        b.verify_trees({slot: ([1] * 12, [0] * 12)})
    assert d.pages == pages
