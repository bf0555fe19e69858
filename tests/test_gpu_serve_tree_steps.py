"""Tree steps of the engine outside ``Batcher.verify_trees``: captured ahead of time, or run before any tree was queued (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def weights(dev):
    from georefine_b200 import serve

    return serve.DecoderWeights.synthetic(serve.DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000), dev, seed=3, max_m=64)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_captured_ahead_of_time(dev, weights, fmt):
    from georefine_b200 import serve

    trees = {0: ([3, 8, 5, 2], [0, 0, 2, 2])}
    got = []
    for ahead in (False, True):
        d = serve.BatchDecoder(weights, max_rows=64, max_slots=4, max_context=512, device=dev, kv_format=fmt)
        if ahead:
            before = d.kv.view(torch.uint8).clone()
            d.capture([("tree", 8), ("tree", 4)])
            assert ("tree", 8) in d.graphs and torch.equal(d.kv.view(torch.uint8), before)          # rows of no sequence store nothing
        b = serve.Batcher(d)
        slot = b.admit([5, 6, 7, 8, 9])
        got.append([b.verify_trees({slot: trees[0]})[slot] for _ in range(3)] + [b.step()[slot]])
        assert ("tree", 8) in d.graphs
    assert got[0] == got[1]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("graph", [False, True])
def test_run_before_any_tree_was_queued(dev, weights, fmt, graph):
    """The masks are empty then: rows that see nothing."""
    from georefine_b200 import serve

    d = serve.BatchDecoder(weights, max_rows=64, max_slots=4, max_context=512, device=dev, kv_format=fmt)
    d.run("tree", 2, graph=graph)
    assert bool((d.ctx[:2] == 0).all()) and bool(torch.isfinite(d.logits[:2].float()).all())


def test_masks_that_are_refused_leave_the_rows_as_they_were(dev, weights):
    from georefine_b200 import serve

    d = serve.BatchDecoder(weights, max_rows=64, max_slots=4, max_context=512, device=dev)
    d.set_tree_rows([0, 1], [3, 4], [5, 6], [3, 4], [3, 4], [[1], [1]])
    held = [t.clone() for t in (d.row_seq, d.row_pos, d.tokens, d.row_base, d.row_rope, d.row_mask)]
    for bad in ([[1, 1], [1, 1]], [[1]], [1, 1]):
        with pytest.raises(ValueError, match="masks"):
            d.set_tree_rows([2, 3], [7, 8], [9, 9], [7, 8], [7, 8], bad)
        assert all(torch.equal(a, b) for a, b in zip(held, (d.row_seq, d.row_pos, d.tokens, d.row_base, d.row_rope, d.row_mask)))
