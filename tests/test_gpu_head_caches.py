"""Draft heads come and go over one decoder: the cache of one that is gone is neither held nor copied (needs a B200)."""
import gc

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("fmt", ["bf16", "q4"])
def test_a_head_that_is_gone_leaves_nothing_behind(dev, fmt, monkeypatch):
    from georefine_b200 import ops, serve

    cfg = serve.DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
    d = serve.BatchDecoder(serve.DecoderWeights.synthetic(cfg, dev, seed=3, max_m=64), max_rows=64, max_slots=8, max_context=1024, device=dev, kv_format=fmt)
    copied = []
    copy = ops.kv_copy
    monkeypatch.setattr(ops, "kv_copy", lambda src, dst, pages, **kw: (copied.append(pages), copy(src, dst, pages, **kw)))
    prompt = torch.randint(0, cfg.vocab, (300,), generator=torch.Generator().manual_seed(7)).tolist()

    def serve_some():
        spec = serve.MTPSpeculator(serve.Batcher(d), serve.MTPHead.synthetic(d), k=2)
        slot = spec.admit(prompt)
        child, = spec.fork(slot)
        for _ in range(3):
            spec.cycle()
        tokens = [spec.b.active[s]["tokens"] for s in (slot, child)]
        assert tokens[0] == tokens[1] and list(d.page_sets) == [spec.head.cache] and set(copied) == {spec.head.cache}
        spec.retire(slot)
        spec.retire(child)
        return tokens[0]

    serve_some()                                  # (kernels are loaded, graphs' pools are there)
    copied.clear()
    gc.collect()
    assert not list(d.page_sets)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated(dev)
    first = serve_some()
    copied.clear()
    gc.collect()
    assert not list(d.page_sets) and torch.cuda.memory_allocated(dev) <= held
    b = serve.Batcher(d)
    slot = b.admit(prompt)
    d.fork_slot(slot, 300)
    assert not copied                             # the trunk's pages are forked in one call, and there are no others
    assert serve_some() == first
