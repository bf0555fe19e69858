"""The engine over an 8-bit cache, and draft trees through the engine (needs a B200): the operators together, as a user runs them."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.fixture(scope="module")
def small(dev):
    from georefine_b200 import serve

    cfg = serve.DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000)
    return cfg, serve.DecoderWeights.synthetic(cfg, dev, seed=3, max_m=64)


def _decoder(small, dev, **kw):
    from georefine_b200 import serve

    return serve.BatchDecoder(small[1], max_rows=64, max_slots=8, max_context=1024, device=dev, **kw)


def _prompts(cfg, *lengths):
    g = torch.Generator().manual_seed(7)
    return [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in lengths]


def _greedy(d, prompt, n):
    from georefine_b200 import serve

    b = serve.Batcher(d)
    slot = b.admit(prompt)
    out = list(b.active[slot]["tokens"])
    while len(out) < n:
        out.append(b.step()[slot])
    b.retire(slot)
    return out


def test_an_8_bit_cache_holds_what_the_bf16_cache_holds_to_its_rounding(dev, small):
    """The first layer's keys and values depend on the prompt alone: there the two caches differ by the code's rounding (2^-4 of a
    value, or half the smallest code of its entry); and the logits of one step stay near."""
    from georefine_b200 import ops, serve

    cfg, _ = small
    prompt, = _prompts(cfg, 300)
    logits, caches = [], []
    for fmt in ops.KV_FORMATS:
        d = _decoder(small, dev, kv_format=fmt)
        b = serve.Batcher(d)
        slot = b.admit(prompt)
        d._tree_attention()
        k, v = (torch.empty(300, cfg.kv_heads, 128, device=dev, dtype=torch.bfloat16) for _ in range(2))
        i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device=dev)
        ops.kv_read(i32([slot] * 300), i32(range(300)), d.page_table, d.pages.layer(0), k, v)
        caches.append((k.float(), v.float()))
        logits.append(d.logits[(len(prompt) - 1) % d.max_rows].float())
        assert d.streamed_bytes([100])["kv"] == 100 * cfg.kv_heads * 2 * cfg.layers * (256 if fmt == "bf16" else 129)
    for which in range(2):
        a, q = caches[0][which], caches[1][which]
        top = a.abs().amax(-1, keepdim=True)
        # (keys of the BF16 cache are themselves off by up to three roundings of 2^-8 of the larger of the two that the rotation mixes)
        assert bool(((a - q).abs() <= 2.0 ** -4 * q.abs() + 2.0 ** -10 * top / 224 + (3 * 2.0 ** -8 * top * 1.5 if which == 0 else 0)).all())
    assert float((logits[0] - logits[1]).norm() / logits[0].norm()) < 0.2


def test_tokens_over_an_8_bit_cache_do_not_depend_on_batch_or_speculation(dev, small):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format="e4m3")
    prompts = _prompts(cfg, 5, 70, 256, 257, 31)
    alone = [_greedy(d, p, 12) for p in prompts]
    b = serve.Batcher(d)
    slots = [b.admit(p) for p in prompts]
    for _ in range(4):
        b.step()
    for s, want in zip(slots, alone):
        assert b.active[s]["tokens"] == want[:5]
    # chains: right drafts, wrong drafts, mixed
    out = b.verify({slots[0]: alone[0][5:8], slots[1]: [0, 0], slots[2]: [alone[2][5], 0], slots[3]: alone[3][5:9]})
    assert out[slots[0]] == alone[0][5:9] and out[slots[1]] == alone[1][5:6] and out[slots[3]] == alone[3][5:10]
    assert out[slots[2]] == alone[2][5:5 + len(out[slots[2]])]
    for s, want in zip(slots, alone):
        while len(b.active[s]["tokens"]) < 11:
            b.step(only=[s])
        assert b.active[s]["tokens"][:11] == want[:11]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_trees_emit_the_tokens_of_plain_decoding(dev, small, fmt):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format=fmt)
    prompts = _prompts(cfg, 9, 250, 300)
    want = [_greedy(d, p, 16) for p in prompts]
    b = serve.Batcher(d)
    slots = [b.admit(p) for p in prompts]
    trees = lambda at: {slots[0]: ([3, want[0][at], 5, want[0][at + 1], want[0][at + 2]], [0, 0, 0, 2, 4]),            # three right ones among wrong
                        slots[1]: ([1, 2, 4], [0, 1, 0]),                                                              # none
                        slots[2]: ([want[2][at], 7, want[2][at + 1], 8, 9, 11, want[2][at + 2]], [0, 1, 1, 2, 3, 0, 3])}
    out = b.verify_trees(trees(1))
    assert out[slots[0]] == want[0][1:5] and out[slots[1]] == want[1][1:2] and out[slots[2]] == want[2][1:5]
    b.step()
    out = b.verify_trees({s: t for s, t in trees(6).items() if s != slots[1]})          # over what the first trees kept
    assert out[slots[0]] == want[0][6:10] and out[slots[2]] == want[2][6:10]
    while len(b.active[slots[0]]["tokens"]) < 14:
        b.step()
    for s, w in zip(slots, want):
        got = b.active[s]["tokens"]
        assert got[:14] == w[:len(got)][:14]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_sampled_trees(dev, small, fmt, top_p):
    """At a temperature near zero sampling is the arg-max path; at 1 the run is reproducible and stays in the nucleus."""
    from georefine_b200 import sampling, serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format=fmt)
    prompt, = _prompts(cfg, 40)
    want = _greedy(d, prompt, 10)
    b = serve.Batcher(d)
    slot = b.admit(prompt)
    cold = sampling.Sampler(1e-4, top_p, device=dev, seed=5)
    out = b.verify_trees({slot: ([8, want[1], want[2], 9], [0, 0, 2, 3])}, sampler=cold)
    assert out[slot] == want[1:4]
    assert b.step() == {slot: want[4]}
    got = []
    for _ in range(2):
        warm = sampling.Sampler(1.0, top_p, device=dev, seed=6)
        s = b.admit(prompt)
        tokens = []
        for _ in range(4):
            tokens += b.verify_trees({s: ([want[1], 3, want[2]], [0, 0, 1])}, sampler=warm)[s]
        got.append(tokens)
        b.retire(s)
    assert got[0] == got[1] and len(got[0]) >= 4


def test_a_session_with_an_8_bit_cache_and_a_tree_drafter(dev, small):
    from georefine_b200 import serve

    cfg, w = small
    session = serve.FastSession.load(weights=w, device=dev, max_len=1024, max_rows=64, kv_format="e4m3")
    prompt, = _prompts(cfg, 33)
    st = session.prefill(token_ids=prompt)
    plain = list(session.generate(st, max_tokens=12))
    session.close(st)
    st = session.prefill(token_ids=prompt)

    def drafter(state):
        n = len(session.batcher.active[state.slot]["tokens"])
        right = (plain + [0] * 4)[n:n + 2]
        return [1, right[0], right[1], 2], [0, 0, 2, 2]

    assert list(session.generate(st, max_tokens=12, tree_drafter=drafter)) == plain
    session.rollback(st, 4)
    session.extend(st, [5, 6, 7])
    more = list(session.generate(st, max_tokens=3))
    session.close(st)
    st = session.prefill(token_ids=prompt + plain[:-4] + [5, 6, 7])
    assert list(session.generate(st, max_tokens=3)) == more


def test_a_draft_head_over_an_8_bit_cache(dev, small):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format="e4m3")
    prompt, = _prompts(cfg, 20)
    want = _greedy(d, prompt, 10)
    b = serve.Batcher(d)
    spec = serve.MTPSpeculator(b, serve.MTPHead.synthetic(d, seed=4), k=3)
    slot = spec.admit(prompt)
    while len(b.active[slot]["tokens"]) < 10:
        spec.cycle()
    assert b.active[slot]["tokens"][:10] == want


def test_refusals(dev, small):
    with pytest.raises(ValueError, match="format"):
        _decoder(small, dev, kv_format="int8")
    d = _decoder(small, dev)
    with pytest.raises(ValueError, match="kind"):
        d.run("trees", 2)
    with pytest.raises(ValueError, match="words"):
        d.set_tree_rows([0], [0], [0], [0], [0], [[1, 1]])
