"""The engine over a 4-bit cache, sequences forked from one prompt, pages compacted, other rotary positions: the operators together, as a
user runs them (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "e4m3", "q4"]


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

    return serve.BatchDecoder(small[1], **{**dict(max_rows=64, max_slots=8, max_context=1024, device=dev), **kw})


def _prompt(cfg, n, seed=7):
    return torch.randint(0, cfg.vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def _greedy(d, prompt, n):
    from georefine_b200 import serve

    b = serve.Batcher(d)
    slot = b.admit(prompt)
    while len(b.active[slot]["tokens"]) < n:
        b.step()
    out = b.active[slot]["tokens"]
    b.retire(slot)
    return out[:n]


def _consistent(d):
    """The host's books: every page is free, or named by as many places as its count says; the device's table agrees."""
    named = [int(p) for p in d._table_host.flatten() if p >= 0]
    for p in range(d.scratch_page):
        assert d._refs[p] == named.count(p) and (p in d._free_pages) == (d._refs[p] == 0)
    assert len(set(d._free_pages)) == len(d._free_pages)
    table = d.page_table.cpu().numpy()
    assert ((table == d._table_host) | ((d._table_host < 0) & (table == d.scratch_page))).all()


def test_a_4_bit_cache_in_the_engine(dev, small):
    """Batches, chains and trees of drafts give the tokens of plain decoding; the bytes of a step are what they should be."""
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format="q4")
    assert d.streamed_bytes([100])["kv"] == 100 * cfg.kv_heads * 2 * cfg.layers * 69
    prompts = [_prompt(cfg, n, n) for n in (5, 250, 257, 31)]
    alone = [_greedy(d, p, 12) for p in prompts]
    b = serve.Batcher(d)
    slots = [b.admit(p) for p in prompts]
    for _ in range(4):
        b.step()
    assert all(b.active[s]["tokens"] == want[:5] for s, want in zip(slots, alone))
    out = b.verify({slots[0]: alone[0][5:8], slots[1]: [0, 0], slots[2]: [alone[2][5], 0]})
    assert out[slots[0]] == alone[0][5:9] and out[slots[1]] == alone[1][5:6] and out[slots[2]] == alone[2][5:5 + len(out[slots[2]])]
    tree = b.verify_trees({slots[3]: ([3, alone[3][5], 7, alone[3][6]], [0, 0, 1, 2])})
    assert tree[slots[3]] == alone[3][5:8]
    while any(len(b.active[s]["tokens"]) < 12 for s in slots):
        b.step(only=[s for s in slots if len(b.active[s]["tokens"]) < 12])
    assert all(b.active[s]["tokens"][:12] == want for s, want in zip(slots, alone))
    _consistent(d)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("length", [255, 256, 300, 513])
def test_forks_go_on_as_sequences_of_their_own(dev, small, fmt, length):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format=fmt)
    prompt = _prompt(cfg, length)
    want = _greedy(d, prompt, 8)
    forced = {}
    for t in (5, 6):                              # what a sequence does that is given another next token
        forced[t] = _greedy(d, prompt + [t], 6)
    b = serve.Batcher(d)
    slot = b.admit(prompt)
    free = len(d._free_pages)
    children = b.fork(slot, 3)
    shared = length // 256
    assert free - len(d._free_pages) == (3 if length % 256 else 0) and int(d._refs[d._table_host[slot, 0]]) == (4 if shared else 1)
    _consistent(d)
    for child, t in zip(children[1:], forced):
        b.active[child]["tokens"][-1] = t
        b._dirty = True
    for _ in range(5):
        b.step()
    assert b.active[slot]["tokens"] == want[:6] and b.active[children[0]]["tokens"] == want[:6]
    for child, t in zip(children[1:], forced):
        assert b.active[child]["tokens"][1:] == forced[t][:5]
    # a fork of a fork, after the parent has ended
    b.retire(slot)
    grandchild, = b.fork(children[0])
    b.retire(children[0])
    b.step()
    assert b.active[grandchild]["tokens"] == want[:7]
    _consistent(d)
    for s in list(b.active):
        b.retire(s)
    assert len(d._free_pages) == free + d.pages_per_seq * 0 + -(-(length + 1) // 256) and int(d._refs.sum()) == 0


@pytest.mark.parametrize("fmt", FORMATS)
def test_going_back_into_shared_pages_copies_them(dev, small, fmt):
    """A state rolled back behind a fork writes to pages that its sibling reads: the sibling's tokens stay."""
    from georefine_b200 import serve

    cfg, _ = small
    session = serve.FastSession(_decoder(small, dev, kv_format=fmt))
    prompt = _prompt(cfg, 250)
    st = session.prefill(token_ids=prompt)
    tokens = list(session.generate(st, max_tokens=20))
    child, = session.fork(st)
    session.rollback(child, 15)                   # to position 254, in the page that both share
    session.extend(child, [9, 8, 7, 6, 5])
    assert int(session.d._refs[session.d._table_host[st.slot, 0]]) == 1
    _consistent(session.d)
    went = list(session.generate(child, max_tokens=4))
    more = list(session.generate(st, max_tokens=6))
    check = session.prefill(token_ids=prompt)
    assert list(session.generate(check, max_tokens=26)) == tokens + more
    session.rollback(check, 21)
    session.extend(check, [9, 8, 7, 6, 5])
    assert list(session.generate(check, max_tokens=4)) == went
    _consistent(session.d)


@pytest.mark.parametrize("fmt", FORMATS)
def test_compacted_pages_read_as_before(dev, small, fmt):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, kv_format=fmt)
    prompts = [_prompt(cfg, n, n) for n in (300, 520, 100, 700)]
    want = [_greedy(d, p, 12) for p in prompts]
    b = serve.Batcher(d)
    slots = [b.admit(p) for p in prompts]
    child, = b.fork(slots[3])
    for _ in range(3):
        b.step()
    b.retire(slots[0])
    b.retire(slots[2])
    used = d.compact_pages()
    assert used == len({int(p) for p in d._table_host.flatten() if p >= 0}) and d._table_host.max() < used
    _consistent(d)
    late = b.admit(prompts[0])
    for _ in range(8):
        b.step()
    for s, i in ((slots[1], 1), (slots[3], 3), (child, 3)):
        assert b.active[s]["tokens"] == want[i]
    assert b.active[late]["tokens"] == want[0][:9] and d.compact_pages() == used + 2
    _consistent(d)


def test_full_pools_are_refused_and_nothing_is_lost(dev, small):
    from georefine_b200 import serve

    cfg, _ = small
    d = _decoder(small, dev, max_slots=3, max_context=256, kv_format="q4")
    b = serve.Batcher(d)
    slot = b.admit(_prompt(cfg, 100))
    with pytest.raises(RuntimeError, match="slot"):
        b.fork(slot, 3)
    for bad in (0, 300, 257):
        with pytest.raises(ValueError, match="positions"):
            d.fork_slot(slot, bad)
    b.fork(slot, 2)
    _consistent(d)
    with pytest.raises(RuntimeError, match="slot"):
        b.fork(slot)
    _consistent(d)


def test_a_draft_head_forks_with_its_trunk(dev, small):
    from georefine_b200 import serve

    for fmt in FORMATS:
        d = _decoder(small, dev, kv_format=fmt)
        spec = serve.MTPSpeculator(serve.Batcher(d), serve.MTPHead.synthetic(d), k=2)
        prompt = _prompt(small[0], 300)
        want = _greedy(d, prompt, 20)
        slot = spec.admit(prompt)
        spec.cycle()
        child, = spec.fork(slot)
        heads = []
        for _ in range(4):
            spec.cycle()
            heads.append((spec.first[slot], spec.first[child]))
        assert spec.b.active[slot]["tokens"] == spec.b.active[child]["tokens"]
        n = min(20, len(spec.b.active[slot]["tokens"]))
        assert spec.b.active[slot]["tokens"][:n] == want[:n] and all(a == c for a, c in heads)
        _consistent(d)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("length", [255, 256, 300])
def test_a_forked_draft_head_has_seen_the_pending_token(dev, small, length, fmt):
    """The head's entries are the parent's up to the pending token's, whose page the trunk may not have asked for; cycles go on alike."""
    from georefine_b200 import ops, serve

    d = _decoder(small, dev, kv_format=fmt)
    # (pages that forks may get hold something else than zeros)
    spec = serve.MTPSpeculator(serve.Batcher(d), serve.MTPHead.synthetic(d), k=3)
    spec.retire(spec.admit(_prompt(small[0], 900, 8)))
    slot = spec.admit(_prompt(small[0], length))
    children = spec.fork(slot, 2)
    _consistent(d)
    n = length + 1

    def entries(s):                               # (the head's first is that of position 1)
        k, v = (torch.empty(n - 1, 2, 128, device=dev, dtype=torch.bfloat16) for _ in range(2))
        i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device=dev)
        ops.kv_read(i32([s] * (n - 1)), i32(range(1, n)), d.page_table, spec.head.cache, k, v)
        return torch.stack([k, v])

    want = entries(slot)
    assert bool(want.abs().amax(dim=(0, 2, 3)).gt(0).all()) and all(torch.equal(entries(c), want) for c in children)
    for _ in range(3):
        spec.cycle()
        for c in children:
            assert spec.first[c] == spec.first[slot] and torch.equal(spec.hidden[c], spec.hidden[slot])
    assert all(spec.b.active[c]["tokens"] == spec.b.active[slot]["tokens"] for c in children)
    _consistent(d)


ROPES = {"interleaved": dict(rope_layout="interleaved"), "part": dict(rope_dim=64), "both": dict(rope_layout="interleaved", rope_dim=32),
         "yarn": dict(rope_scaling={"kind": "yarn", "factor": 4.0, "original": 256}), "part, linear": dict(rope_dim=96, rope_scaling={"kind": "linear", "factor": 2.0})}


@pytest.mark.parametrize("name", ROPES)
@pytest.mark.parametrize("fmt", ["bf16", "q4"])
def test_other_rotary_positions_in_the_engine(dev, name, fmt):
    """First-layer keys are the formula's, and batches, verify passes and trees agree with plain decoding."""
    from georefine_b200 import ops, serve

    cfg = serve.DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=1024, vocab=1000, **ROPES[name])
    assert hash(cfg) == hash(serve.DecoderConfig(**{f: getattr(cfg, f) for f in cfg.__dataclass_fields__}))
    small = cfg, serve.DecoderWeights.synthetic(cfg, dev, seed=3, max_m=64)
    d = _decoder(small, dev, kv_format=fmt)
    prompt = _prompt(cfg, 60)
    b = serve.Batcher(d)
    slot = b.admit(prompt)
    if fmt == "bf16":                             # (whose keys are off by their roundings alone)
        d._tree_attention()
        k, v = (torch.empty(60, 2, 128, device=dev, dtype=torch.bfloat16) for _ in range(2))
        i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device=dev)
        ops.kv_read(i32([slot] * 60), i32(range(60)), d.page_table, d.pages.layer(0), k, v)
        w = d.w
        x, h = torch.empty(60, 512, device=dev, dtype=torch.bfloat16), w.embed[torch.tensor(prompt, device=dev)].clone()
        ops.rmsnorm(h, w.layers[0].norm1, x, eps=cfg.eps)
        qkv = torch.empty(60, cfg.qkv_rows, device=dev, dtype=torch.bfloat16)
        w.layers[0].qkv(x, qkv)
        rope = ops.Rope(cfg.rope_dim or 128, cfg.rope_theta, layout=cfg.rope_layout, scaling=cfg.rope_options, device=dev)
        raw = qkv[:, 512:768].unflatten(1, (2, 128)).float().contiguous()
        want = ops.rotary(raw.clone(), torch.arange(60, device=dev), rope)
        # one rounding of the rotated key (2^-8), or tables, products and sums rounded (four of them, of either component)
        pair = raw.abs() + raw.abs().amax(-1, keepdim=True)
        assert bool(((k.float() - want).abs() <= 2.0 ** -8 * want.abs() + (4 * 2.0 ** -8 * pair * rope.factor if d.rope is None else 0)).all())
        assert torch.equal(v, qkv[:, 768:].unflatten(1, (2, 128)))
    for _ in range(5):
        b.step()
    plain = b.active[slot]["tokens"]
    other = b.admit(prompt)
    assert b.verify({other: plain[1:4]})[other] == plain[1:5]
    third = b.admit(prompt)
    got = b.verify_trees({third: ([plain[1], 3, plain[2]], [0, 0, 1])})[third]
    # A tree over a BF16 cache rounds elsewhere than a step: where its walk leaves plain decoding, the two tokens' logits are within that
    # rounding - a layer's attention and the logits themselves rounded to BF16 once in either pass, with the norms and linears between: eight halves of a step of 2^-8.
    for row, (a, c) in zip((0, 1, 3), zip(got, plain[1:])):
        if a != c:
            logits = d.logits[row].float()
            assert fmt == "bf16" and float((logits[a] - logits[c]).abs()) <= 8 * 2.0 ** -8 * float(logits.abs().amax())
            break
