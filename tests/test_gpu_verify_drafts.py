"""Verification of drafted tokens from given random numbers, against a walk in plain Python with 64-bit numbers (needs a B200).

Tokens, nodes and counts are whole numbers and have to be equal.  The kernel compares with probabilities off by their exponentials'
2^-22; a case in which the definition itself is nearer to a border than four times that says nothing and is not drawn here."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from spec_reference import walk  # noqa: E402


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _logits(g, rows, vocab, dtype, dev, sharp=6.0):
    x = torch.randn(rows, vocab, generator=g, device=dev)
    likely = torch.randint(vocab, (rows, 4), generator=g, device=dev)
    return x.scatter_add(1, likely, sharp + torch.randn(rows, 4, generator=g, device=dev)).to(dtype)


def _compare(v, logits, tokens, parents, u_keep, u_draw, temperature, *, chain, q=None, width=None):
    """``tokens``, ``parents`` and ``u_keep`` per sequence."""
    dev, starts = logits.device, [0]
    for t in tokens:
        starts.append(starts[-1] + len(t))
    flat = lambda xs: [x for ys in xs for x in ys]
    got = v(logits, _i32(flat(tokens), dev), _i32(starts, dev), torch.tensor(flat(u_keep), device=dev), torch.tensor(u_draw, device=dev), temperature=temperature,
            parent=None if chain else _i32(flat(parents), dev), draft_probs=q)
    out, rows, count = (t.tolist() for t in got)
    for s, (t, p, u) in enumerate(zip(tokens, parents, u_keep)):
        part = slice(starts[s], starts[s + 1])
        want, path, near = walk(logits[part].cpu(), t, p, [float(torch.tensor(x)) for x in u], float(torch.tensor(u_draw[s])), temperature, None if q is None else q[part].cpu())
        assert near > 1e-6, "the inputs are too near to a border to decide"
        assert count[s] == len(want) and out[s] == want + [-1] * (v.width - len(want)) and rows[s] == path + [-1] * (v.width - len(path)), s
    return out, count


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [2, 7, 255, 256, 257, 1003, 20011])
def test_chains(dev, dtype, vocab):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(vocab)
    lengths = [1, 2, 6, 3, 9, 1, 4, 6]
    rows = sum(lengths)
    logits = _logits(g, rows, vocab, dtype, dev)
    best = logits.float().argmax(1).tolist()
    tokens, u, at = [], [], 0
    for i, n in enumerate(lengths):
        tokens.append([0] + [best[at + j] if (i + j) % 4 else (j * 37) % vocab for j in range(n - 1)])
        at += n
        u.append(torch.rand(n, generator=g, device=dev).tolist())
    u_draw = torch.rand(8, generator=g, device=dev).tolist()
    v = sampling.DraftVerifier(rows, 8, 10, dev)
    for temperature in (1.0, 0.6):
        _compare(v, logits, tokens, [list(range(-1, n - 1)) for n in lengths], u, u_draw, temperature, chain=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab,sharp", [(50, 2.0), (4099, 7.0)])
def test_trees(dev, dtype, vocab, sharp):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(vocab)
    trees = [[-1], [-1, 0, 0, 0, 0], [-1, 0, 0, 1, 1, 2, 2, 3, 3, 3], [-1] + [i // 2 for i in range(60)], [-1] + [0] * 99, list(range(-1, 30)), [-1, 0, 1, 0, 3, 2, 2]]
    rows = sum(map(len, trees))
    logits = _logits(g, rows, vocab, dtype, dev, sharp)
    tokens, u, at = [], [], 0
    for parents in trees:
        top = logits[at:at + len(parents)].float().topk(8, dim=1).indices.tolist()
        order = [sum(1 for j in range(1, i) if parents[j] == parents[i]) for i in range(len(parents))]      # (a node's 9th child repeats the first one's token)
        tokens.append([0] + [top[p][order[i] % 8] for i, p in enumerate(parents) if i])
        u.append(torch.rand(len(parents), generator=g, device=dev).tolist())
        at += len(parents)
    v = sampling.DraftVerifier(rows, len(trees), 40, dev)
    for seed in range(3):
        u_draw = torch.rand(len(trees), generator=g, device=dev).tolist()
        _compare(v, logits, tokens, trees, u, u_draw, 0.9, chain=False)
        u = [torch.rand(len(x), generator=g, device=dev).tolist() for x in u]


@pytest.mark.parametrize("vocab", [3, 1000, 4101])
def test_draft_probabilities(dev, vocab):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(vocab)
    lengths = [1, 2, 5, 5, 8, 3]
    rows = sum(lengths)
    logits = _logits(g, rows, vocab, torch.float32, dev, 3.0)
    q = torch.zeros(rows, vocab, device=dev)
    tokens, at = [], 0
    for n in lengths:
        near = logits[at:at + n - 1] + 0.8 * torch.randn(n - 1, vocab, generator=g, device=dev)
        q[at + 1:at + n] = torch.softmax(near, dim=1)
        tokens.append([0] + (torch.multinomial(q[at + 1:at + n], 1, generator=g)[:, 0].tolist() if n > 1 else []))
        at += n
    v = sampling.DraftVerifier(rows, len(lengths), 8, dev)
    seen = set()
    for seed in range(4):
        u = [torch.rand(n, generator=g, device=dev).tolist() for n in lengths]
        out, count = _compare(v, logits, tokens, [list(range(-1, n - 1)) for n in lengths], u, torch.rand(len(lengths), generator=g, device=dev).tolist(), 1.0, chain=True, q=q)
        seen |= set(count)
    assert len(seen) > 2


def test_what_a_draw_gives_at_the_ends(dev):
    """The smallest and largest random numbers, masses of zero, tokens of probability one, infinities, nothing left."""
    from georefine_b200 import sampling

    inf = float("inf")
    logits = torch.full((8, 1000), -inf, device=dev)
    logits[0, [5, 900]] = 0.0                              # two tokens of one half
    logits[1, 999] = 3.0                                   # one certain token, the last of all
    logits[2, 0] = -2.0                                    # and the first
    logits[3] = 0.0                                        # all alike
    logits[4, :] = -inf                                    # none at all
    logits[5, [10, 20]] = torch.tensor([0.0, 200.0], device=dev)     # the first has less than 2^-100 of the second
    logits[6, 77] = 1.0
    logits[7, 77] = 1.0
    top = 1 - 2.0 ** -24
    v = sampling.DraftVerifier(8, 8, 2, dev)
    go = lambda u_draw, starts=range(9), tokens=[0] * 8, u_keep=[0.0] * 8: [t.tolist() for t in v(logits, _i32(tokens, dev), _i32(list(starts), dev), torch.tensor(u_keep, device=dev),
                                                                                                  torch.tensor(u_draw, device=dev), temperature=0.5)]
    first = lambda r: [t[0] for t in r[0]]
    assert first(go([0.0] * 8)) == [5, 999, 0, 0, 0, 20, 77, 77]
    assert first(go([top] * 8)) == [900, 999, 0, 999, 0, 20, 77, 77]
    assert first(go([0.5] * 8)) == [900, 999, 0, 500, 0, 20, 77, 77]         # (the cumulative mass has to exceed the target)
    # rows 6 and 7 as a chain: a certain draft that is kept, whatever the number; one that is impossible
    out, rows, count = go([0.25], [6, 8], [0] * 7 + [77], [0.0] * 7 + [top])
    assert (out, rows, count) == ([[77, 77]], [[0, 1]], [2])
    out, rows, count = go([0.25], [6, 8], [0] * 7 + [78], [0.0] * 8)
    assert (out, rows, count) == ([[77, -1]], [[0, -1]], [1])
    for absurd in (-1, 1000, 2 ** 31 - 1):                 # tokens outside the vocabulary are never kept
        assert go([0.25], [6, 8], [0] * 7 + [absurd], [0.0] * 8)[2] == [1]


def test_nan_and_bad_ranges_stay_inside_the_outputs(dev):
    from georefine_b200 import sampling

    logits = torch.zeros(4, 300, device=dev, dtype=torch.bfloat16)
    logits[0, 7] = float("nan")
    logits[1, 7] = float("inf")
    v = sampling.DraftVerifier(4, 4, 3, dev)
    out, rows, count = v(logits, _i32([0] * 4, dev), _i32([0, 1, 2, 2, 9], dev), torch.zeros(4, device=dev), torch.full((4,), 0.5, device=dev))
    assert count.tolist() == [1, 1, 0, 0] and out[2:].tolist() == [[-1] * 3] * 2 and rows[2:].tolist() == [[-1] * 3] * 2       # no rows; rows that do not exist
    assert 0 <= int(out[0, 0]) < 300 and 0 <= int(out[1, 0]) < 300 and out[:2, 1:].tolist() == [[-1] * 2] * 2
    # parents that are no parents: such nodes are never reached
    out, rows, count = v(logits[2:], _i32([0, 5], dev), _i32([0, 2], dev), torch.zeros(2, device=dev), torch.full((1,), 0.5, device=dev), parent=_i32([-1, 1], dev))
    assert count.tolist() == [1]


def test_a_walk_stops_at_the_outputs_width(dev):
    from georefine_b200 import sampling

    logits = torch.full((6, 64), -30.0, device=dev)
    for i in range(6):
        logits[i, i + 1] = 30.0
    v = sampling.DraftVerifier(6, 1, 3, dev)
    out, rows, count = v(logits, _i32([0, 1, 2, 3, 4, 5], dev), _i32([0, 6], dev), torch.full((6,), 0.3, device=dev), torch.full((1,), 0.3, device=dev))
    assert out.tolist() == [[1, 2, 3]] and rows.tolist() == [[0, 1, 2]] and count.tolist() == [3]      # (3: drawn, its draft not tried)


def test_strides_unaligned_rows_and_fewer_sequences_than_the_verifier_holds(dev):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(8)
    for dtype in (torch.bfloat16, torch.float32):
        wide = _logits(g, 7, 1203, dtype, dev)
        logits = wide[:, 3:1006]                           # rows that start anywhere
        best = logits.float().argmax(1).tolist()
        tokens = [[0, best[0], best[1], 9], [0, best[4], best[5]]]
        u = [[0.2] * 4, [0.1] * 3]
        v = sampling.DraftVerifier(20, 9, 4, dev)
        _compare(v, logits, tokens, [[-1, 0, 1, 2], [-1, 0, 1]], u, [0.4, 0.9], 0.8, chain=True)
        q = torch.rand(7, 1100, generator=g, device=dev)[:, 5:1008]
        _compare(v, logits, tokens, [[-1, 0, 1, 2], [-1, 0, 1]], u, [0.4, 0.9], 0.8, chain=True, q=q)


def test_a_large_vocabulary_flat_and_sharp(dev):
    """Draws next to 152064 and 524288 borders, against running sums in 64 bits."""
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(1)
    for vocab, dtype in ((152064, torch.bfloat16), (524288, torch.float32)):
        for sharp in (0.3, 3.0):
            logits = (sharp * torch.randn(64, vocab, generator=g, device=dev)).to(dtype)
            u = torch.rand(64, generator=g, device=dev)
            v = sampling.DraftVerifier(64, 64, 1, dev)
            out, rows, count = v(logits, _i32([0] * 64, dev), _i32(range(65), dev), torch.zeros(64, device=dev), u, temperature=0.9)
            p = torch.exp((logits.double() - logits.double().amax(1, keepdim=True)) / 0.9)
            run = p.cumsum(1)
            want = (run <= u.double()[:, None] * run[:, -1:]).sum(1)
            assert torch.equal(out[:, 0].long(), want) and bool((count == 1).all()) and bool((rows == 0).all())


def test_the_tokens_are_distributed_as_the_target_s(dev):
    """40000 chains of one certain draft, and 40000 trees of two: the first emitted token's frequencies are the target's
    probabilities, each within five standard deviations."""
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(11)
    n, vocab = 40000, 5
    for children in (1, 2):
        rows = n * (1 + children)
        logits = torch.tensor([0.5, 1.5, -0.2, 0.9, 0.1], device=dev).expand(rows, vocab).contiguous()
        p = torch.softmax(logits[0].double() / 0.8, dim=0)
        tokens = torch.tensor([0, 1, 3][:1 + children], dtype=torch.int32, device=dev).repeat(n)
        parent = _i32([-1, 0, 0][:1 + children], dev).repeat(n)
        v = sampling.DraftVerifier(65535, 30000, 2, dev)
        first = []
        per = 20000
        for lo in range(0, n, per):
            part = slice(lo * (1 + children), (lo + per) * (1 + children))
            out, _, _ = v(logits[part], tokens[part], _i32(list(range(0, per * (1 + children) + 1, 1 + children)), dev), torch.rand(per * (1 + children), generator=g, device=dev),
                          torch.rand(per, generator=g, device=dev), temperature=0.8, parent=parent[part])
            first.append(out[:, 0].clone())
        share = torch.bincount(torch.cat(first).long(), minlength=vocab).double() / n
        assert bool(((share - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all())


def test_captured_and_replayed_and_on_another_stream(dev):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(3)
    logits = _logits(g, 12, 5000, torch.bfloat16, dev)
    tokens, starts = _i32([0, 1, 2] * 4, dev), _i32([0, 3, 6, 9, 12], dev)
    u, d = torch.rand(12, generator=g, device=dev), torch.rand(4, generator=g, device=dev)
    v, plain = (sampling.DraftVerifier(12, 4, 3, dev) for _ in range(2))
    v(logits, tokens, starts, u, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = v(logits, tokens, starts, u, d)
    for _ in range(3):
        logits.copy_(_logits(g, 12, 5000, torch.bfloat16, dev))
        u.copy_(torch.rand(12, generator=g, device=dev)); d.copy_(torch.rand(4, generator=g, device=dev))
        tokens.copy_(logits.argmax(1).int().roll(1))
        graph.replay()
        for a, b in zip(got, plain(logits, tokens, starts, u, d)):
            assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = plain(logits, tokens, starts, u, d)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, again))
