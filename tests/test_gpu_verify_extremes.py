"""Verification of drafts where logits or temperatures are extreme: masks of the type's lowest value, logits far from zero, temperatures
near zero (needs a B200).  Expected tokens come from a walk in plain Python with 64-bit numbers, or from the arg-max."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_verify_drafts import _compare, _i32, _logits  # noqa: E402


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _chains(logits, lengths, every=3):
    """Tokens of chains whose drafts are mostly the arg-max."""
    best, tokens, at = logits.float().argmax(1).tolist(), [], 0
    for n in lengths:
        tokens.append([0] + [best[at + j] if (at + j) % every else 1 for j in range(n - 1)])
        at += n
    return tokens, [list(range(-1, n - 1)) for n in lengths]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low", [-1e9, -1e10, -1e30, None])
@pytest.mark.parametrize("vocab,share", [(300, 0.1), (20011, 0.3), (152064, 0.0001)])
def test_masked_tokens(dev, dtype, low, vocab, share):
    """Tokens that a mask leaves out, at a large negative number or the type's lowest: as if they were -infinity."""
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(vocab)
    lengths = [1, 4, 2, 3]
    rows = sum(lengths)
    logits = _logits(g, rows, vocab, dtype, dev, 3.0)
    allowed = torch.rand(rows, vocab, generator=g, device=dev) < share
    allowed[:, [5, vocab // 2, vocab - 2]] = True
    logits = logits.masked_fill(~allowed, torch.finfo(dtype).min if low is None else low)
    tokens, parents = _chains(logits, lengths)
    v = sampling.DraftVerifier(rows, 4, 5, dev)
    for temperature in (1.0, 0.01):
        u = [torch.rand(n, generator=g, device=dev).tolist() for n in lengths]
        out, count = _compare(v, logits, tokens, parents, u, torch.rand(4, generator=g, device=dev).tolist(), temperature, chain=True)
        for s, n in enumerate(count):          # the drawn token is an allowed one
            row = sum(lengths[:s]) + n - 1
            assert bool(allowed[row, out[s][n - 1]])


def test_masked_tokens_with_the_drafter_s_probabilities(dev):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(2)
    lengths, vocab = [3, 5, 2], 4101
    rows = sum(lengths)
    logits = _logits(g, rows, vocab, torch.float32, dev, 3.0)
    allowed = torch.rand(rows, vocab, generator=g, device=dev) < 0.05
    allowed[:, 7] = True
    logits = logits.masked_fill(~allowed, torch.finfo(torch.float32).min)
    q, tokens, at = torch.zeros(rows, vocab, device=dev), [], 0
    for n in lengths:
        q[at + 1:at + n] = torch.softmax(logits[at:at + n - 1] + 0.8 * torch.randn(n - 1, vocab, generator=g, device=dev), dim=1)
        tokens.append([0] + torch.multinomial(q[at + 1:at + n], 1, generator=g)[:, 0].tolist())
        at += n
    v = sampling.DraftVerifier(rows, 3, 5, dev)
    for _ in range(3):
        u = [torch.rand(n, generator=g, device=dev).tolist() for n in lengths]
        _compare(v, logits, tokens, [list(range(-1, n - 1)) for n in lengths], u, torch.rand(3, generator=g, device=dev).tolist(), 1.0, chain=True, q=q)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [9.0, 12.5, -7.3, 1e5, -3e20])
@pytest.mark.parametrize("temperature", [1e-4, 1e-6, 1e-8, 1e-9, 1e-10, 1e-20, 1e-30])
def test_temperatures_near_zero_are_the_arg_max(dev, dtype, top, temperature):
    from georefine_b200 import sampling

    g = torch.Generator(device=dev).manual_seed(4)
    vocab = 3001
    logits = (top + abs(top) * (0.01 * torch.rand(6, vocab, generator=g, device=dev) - 0.06)).to(dtype)
    best = torch.randint(vocab, (6,), generator=g, device=dev)
    logits.scatter_(1, best[:, None], top)
    best = best.tolist()
    v = sampling.DraftVerifier(6, 3, 3, dev)
    # a right draft, a wrong one, a tree whose second child is right
    tokens = _i32([0, best[0], 0, (best[2] + 1) % vocab, 0, best[4]], dev)
    for u in (0.0, 0.5, 1 - 2.0 ** -24):
        out, rows, count = v(logits, tokens, _i32([0, 2, 4, 6], dev), torch.full((6,), max(u, 2.0 ** -24), device=dev), torch.full((3,), u, device=dev), temperature=temperature)
        assert out.tolist() == [[best[0], best[1], -1], [best[2], -1, -1], [best[4], best[5], -1]] and count.tolist() == [2, 1, 2], u
    out, rows, count = v(logits[:3], _i32([0, (best[0] + 1) % vocab, best[0]], dev), _i32([0, 3], dev), torch.full((3,), 0.5, device=dev), torch.full((1,), 0.5, device=dev),
                         temperature=temperature, parent=_i32([-1, 0, 0], dev))
    assert out.tolist() == [[best[0], best[2], -1]] and rows.tolist() == [[0, 2, -1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_all_alike_far_from_zero(dev, dtype):
    """Every token as likely as every other, at any size of the logits: the draw is u times the vocabulary, rounded down."""
    from georefine_b200 import sampling

    vocab, sizes = 5003, [0.0, 1e4, -1e9, 3e15, -2e30, torch.finfo(dtype).max, torch.finfo(dtype).min]
    logits = torch.tensor(sizes, dtype=torch.float64, device=dev).to(dtype)[:, None].expand(-1, vocab).contiguous()
    v = sampling.DraftVerifier(len(sizes), len(sizes), 1, dev)
    for u in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
        for temperature in (0.7, 1.0, 30.0):
            out, _, _ = v(logits, _i32([0] * len(sizes), dev), _i32(range(len(sizes) + 1), dev), torch.zeros(len(sizes), device=dev),
                          torch.full((len(sizes),), u, device=dev), temperature=temperature)
            assert out[:, 0].tolist() == [int(float(torch.tensor(u)) * vocab)] * len(sizes), (u, temperature)
    # two tokens far above the others, whose distances no 32-bit exponent holds
    logits[:, [40, 4000]] = torch.tensor([3.0, 1e5, 5e9, 3e16, 1e31, torch.finfo(dtype).max, 1e38], dtype=torch.float64, device=dev).to(dtype)[:, None]
    for u, want in ((0.1, 40), (0.9, 4000)):
        out, _, _ = v(logits[1:], _i32([0] * 6, dev), _i32(range(7), dev), torch.zeros(6, device=dev), torch.full((6,), u, device=dev), temperature=1.0)
        assert out[:, 0].tolist() == [want if i != 4 else int(float(torch.tensor(u)) * vocab) for i in range(6)], u


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_minus_infinity_is_below_the_lowest_value(dev, dtype):
    """Tokens at the type's lowest value in a row of -infinity otherwise, at the highest temperature too: only they are drawn."""
    from georefine_b200 import sampling

    vocab, held = 1003, [3, 500, 1002]
    logits = torch.full((1, vocab), -float("inf"), device=dev, dtype=dtype)
    logits[:, held] = torch.finfo(dtype).min
    v = sampling.DraftVerifier(1, 1, 1, dev)
    for temperature in (1e-30, 1.0, 1e20):
        got = [int(v(logits, _i32([0], dev), _i32([0, 1], dev), torch.zeros(1, device=dev), torch.full((1,), u, device=dev), temperature=temperature)[0][0, 0])
               for u in (0.0, 0.32, 0.34, 0.66, 0.67, 1 - 2.0 ** -24)]
        assert got == [3, 3, 500, 500, 1002, 1002]
