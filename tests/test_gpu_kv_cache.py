"""Storing rows in a paged cache, reading them back, and moving what a draft tree keeps (needs a B200).

All of it is exact: codes, exponents and values have to equal the definition, evaluated in 64 bits."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from spec_reference import entry  # noqa: E402

BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _pages(ops, n, nkv, dev, fmt, fill=0x7F, layers=None):
    """Pages holding what memory nobody wrote may hold: NaN everywhere."""
    p = ops.KVPages.alloc(n, nkv, dev, kv_format=fmt, layers=layers)
    for t in (p.k, p.v):
        t.view(torch.uint8).fill_(fill if fmt == "e4m3" else 0xFF)
    for t in (p.k_exp, p.v_exp):
        if t is not None:
            t.fill_(0)
    return p


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("nkv,tokens", [(1, 1), (2, 37), (3, 255), (8, 513)])
def test_write_and_read(dev, fmt, nkv, tokens):
    from georefine_b200 import ops

    g = torch.Generator(device=dev).manual_seed(nkv * 1000 + tokens)
    slots, per = 3, -(-tokens // 256)
    table = torch.randperm(slots * per + 2, generator=g, device=dev)[:slots * per].reshape(slots, per).int()
    pages = _pages(ops, slots * per + 2, nkv, dev, fmt)
    before = [t.clone() for t in (pages.k.view(torch.uint8), pages.v.view(torch.uint8))]
    rows = slots * tokens
    seq, pos = torch.arange(slots, device=dev).repeat_interleave(tokens).int(), torch.arange(tokens, device=dev).repeat(slots).int()
    order = torch.randperm(rows, generator=g, device=dev)
    seq, pos = seq[order].contiguous(), pos[order].contiguous()
    wide = torch.randn(rows, 2 * nkv * 128 + 64, generator=g, device=dev) * torch.exp(3 * torch.randn(rows, 1, generator=g, device=dev))
    wide = wide.to(BF)                                         # rows of a wider matrix, as of a step's qkv
    k, v = (wide[:, i * nkv * 128:(i + 1) * nkv * 128].unflatten(1, (nkv, 128)) for i in range(2))
    ops.kv_write(k, v, seq, pos, table, pages)
    k_out, v_out = (torch.zeros(rows, nkv, 128, device=dev, dtype=BF) for _ in range(2))
    ops.kv_read(seq, pos, table, pages, k_out, v_out)
    page, at = table[seq.long(), (pos // 256).long()].long(), (pos % 256).long()
    for x, out, held, exps, old in ((k, k_out, pages.k, pages.k_exp, before[0]), (v, v_out, pages.v, pages.v_exp, before[1])):
        if fmt == "e4m3":
            code, byte, value = entry(x)
            assert torch.equal(held.view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn).double(), code)
            assert torch.equal(exps[page, :, at], byte) and torch.equal(out.double(), value)
        else:
            assert torch.equal(held[page, :, at], x) and torch.equal(out, x)
        held = held.view(torch.uint8).clone()
        written = torch.zeros(held.shape[:3], dtype=torch.bool, device=dev)
        written[page, :, at] = True
        assert torch.equal(held[~written], old[~written])      # nothing else was touched


def test_entries_at_the_ends_of_the_format(dev):
    from georefine_b200 import ops

    top = torch.finfo(BF).max
    rows = torch.zeros(16, 1, 128)
    rows[0] = 0.0                                              # zeros: the smallest exponent
    rows[1, 0, 5] = 448.0                                      # exactly the largest code at e = 0
    rows[2, 0, 5] = 450.0                                      # just above: e = 1
    rows[3, 0, 7] = 57344.0                                    # the largest value held
    rows[4, 0, 7] = 60000.0                                    # above it: held as 57344
    rows[5, 0, 7] = -top
    rows[6, 0, 0], rows[6, 0, 1] = 2.0 ** -60, -2.0 ** -60     # below the smallest exponent: zero
    rows[7, 0, 0], rows[7, 0, 1] = 448 * 2.0 ** -40, 2.0 ** -49
    rows[8, 0, 3] = float("inf")
    rows[9, 0, 3] = float("nan")
    rows[9, 0, 4] = 1.0
    rows[10, 0, 127] = -float("inf")
    rows[11] = torch.linspace(-1, 1, 128)
    rows[12, 0] = torch.tensor([(1 + m / 16) * 2.0 ** (i % 5) for i, m in enumerate(list(range(16)) * 8)])   # ties between codes
    rows[13, 0, 0], rows[13, 0, 1] = 448.0, 448 * 2.0 ** -18   # below half of the smallest code
    rows[14, 0, 0], rows[14, 0, 1:4] = 448.0, torch.tensor([2.0 ** -9, 1.5 * 2.0 ** -9, 2.0 ** -10])         # the smallest codes, and a tie to zero
    rows[15, 0, 0] = 2.0 ** -126
    rows = rows.to(BF).to(dev)
    pages = ops.KVPages.alloc(1, 1, dev, kv_format="e4m3")
    seq, pos, table = _i32([0] * 16, dev), _i32(range(16), dev), _i32([[0]], dev)
    ops.kv_write(rows, rows, seq, pos, table, pages)
    out = [torch.empty_like(rows) for _ in range(2)]
    ops.kv_read(seq, pos, table, pages, *out)
    code, byte, value = entry(rows)
    assert torch.equal(pages.k.view(torch.uint8)[0, 0, :16].view(torch.float8_e4m3fn).double(), code[:, 0])
    assert torch.equal(pages.v_exp[0, 0, :16], byte[:, 0])
    for o in out:
        assert torch.equal(torch.nan_to_num(o.double(), nan=-7.0), torch.nan_to_num(value, nan=-7.0))
    assert bool(out[0][8:11].isnan().all()) and float(out[0][4].max()) == 57344.0 and float(out[0][6].abs().max()) == 0.0
    finite = torch.isfinite(rows.float()).all(-1) & (rows.float().abs().amax(-1) <= 57344)
    assert bool(((out[0].double() - rows.double()).abs() <= torch.maximum(2.0 ** -4 * rows.double().abs(), 2.0 ** -10 * torch.exp2(byte.double() - 127)[..., None]))[finite].all())


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_rows_that_are_left_out(dev, fmt):
    from georefine_b200 import ops

    pages = _pages(ops, 3, 2, dev, fmt)
    before = pages.k.view(torch.uint8).clone()
    table = _i32([[0, 1], [2, 7], [-1, 1]], dev)               # page 7 and page -1 are outside the pool
    seq, pos = _i32([-1, 3, 0, 0, 1, 2], dev), _i32([0, 0, 512, -1, 300, 5], dev)
    x = torch.ones(6, 2, 128, device=dev, dtype=BF)
    ops.kv_write(x, x, seq, pos, table, pages)
    assert torch.equal(pages.k.view(torch.uint8), before)
    out = torch.full((6, 2, 128), 3.0, device=dev, dtype=BF)
    ops.kv_read(seq, pos, table, pages, out, out.clone())
    assert bool((out == 3.0).all())
    none = torch.empty(0, 2, 128, device=dev, dtype=BF)
    ops.kv_write(none, none, seq[:0], pos[:0], table, pages)   # no rows at all
    assert torch.equal(pages.k.view(torch.uint8), before)


def test_a_pool_beyond_32_bits_of_offsets(dev):
    from georefine_b200 import ops

    n, nkv = 16500, 8                                          # 4.3 GB of codes for the keys alone
    pages = ops.KVPages.alloc(n, nkv, dev, kv_format="e4m3")
    table = _i32([[0, n - 1]], dev)
    seq, pos = _i32([0, 0], dev), _i32([3, 256 + 255], dev)
    g = torch.Generator(device=dev).manual_seed(5)
    k, v = (torch.randn(2, nkv, 128, generator=g, device=dev).to(BF) for _ in range(2))
    ops.kv_write(k, v, seq, pos, table, pages)
    out = [torch.empty_like(k) for _ in range(2)]
    ops.kv_read(seq, pos, table, pages, *out)
    assert torch.equal(out[0].double(), entry(k)[2]) and torch.equal(out[1].double(), entry(v)[2])
    assert torch.equal(pages.v.view(torch.uint8)[n - 1, :, 255].view(torch.float8_e4m3fn).double(), entry(v)[0][1])
    assert int(pages.k.view(torch.uint8)[1:n - 1].any()) == 0
    # the last entry of the pool moved to the first position behind a root at 0, across the whole pool
    ops.kv_keep(_i32([0], dev), _i32([3], dev), _i32([[0, 508]], dev), _i32([2], dev), table, pages)
    ops.kv_read(_i32([0], dev), _i32([4], dev), table, pages, out[0][:1], out[1][:1])
    assert torch.equal(out[0][0].double(), entry(k)[2][1])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("layers,nkv", [(1, 1), (3, 8), (2, 70)])
def test_keep(dev, fmt, layers, nkv):
    from georefine_b200 import ops

    g = torch.Generator(device=dev).manual_seed(layers)
    slots, per = 5, 3
    both = torch.randint(0, 120, (layers, 2, slots * per, nkv, 256, 128 * (2 if fmt == "bf16" else 1)), generator=g, device=dev, dtype=torch.uint8)
    held = both.view(BF if fmt == "bf16" else torch.float8_e4m3fn)
    exps = torch.randint(90, 130, (layers, 2, slots * per, nkv, 256), generator=g, device=dev, dtype=torch.uint8)
    pages = ops.KVPages(held[:, 0], held[:, 1], *((exps[:, 0], exps[:, 1]) if fmt == "e4m3" else ()))     # layers of a wider stack
    table = torch.randperm(slots * per, generator=g, device=dev).reshape(slots, per).int()
    base = [0, 250, 255, 640, 100]
    path = [[0, 1, 2, 3, -1, -1], [0, 2, 3, 9, 10, 11], [0, 5, -1, -1, -1, -1], [0, 7, 30, 60, 64, 127], [0, 3, 4, 5, 6, 7]]
    count = [4, 6, 2, 6, 9]                                    # (the last: more than there are columns)
    order = [3, 1, 0, -1, 2]                                   # slots; the fourth sequence is left out
    want = [t.clone() for t in (both, exps)]
    for i, slot in enumerate(order):
        if slot < 0:
            continue
        for x in want:
            old = x.clone()
            for j in range(1, min(count[i], 6)):
                s, d = base[i] + path[i][j], base[i] + j
                if s >= per * 256:
                    continue
                x[:, :, int(table[slot, d // 256]), :, d % 256] = old[:, :, int(table[slot, s // 256]), :, s % 256]
    ops.kv_keep(_i32(order, dev), _i32(base, dev), _i32(path, dev), _i32(count, dev), table, pages)
    assert torch.equal(both, want[0])
    assert fmt == "bf16" or torch.equal(exps, want[1])
    ops.kv_keep(_i32(order, dev), _i32(base, dev), _i32(path, dev), _i32([0, 1, -3, 1, 1], dev), table, pages)     # nothing behind the roots
    ops.kv_keep(_i32(order, dev), _i32(base, dev), _i32(path, dev)[:, :1], _i32(count, dev), table, pages)
    assert torch.equal(both, want[0])


def test_a_long_path_moves_in_order(dev):
    """200 entries from odd places to consecutive ones: more than a batch, each target the source of a later move."""
    from georefine_b200 import ops

    pages = ops.KVPages.alloc(3, 8, dev, kv_format="bf16")
    pages.k.copy_(torch.arange(3 * 256, device=dev).view(3, 1, 256, 1).expand_as(pages.k))
    pages.v.copy_(-pages.k)
    path = [0] + [2 * j + 1 for j in range(1, 200)]
    ops.kv_keep(_i32([0], dev), _i32([20], dev), _i32([path], dev), _i32([200], dev), _i32([[0, 1, 2]], dev), pages)
    got = pages.k[:, 3].reshape(-1, 128)[20:220, 64].tolist()
    want = torch.tensor([20.0 + p for p in path]).to(BF).float().tolist()
    assert got == want and pages.v[:, 7].reshape(-1, 128)[20:220, 0].tolist() == [-x for x in want]


def test_refusals(dev):
    from georefine_b200 import ops

    pages = ops.KVPages.alloc(2, 2, dev, kv_format="e4m3", layers=2)
    one = pages.layer(1)
    table, seq = _i32([[0, 1]], dev), _i32([0], dev)
    x = torch.zeros(1, 2, 128, device=dev, dtype=BF)
    for bad in (lambda: ops.kv_write(x, x, seq, seq, table, pages), lambda: ops.kv_write(x.float(), x, seq, seq, table, one), lambda: ops.kv_write(x[:, :1], x, seq, seq, table, one),
                lambda: ops.kv_write(x, x, seq.long(), seq, table, one), lambda: ops.kv_write(x, x, seq, _i32([0, 1], dev), table, one), lambda: ops.kv_write(x, x.cpu(), seq, seq, table, one),
                lambda: ops.kv_write(x, x, seq, seq, table.long(), one), lambda: ops.kv_write(x, x, seq, seq, table[0], one),
                lambda: ops.kv_read(seq, seq, table, one, torch.zeros(1, 128, 2, device=dev, dtype=BF).transpose(1, 2), x),
                lambda: ops.KVPages(one.k, one.v), lambda: ops.KVPages(one.k, one.v, one.k_exp, one.v_exp[:1]), lambda: ops.KVPages(one.k.view(torch.uint8), one.v.view(torch.uint8)),
                lambda: ops.KVPages(one.k[:, :1], one.v[:, :1], one.k_exp[:, :1], one.v_exp[:, :1]), lambda: ops.KVPages(pages.k, pages.v[:1], pages.k_exp, pages.v_exp),
                lambda: ops.kv_keep(seq, seq, _i32([0, 1], dev), seq, table, pages), lambda: ops.kv_keep(seq, seq, _i32([[0, 1]], dev).long(), seq, table, pages),
                lambda: ops.kv_keep(seq, _i32([0, 0], dev), _i32([[0, 1]], dev), seq, table, pages)):
        with pytest.raises(ValueError):
            bad()


def test_calls_in_a_graph_and_on_another_stream(dev):
    from georefine_b200 import ops

    pages, table = ops.KVPages.alloc(2, 2, dev, kv_format="e4m3"), _i32([[1, 0]], dev)
    seq, pos = _i32([0] * 40, dev), _i32(range(230, 270), dev)
    k, v = (torch.zeros(40, 2, 128, device=dev, dtype=BF) for _ in range(2))
    out = [torch.empty_like(k) for _ in range(2)]

    def both():
        ops.kv_write(k, v, seq, pos, table, pages)
        ops.kv_read(seq, pos, table, pages, *out)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    g = torch.Generator(device=dev).manual_seed(2)
    for _ in range(2):
        k.copy_(torch.randn(k.shape, generator=g, device=dev)); v.copy_(torch.randn(k.shape, generator=g, device=dev))
        graph.replay()
        assert torch.equal(out[0].double(), entry(k)[2]) and torch.equal(out[1].double(), entry(v)[2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        k.mul_(3)
        both()
    side.synchronize()
    assert torch.equal(out[0].double(), entry(k)[2])
