"""Attention of causal rows and draft trees over a BF16 or an 8-bit cache, against its definition in 64 bits (needs a B200)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from spec_reference import attend, entry, rotate  # noqa: E402

BF = torch.bfloat16
POISON = {"bf16": 0xFF, "e4m3": 0x7F}          # NaN, as memory that nobody wrote may hold


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Setup:
    """Sequences with cached positions in scattered pages, and the rows of one call."""

    def __init__(self, dev, fmt, nq, nkv, lengths, per_slot, seed=0, scale=1.0):
        from georefine_b200 import ops

        self.dev, self.fmt, self.nq, self.nkv, self.ops = dev, fmt, nq, nkv, ops
        self.g = torch.Generator(device=dev).manual_seed(1000 * nq + nkv + seed)
        slots = len(lengths)
        self.table = torch.randperm(slots * per_slot, generator=self.g, device=dev).reshape(slots, per_slot).int()
        self.pages = ops.KVPages.alloc(slots * per_slot, nkv, dev, kv_format=fmt)
        for t in (self.pages.k, self.pages.v):
            t.view(torch.uint8).fill_(POISON[fmt])
        self.cos, self.sin = ops.rope_tables(per_slot * 256, device=dev)
        self.lengths = list(lengths)
        for slot, n in enumerate(lengths):
            if n:
                k, v = (scale * torch.randn(n, nkv, 128, generator=self.g, device=dev) * torch.exp(0.7 * torch.randn(n, 1, 1, generator=self.g, device=dev)) for _ in range(2))
                ops.kv_write(k.to(BF), v.to(BF), _i32([slot] * n, dev), _i32(range(n), dev), self.table, self.pages)

    def qkv(self, rows, q_scale=1.5):
        x = torch.randn(rows, (self.nq + 2 * self.nkv) * 128, generator=self.g, device=self.dev)
        x[:, :self.nq * 128] *= q_scale
        return x.to(BF)

    def held(self, slot, n):
        """Keys and values of positions 0 .. n - 1 as the cache holds them."""
        k, v = (torch.full((n, self.nkv, 128), 7.0, device=self.dev, dtype=BF) for _ in range(2))
        self.ops.kv_read(_i32([slot] * n, self.dev), _i32(range(n), self.dev), self.table, self.pages, k, v)
        return k.double(), v.double()

    def check(self, qkv, seq, pos, out, seen, rope=None):
        """Every row against the definition over what the cache holds after the call; ``seen(row, positions)`` -> bool tensor."""
        half = {"bf16": 2.0 ** -16, "e4m3": 2.0 ** -11}[self.fmt]     # (BF16: rounded twice, the second time what the first left out)
        for r, (s, p) in enumerate(zip(seq, pos)):
            if s < 0:
                continue
            turn = p if rope is None else rope[r]
            x = qkv[r].view(-1, 128)
            q = rotate(x[:self.nq], self.cos[turn], self.sin[turn])
            k_new, v_new = rotate(x[self.nq:self.nq + self.nkv], self.cos[turn], self.sin[turn]), x[self.nq + self.nkv:].double()
            n = self.table.shape[1] * 256
            k, v = self.held(s, n)
            if self.fmt == "e4m3":
                # (the rotation is rounded once to 32 bits before the code is chosen)
                assert bool(((k[p] - entry(k_new.float())[2]).abs() <= 2.0 ** -23 * k_new.abs()).all()) and torch.equal(v[p], entry(v_new)[2])
            else:
                assert bool(((k[p] - k_new).abs() <= 4 * 2.0 ** -8 * k_new.abs().amax()).all()) and torch.equal(v[p], v_new)
            want, bound = attend(q, k, v, seen(r, torch.arange(n, device=self.dev)), half, half)
            got = out[r].view(self.nq, 128).double()
            assert bool(((got - want).abs() <= bound).all()), (r, float(((got - want).abs() / bound).max()))


def _causal(pos):
    return lambda r, p: p <= pos[r]


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(5, 1), (4, 4), (6, 2), (16, 1), (14, 2), (8, 1), (10, 2)])
def test_causal_rows(dev, fmt, nq, nkv):
    """Decode rows, chains of rows and prompt chunks together; lengths at the borders of pages and parts."""
    lengths = [0, 1, 127, 128, 255, 256, 511, 600]
    s = Setup(dev, fmt, nq, nkv, lengths, 4)
    per = [3, 1, 2, 1, 1, 4, 2, 21]
    seq = [i for i, n in enumerate(per) for _ in range(n)]
    pos = [lengths[i] + j for i, n in enumerate(per) for j in range(n)]
    qkv = s.qkv(len(seq))
    out = torch.full((len(seq), nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(nq, nkv, len(seq), 4, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out)
    s.check(qkv, seq, pos, out, _causal(pos))
    # a row alone, and the rows in another order, give the same bits
    solo = torch.empty(1, nq * 128, device=dev, dtype=BF)
    for r in (0, 5, len(seq) - 1):
        attn(qkv[r:r + 1], s.cos, s.sin, _i32(seq[r:r + 1], dev), _i32(pos[r:r + 1], dev), s.table, s.pages, solo)
        assert torch.equal(solo[0], out[r])
    back = list(range(len(seq)))[::-1]
    again = torch.empty_like(out)
    attn(qkv[back].contiguous(), s.cos, s.sin, _i32([seq[i] for i in back], dev), _i32([pos[i] for i in back], dev), s.table, s.pages, again)
    assert torch.equal(again[back], out)


def test_steps_and_a_chain_give_the_same_bits(dev):
    """Tokens decoded one by one over an 8-bit cache, and the same tokens as rows of one verify pass."""
    bits = []
    for chain in (False, True):
        s = Setup(dev, "e4m3", 10, 2, [300], 2, seed=3)
        qkv = s.qkv(9)
        attn = s.ops.TreeAttention(10, 2, 9, 2, dev, kv_format="e4m3")
        out = torch.empty(9, 1280, device=dev, dtype=BF)
        for rows in ([slice(0, 9)] if chain else [slice(i, i + 1) for i in range(9)]):
            pos = list(range(300, 309))[rows]
            attn(qkv[rows], s.cos, s.sin, _i32([0] * len(pos), dev), _i32(pos, dev), s.table, s.pages, out[rows])
        bits.append(out.clone())
    assert torch.equal(*bits)


TREES = {"one": [-1], "pair": [-1, 0], "star": [-1] + [0] * 9, "chain": list(range(-1, 15)), "bushy": [-1, 0, 0, 0, 1, 1, 2, 4, 4, 7, 3, 10, 11, 5],
         "wide": [-1] + [i // 3 for i in range(63)], "words": [-1] + [(i * 7) // 11 for i in range(129)]}


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(5, 1), (8, 2), (6, 1), (16, 1)])
def test_trees(dev, fmt, nq, nkv):
    """Trees of 1 to 130 nodes behind contexts of no position, some, and pages full, in one call."""
    lengths = [0, 300, 1, 256, 250, 700, 505]
    s = Setup(dev, fmt, nq, nkv, lengths, 4)
    seq, pos, base, rope, mask = [], [], [], [], []
    for slot, parents in enumerate(TREES.values()):
        depth, masks = s.ops.TreeRows.masks(parents, words=3)
        n = len(parents)
        seq += [slot] * n
        pos += [lengths[slot] + i for i in range(n)]
        base += [lengths[slot]] * n
        rope += [lengths[slot] + d for d in depth]
        mask += masks
    rows = len(seq)
    qkv = s.qkv(rows)
    out = torch.full((rows, nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(nq, nkv, rows, 4, dev, kv_format=fmt)
    tree = s.ops.TreeRows(_i32(base, dev), _i32(rope, dev), torch.tensor(mask, dtype=torch.int64, device=dev))
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, tree=tree)

    def seen(r, p):
        node = p - base[r]
        bits = torch.tensor([mask[r][w] >> b & 1 for w in range(3) for b in range(64)], device=dev).bool()
        return (node < 0) | ((node >= 0) & (node < 192) & bits[node.clamp(0, 191)])

    s.check(qkv, seq, pos, out, seen, rope)
    # a sequence's rows alone give the same bits
    at = seq.index(5)
    n = seq.count(5)
    rows5 = slice(at, at + n)
    alone = torch.empty(n, nq * 128, device=dev, dtype=BF)
    attn(qkv[rows5], s.cos, s.sin, _i32(seq[rows5], dev), _i32(pos[rows5], dev), s.table, s.pages, alone,
         tree=s.ops.TreeRows(tree.base[rows5], tree.rope[rows5], tree.mask[rows5]))
    assert torch.equal(alone, out[rows5])


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("n", [8, 20])
def test_a_chain_as_a_tree_is_a_causal_chain(dev, fmt, n):
    """Eight rows of four heads a group run in the same kernel either way and give the same bits; a tree of more goes through the
    wide one, and agrees with the definition as the chain does."""
    s = Setup(dev, fmt, 8, 2, [400], 2)
    qkv = s.qkv(n)
    out = [torch.empty(n, 1024, device=dev, dtype=BF) for _ in range(2)]
    attn = s.ops.TreeAttention(8, 2, n, 2, dev, kv_format=fmt)
    positions = list(range(400, 400 + n))
    pos, seq = _i32(positions, dev), _i32([0] * n, dev)
    attn(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, out[0])
    depth, masks = s.ops.TreeRows.masks(list(range(-1, n - 1)))
    tree = s.ops.TreeRows(_i32([400] * n, dev), _i32([400 + d for d in depth], dev), torch.tensor(masks, device=dev))
    attn(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, out[1], tree=tree)
    assert attn.check_status() == 0
    if n == 8:
        assert torch.equal(*out)
    for o in out:
        s.check(qkv, [0] * n, positions, o, _causal(positions))


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_rows_that_see_nothing_and_rows_left_out(dev, fmt):
    s = Setup(dev, fmt, 8, 2, [0, 300, 20], 2)
    seq, pos = [0, 0, -1, 1, 1, 2, 1], [0, 1, 5, 300, 310, 999, 301]         # (position 999 lies outside the table)
    base, rope, mask = [0, 0, 0, 300, 0, 20, 300], [0, 1, 5, 300, 310, 22, 700], [[0], [2], [1], [1], [0], [1], [2]]     # (row 6: outside the rotary tables)
    qkv = s.qkv(7)
    out = torch.full((7, 1024), 5.0, device=dev, dtype=BF)
    before = s.pages.k.view(torch.uint8).clone()
    attn = s.ops.TreeAttention(8, 2, 7, 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, tree=s.ops.TreeRows(_i32(base, dev), _i32(rope, dev), torch.tensor(mask, device=dev)))
    assert bool((out[[2, 5, 6]] == 5.0).all())                              # left out: as they were
    assert bool((out[[0, 4]] == 0.0).all())                                 # an empty mask and no base: zeros
    node = lambda r, p: (p < base[r]) | ((p - base[r] >= 0) & (p - base[r] < 64) & ((mask[r][0] >> (p - base[r]).clamp(0, 63)) & 1).bool())
    s.check(qkv, [0, 0, -1, 1, 1, -1, -1], pos, out, node, rope)
    touched = (s.pages.k.view(torch.uint8) != before).flatten(3).any(-1).any(1)
    assert int(touched.sum()) == 4
    attn(qkv[:0], s.cos, s.sin, _i32([], dev), _i32([], dev), s.table, s.pages, out[:0])          # no rows at all


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_nan_and_infinity_stay_with_the_rows_that_see_them(dev, fmt):
    s = Setup(dev, fmt, 8, 2, [260, 260], 2)
    parents = [-1, 0, 0, 2]
    depth, masks = s.ops.TreeRows.masks(parents)
    n, half = 8, 4
    qkv = s.qkv(n)
    qkv[1, 8 * 128 + 5] = float("nan")                                      # node 1's key
    qkv[5, 10 * 128 + 5] = float("inf")                                     # the other sequence's node 1: a value, kv head 0
    seq, pos = [0] * 4 + [1] * 4, [260 + i for i in range(4)] * 2
    tree = s.ops.TreeRows(_i32([260] * 8, dev), _i32([260 + d for d in depth] * 2, dev), torch.tensor(masks * 2, device=dev))
    out = torch.empty(n, 1024, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, n, 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, tree=tree)
    bad = (~torch.isfinite(out.float())).view(n, 2, 4, 128).any(-1).any(-1).tolist()             # by row and kv head
    assert bad == [[r in (1, 5), False] for r in range(n)]
    # a query that is not finite: its head alone
    qkv = s.qkv(n)
    qkv[2, 3 * 128 + 7] = float("inf")
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, tree=tree)
    bad = (~torch.isfinite(out.float())).view(n, 8, 128).any(-1)
    assert bool(bad[2, 3]) and int(bad.sum()) == 1
    # the cached context: every row sees it
    if fmt == "e4m3":
        s.pages.v_exp.view(-1, 2, 256)[int(s.table[0, 0]), 1, 17] = 255
        s.pages.v.view(torch.uint8)[int(s.table[0, 0]), 1, 17] = 0
    else:
        s.pages.v[int(s.table[0, 0]), 1, 17] = float("nan")
    qkv = s.qkv(n)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, tree=tree)
    bad = out.float().isnan().view(n, 2, 4 * 128).any(-1).tolist()
    assert bad == [[False, r < 4] for r in range(n)]


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_holes_between_a_tree_s_nodes_may_hold_anything(dev, fmt):
    """Only nodes 0, 5 and 40 were ever stored: the others' places hold NaN, and no row sees them."""
    s = Setup(dev, fmt, 10, 2, [250], 2)
    nodes = [0, 5, 40]
    masks = [[1], [1 | 1 << 5], [1 | 1 << 40]]
    pos, rope = [250 + i for i in nodes], [250, 251, 251]
    qkv = s.qkv(3)
    out = torch.empty(3, 1280, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(10, 2, 3, 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32([0] * 3, dev), _i32(pos, dev), s.table, s.pages, out, tree=s.ops.TreeRows(_i32([250] * 3, dev), _i32(rope, dev), torch.tensor(masks, device=dev)))
    s.check(qkv, [0] * 3, pos, out, lambda r, p: (p < 250) | ((p >= 250) & ((masks[r][0] >> (p - 250).clamp(0, 63)) & 1).bool() & (p < 314)), rope)


@pytest.mark.parametrize("scale", [1e-7, 1e3, 0.0])
def test_sizes_of_values(dev, scale):
    """Values (and keys) whose sizes differ by many powers of two between positions, all tiny, all large, all zero."""
    s = Setup(dev, "e4m3", 8, 2, [520], 3, scale=scale)
    qkv = s.qkv(2, q_scale=1.0 if scale < 1 else 1e-2)
    qkv[:, 8 * 128:] *= scale
    qkv[1, 10 * 128:] *= 2.0 ** -12
    out = torch.empty(2, 1024, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, 2, 3, dev, kv_format="e4m3")
    attn(qkv, s.cos, s.sin, _i32([0, 0], dev), _i32([520, 521], dev), s.table, s.pages, out)
    # FP16 weights below their normal range: 2^-25 of the largest product, of which there are 522
    half = 2.0 ** -11
    for r, p in enumerate((520, 521)):
        k, v = s.held(0, 768)
        q = rotate(qkv[r].view(-1, 128)[:8], s.cos[p], s.sin[p])
        want, bound = attend(q, k, v, torch.arange(768, device=dev) <= p, half, half)
        extra = 522 * 2.0 ** -24 * v[:p + 1].abs().amax()
        assert bool(((out[r].view(8, 128).double() - want).abs() <= bound + extra).all())


def test_sharp_and_flat_scores(dev):
    """Scores of hundreds (one position takes all), and all alike."""
    for q_scale in (40.0, 0.0):
        for fmt in ("e4m3", "bf16"):
            s = Setup(dev, fmt, 4, 2, [700], 3, seed=9)
            qkv = s.qkv(3, q_scale=q_scale)
            out = torch.empty(3, 512, device=dev, dtype=BF)
            attn = s.ops.TreeAttention(4, 2, 3, 3, dev, kv_format=fmt)
            pos = [700, 701, 702]
            attn(qkv, s.cos, s.sin, _i32([0] * 3, dev), _i32(pos, dev), s.table, s.pages, out)
            s.check(qkv, [0] * 3, pos, out, _causal(pos))


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_strides_shared_pages_and_pages_outside_the_pool(dev, fmt):
    s = Setup(dev, fmt, 8, 2, [512, 256], 4)
    wide = torch.randn(4, 3000, generator=s.g, device=dev).to(BF)
    qkv = wide[:, 6:6 + 12 * 128]                                            # rows of a wider matrix, 4-byte aligned
    out = torch.full((4, 1100), 9.0, device=dev, dtype=BF)
    table = torch.full((2, 6), 99, dtype=torch.int32, device=dev)            # a table with more columns than are looked at
    table[0, :2], table[0, 2:4] = s.table[0, :2], s.table[0, 2:]
    table[1, 0], table[1, 1:4] = s.table[0, 0], s.table[1, 1:]               # the second sequence shares the first one's first page
    view = table[:, :4]
    seq, pos = [0, 0, 1, 1], [512, 513, 256, 257]
    attn = s.ops.TreeAttention(8, 2, 4, 4, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), view, s.pages, out[:, 4:1028])
    assert bool((out[:, :4] == 9.0).all()) and bool((out[:, 1028:] == 9.0).all())
    s.table = view
    s.check(qkv, seq, pos, out[:, 4:1028], _causal(pos))
    # a page outside the pool in the middle of a sequence: as if nobody saw its positions
    view[0, 1] = 1000
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), view, s.pages, out[:, 4:1028])
    s.check(qkv, seq, pos, out[:, 4:1028], lambda r, p: (p <= pos[r]) & ((seq[r] == 1) | (p < 256) | (p >= 512)))


def test_many_rows_of_one_sequence(dev):
    """A prompt chunk of 300 rows, more than the planning CTA takes at a time."""
    s = Setup(dev, "e4m3", 4, 2, [100, 40], 3)
    seq = [0] * 300 + [-1] * 5 + [1] * 7
    pos = list(range(100, 400)) + [0] * 5 + list(range(40, 47))
    qkv = s.qkv(len(seq))
    out = torch.full((len(seq), 512), 2.0, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(4, 2, len(seq), 3, dev, kv_format="e4m3")
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out)
    keep = [0, 1, 15, 16, 155, 156, 254, 255, 256, 257, 299, 305, 311]
    s.check(qkv[keep], [seq[i] for i in keep], [pos[i] for i in keep], out[keep], _causal([pos[i] for i in keep]))
    assert bool((out[300:305] == 2.0).all())


def test_a_long_context(dev):
    s = Setup(dev, "e4m3", 5, 1, [20000, 33], 80)
    pos, seq = [20000, 20001, 33], [0, 0, 1]
    qkv = s.qkv(3)
    out = torch.empty(3, 640, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(5, 1, 3, 80, dev, kv_format="e4m3")
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out)
    s.check(qkv, seq, pos, out, _causal(pos))


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_more_wide_units_than_the_gpu_holds_at_a_time(dev, fmt):
    """Trees of 64 and of 9 nodes behind contexts that end within and at the end of a part, of one step to forty: every row has the bits
    of its tree alone and of the call before, and rows here and there agree with the definition."""
    lengths = [6000, 4096, 1024, 1, 2047, 5000, 4100, 17, 8127, 63, 6144, 3000]
    nodes = [64, 64, 9, 64, 64, 9, 64, 64, 64, 9, 64, 64]
    s = Setup(dev, fmt, 40, 8, lengths, 33)
    seq, pos, base, rope, mask = [], [], [], [], []
    for slot, (n, count) in enumerate(zip(lengths, nodes)):
        depth, masks = s.ops.TreeRows.masks([-1] + [(7 * i + slot) % (i + 1) for i in range(count - 1)])
        seq += [slot] * count
        pos += range(n, n + count)
        base += [n] * count
        rope += [n + d for d in depth]
        mask += masks
    qkv = s.qkv(len(seq))
    out = torch.full((len(seq), 5120), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(40, 8, len(seq), 33, dev, kv_format=fmt)
    tree = s.ops.TreeRows(_i32(base, dev), _i32(rope, dev), torch.tensor(mask, device=dev))
    call = lambda at, to: attn(qkv[at], s.cos, s.sin, _i32(seq[at], dev), _i32(pos[at], dev), s.table, s.pages, to,
                               tree=s.ops.TreeRows(tree.base[at], tree.rope[at], tree.mask[at]))
    call(slice(0, None), out)
    again = torch.empty_like(out)
    call(slice(0, None), again)
    assert attn.check_status() == 0 and torch.equal(out, again)
    for slot in range(len(lengths)):
        first = seq.index(slot)
        at = slice(first, first + nodes[slot])
        call(at, again[at].zero_())
    assert attn.check_status() == 0 and torch.equal(out, again)
    keep = [seq.index(slot) + i for slot in range(len(lengths)) for i in (0, nodes[slot] - 1)]

    def seen(i, p):
        node = p - base[keep[i]]
        bits = torch.tensor([mask[keep[i]][0] >> b & 1 for b in range(64)], device=dev).bool()
        return (node < 0) | ((node >= 0) & (node < 64) & bits[node.clamp(0, 63)])

    s.check(qkv[keep], [seq[r] for r in keep], [pos[r] for r in keep], out[keep], seen, [rope[r] for r in keep])


@pytest.mark.parametrize("rows", [1025, 4096])
def test_as_many_rows_as_a_call_takes(dev, rows):
    """Runs of 1, 2, 3 ... rows, and one of the rest that is cut into wide tiles: the plan takes 1024 rows at a time."""
    counts, left = [], rows - 700
    while left > 0:
        counts.append(min(len(counts) % 40 + 1, left))
        left -= counts[-1]
    counts.insert(len(counts) // 2, 700)
    s = Setup(dev, "e4m3", 4, 1, [200 if i % 3 else 0 for i in range(len(counts))], 4)
    seq = [slot for slot, n in enumerate(counts) for _ in range(n)]
    pos = [s.lengths[slot] + i for slot, n in enumerate(counts) for i in range(n)]
    qkv = s.qkv(rows)
    out = torch.full((rows, 512), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(4, 1, rows, 4, dev, kv_format="e4m3")
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, longest_run=700)
    assert attn.check_status() == 0 and bool(torch.isfinite(out.float()).all())
    keep = sorted({0, 1, 2, 255, 256, 1023, 1024, rows - 1} | set(range(5, rows, 97)))
    s.check(qkv[keep], [seq[i] for i in keep], [pos[i] for i in keep], out[keep], _causal([pos[i] for i in keep]))


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_captured_and_replayed_with_other_inputs_and_on_another_stream(dev, fmt):
    s = Setup(dev, fmt, 10, 2, [300, 17], 3)
    attn, plain = (s.ops.TreeAttention(10, 2, 8, 3, dev, kv_format=fmt) for _ in range(2))
    depth, masks = s.ops.TreeRows.masks([-1, 0, 0, 1])
    seq, pos = _i32([0] * 4 + [1] * 4, dev), _i32([300, 301, 302, 303, 17, 18, 19, 20], dev)
    tree = s.ops.TreeRows(_i32([300] * 4 + [17] * 4, dev), _i32([300 + d for d in depth] + [17 + d for d in depth], dev), torch.tensor(masks * 2, device=dev))
    qkv, out, want = s.qkv(8), torch.empty(8, 1280, device=dev, dtype=BF), torch.empty(8, 1280, device=dev, dtype=BF)
    attn(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, out, tree=tree)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, out, tree=tree)
    for shift in (0, 256):
        qkv.copy_(s.qkv(8))
        pos.add_(shift); tree.base.add_(shift); tree.rope.add_(shift)      # (the positions between hold NaN codes until they are written)
        if shift:
            for slot in range(2):
                n = shift + [300, 17][slot]
                k = torch.randn(n, 2, 128, generator=s.g, device=dev).to(BF)
                s.ops.kv_write(k, k, _i32([slot] * n, dev), _i32(range(n), dev), s.table, s.pages)
        graph.replay()
        plain(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, want, tree=tree)
        assert torch.equal(out, want) and bool(torch.isfinite(out.float()).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plain(qkv, s.cos, s.sin, seq, pos, s.table, s.pages, want.zero_(), tree=tree)
    side.synchronize()
    assert torch.equal(out, want)


def test_refusals(dev):
    s = Setup(dev, "e4m3", 8, 2, [10], 2)
    attn = s.ops.TreeAttention(8, 2, 4, 2, dev, kv_format="e4m3")
    i, qkv, out = _i32([0, 0], dev), s.qkv(2), torch.empty(2, 1024, device=dev, dtype=BF)
    tree = s.ops.TreeRows(i, i, torch.ones(2, 1, dtype=torch.int64, device=dev))
    three = s.ops.TreeRows(_i32([0] * 3, dev), _i32([0] * 3, dev), torch.ones(3, 1, dtype=torch.int64, device=dev))
    other = s.ops.KVPages.alloc(2, 2, dev)
    stack = s.ops.KVPages.alloc(2, 2, dev, kv_format="e4m3", layers=2)
    go = lambda qkv=qkv, cos=s.cos, sin=s.sin, seq=i, pos=i, table=s.table, pages=s.pages, out=out, tree=None: attn(qkv, cos, sin, seq, pos, table, pages, out, tree=tree)
    go(tree=tree)
    for bad in (dict(qkv=qkv[:, :-1]), dict(qkv=qkv.float()), dict(qkv=s.qkv(5)), dict(out=out[:1]), dict(out=out.float()), dict(cos=s.cos.float()), dict(cos=s.cos[:, :64]),
                dict(sin=s.sin[:5]), dict(seq=i.long()), dict(pos=i[:1]), dict(pos=_i32([0, 0, 0, 0], dev)[::2]), dict(table=torch.zeros(1, 3, dtype=torch.int32, device=dev)),
                dict(table=s.table.cpu()), dict(pages=other), dict(pages=stack), dict(tree=three), dict(qkv=qkv.t().contiguous().t()), dict(out=out.t().contiguous().t())):
        with pytest.raises(ValueError):
            go(**bad)
