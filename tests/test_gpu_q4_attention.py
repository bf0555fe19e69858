"""Attention of causal rows, prompt chunks and draft trees over a 4-bit cache, against its definition in 64 bits (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from q4_reference import Setup, causal, i32  # noqa: E402
from spec_reference import attend, rotate  # noqa: E402

BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _masks(masks, dev):
    return torch.tensor(masks, dtype=torch.int64, device=dev)


def _seen(base, mask):
    words = len(mask[0])

    def seen(r, p):
        node = p - base[r]
        bits = torch.tensor([mask[r][w] >> b & 1 for w in range(words) for b in range(64)], device=p.device).bool()
        return (node < 0) | ((node >= 0) & (node < 64 * words) & bits[node.clamp(0, 64 * words - 1)])

    return seen


@pytest.mark.parametrize("nq,nkv", [(5, 1), (4, 4), (6, 2), (16, 1), (14, 2), (8, 1), (9, 1), (10, 2), (3, 1)])
def test_causal_rows(dev, nq, nkv):
    """Decode rows, chains and prompt rows together; lengths at the borders of chunks, pages and parts."""
    lengths = [0, 1, 31, 32, 33, 127, 128, 255, 256, 511, 512, 513, 900]
    s = Setup(dev, nq, nkv, lengths, 4)
    per = [3, 1, 1, 2, 1, 1, 1, 4, 1, 2, 1, 1, 21]
    seq = [i for i, n in enumerate(per) for _ in range(n)]
    pos = [lengths[i] + j for i, n in enumerate(per) for j in range(n)]
    rows = len(seq)
    qkv, out = s.qkv(rows), torch.full((rows, nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.attention(rows)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out)
    s.check(qkv, seq, pos, out, causal(pos))
    # a row alone, a row said to be alone, rows that are said to be and are not, and the rows in another order: the same bits
    solo = torch.empty(1, nq * 128, device=dev, dtype=BF)
    for r in (0, 5, 9, rows - 1):
        for longest in (None, 1):
            attn(qkv[r:r + 1], s.cos, s.sin, i32(seq[r:r + 1], dev), i32(pos[r:r + 1], dev), s.table, s.pages, solo, longest_run=longest)
            assert torch.equal(solo[0], out[r])
    again = torch.empty_like(out)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, again, longest_run=1)
    assert torch.equal(again, out)
    back = list(range(rows))[::-1]
    attn(qkv[back].contiguous(), s.cos, s.sin, i32([seq[i] for i in back], dev), i32([pos[i] for i in back], dev), s.table, s.pages, again)
    assert torch.equal(again[back], out)
    assert attn.check_status() == 0


def test_steps_and_a_chain_give_the_same_bits(dev):
    """Tokens decoded one by one, across the end of a part, and the same tokens as rows of one pass."""
    bits = []
    for chain in (False, True):
        s = Setup(dev, 10, 2, [506], 3, seed=3)
        qkv, attn, out = s.qkv(9), s.attention(9), torch.empty(9, 1280, device=dev, dtype=BF)
        for rows in ([slice(0, 9)] if chain else [slice(i, i + 1) for i in range(9)]):
            pos = list(range(506, 515))[rows]
            attn(qkv[rows], s.cos, s.sin, i32([0] * len(pos), dev), i32(pos, dev), s.table, s.pages, out[rows], longest_run=None if chain else 1)
        bits.append(out.clone())
    assert torch.equal(*bits)


@pytest.mark.parametrize("nq,nkv,rows,before", [(5, 1, 64, 0), (10, 2, 64, 449), (8, 2, 65, 500), (16, 1, 70, 1000), (4, 4, 130, 100), (40, 8, 100, 1500), (5, 1, 200, 2500)])
def test_prompt_rows_go_through_the_tensor_cores(dev, nq, nkv, rows, before):
    pages = -(-(before + rows) // 256)
    s = Setup(dev, nq, nkv, [before, 40], pages, seed=rows)
    seq, pos = [0] * rows + [1], list(range(before, before + rows)) + [40]
    qkv, out = s.qkv(rows + 1), torch.full((rows + 1, nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.attention(rows + 1)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, longest_run=rows)
    assert attn.check_status() == 0
    s.check(qkv, seq, pos, out, causal(pos), rows=[0, 1, rows // 2, rows - 2, rows - 1, rows])
    alone = torch.empty(rows, nq * 128, device=dev, dtype=BF)
    attn(qkv[:rows], s.cos, s.sin, i32(seq[:rows], dev), i32(pos[:rows], dev), s.table, s.pages, alone, longest_run=rows)
    assert torch.equal(alone, out[:rows])


TREES = {"one": [-1], "pair": [-1, 0], "star": [-1] + [0] * 9, "chain": list(range(-1, 15)), "bushy": [-1, 0, 0, 0, 1, 1, 2, 4, 4, 7, 3, 10, 11, 5],
         "wide": [-1] + [i // 3 for i in range(63)], "words": [-1] + [(i * 7) // 11 for i in range(129)]}


@pytest.mark.parametrize("nq,nkv", [(5, 1), (8, 2), (6, 1), (16, 1), (4, 4)])
def test_trees(dev, nq, nkv):
    """Trees of 1 to 130 nodes behind contexts of no position, some, and pages full, in one call: in both kernels."""
    lengths = [0, 300, 1, 256, 250, 700, 505]
    s = Setup(dev, nq, nkv, lengths, 4)
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
    qkv, out = s.qkv(rows), torch.full((rows, nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.attention(rows)
    tree = s.ops.TreeRows(i32(base, dev), i32(rope, dev), _masks(mask, dev))
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, tree=tree)
    s.check(qkv, seq, pos, out, _seen(base, mask), rope, rows=list(range(0, 43)) + list(range(43, rows, 9)))
    at, n = seq.index(5), seq.count(5)
    part = slice(at, at + n)
    alone = torch.empty(n, nq * 128, device=dev, dtype=BF)
    attn(qkv[part], s.cos, s.sin, i32(seq[part], dev), i32(pos[part], dev), s.table, s.pages, alone, tree=s.ops.TreeRows(tree.base[part], tree.rope[part], tree.mask[part]))
    assert torch.equal(alone, out[part]) and attn.check_status() == 0


@pytest.mark.parametrize("copies", [1, 20])
def test_rows_that_see_nothing_and_rows_left_out(dev, copies):
    """In the narrow kernel, and (20 rows of a sequence) in the wide one."""
    s = Setup(dev, 8, 2, [0, 300, 20], 2)
    if copies == 1:
        seq, pos = [0, 0, -1, 1, 1, 2, 1], [0, 1, 5, 300, 310, 999, 301]         # (position 999 lies outside the table)
        base, rope, mask = [0, 0, 0, 300, 0, 20, 300], [0, 1, 5, 300, 310, 22, 700], [[0], [2], [1], [1], [0], [1], [2]]     # (row 6: outside the rotary tables)
        nothing, absent = [0, 4], [2, 5, 6]
    else:
        seq, pos, rope = [1] * 20, [300 + i for i in range(20)], [300 + i for i in range(20)]
        base, mask = [300] * 20, [[1 << i] for i in range(20)]
        base[3], mask[3] = 0, [0]
        rope[7] = 9999
        nothing, absent = [3], [7]
    rows = len(seq)
    qkv, out = s.qkv(rows), torch.full((rows, 1024), 5.0, device=dev, dtype=BF)
    attn = s.attention(rows)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, tree=s.ops.TreeRows(i32(base, dev), i32(rope, dev), _masks(mask, dev)))
    assert bool((out[absent] == 5.0).all()) and bool((out[nothing] == 0.0).all())
    keep = [r for r in range(rows) if r not in absent]
    s.check(qkv, seq, pos, out, _seen(base, mask), rope, rows=keep)
    attn(qkv[:0], s.cos, s.sin, i32([], dev), i32([], dev), s.table, s.pages, out[:0])          # no rows at all


@pytest.mark.parametrize("more", [0, 20])
def test_nan_and_infinity_stay_with_the_rows_that_see_them(dev, more):
    """A tree's node, then the cached context; ``more`` rows beside them take the tree to the wide kernel."""
    s = Setup(dev, 8, 2, [260, 260], 2)
    n = 4 + more
    depth, masks = s.ops.TreeRows.masks([-1, 0, 0, 2] + [0] * more)
    qkv = s.qkv(2 * n)
    qkv[1, 8 * 128 + 5] = float("nan")                                      # node 1's key, kv head 0
    qkv[n + 1, 10 * 128 + 5] = float("inf")                                 # the other sequence's node 1: a value, kv head 0
    seq, pos = [0] * n + [1] * n, [260 + i for i in range(n)] * 2
    tree = s.ops.TreeRows(i32([260] * (2 * n), dev), i32([260 + d for d in depth] * 2, dev), _masks(masks * 2, dev))
    out, attn = torch.empty(2 * n, 1024, device=dev, dtype=BF), s.attention(2 * n)
    go = lambda: attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, tree=tree)
    go()
    assert (~torch.isfinite(out.float())).view(2 * n, 2, 4, 128).any(-1).any(-1).tolist() == [[r in (1, n + 1), False] for r in range(2 * n)]
    qkv = s.qkv(2 * n)
    qkv[2, 3 * 128 + 7] = float("inf")                                      # a query that is not finite: its head alone
    go()
    bad = (~torch.isfinite(out.float())).view(2 * n, 8, 128).any(-1)
    assert bool(bad[2, 3]) and int(bad.sum()) == 1
    for which, pages in ((0, s.pages.k), (1, s.pages.v)):                    # the cached context: every row of the sequence sees it
        flat = pages[int(s.table[which, 0]), 1].flatten()
        flat[64 * 17:64 * 18], flat[17408 + 17] = 0x88, 255
        qkv = s.qkv(2 * n)
        go()
        assert out.float().isnan().view(2 * n, 2, 512).any(-1).tolist() == [[False, r < n or which == 1] for r in range(2 * n)]


@pytest.mark.parametrize("nodes", [[0, 5, 40], [0, 5, 40] + list(range(41, 60))])
def test_holes_between_a_trees_nodes_may_hold_anything(dev, nodes):
    """Other places hold bytes that nobody wrote, not-a-number among them, and no row sees them."""
    s = Setup(dev, 10, 2, [250], 2)
    masks, n = [[1 | 1 << i] for i in nodes], len(nodes)
    pos, rope, base = [250 + i for i in nodes], [250] + [251] * (n - 1), [250] * n
    qkv, out = s.qkv(n), torch.empty(n, 1280, device=dev, dtype=BF)
    s.attention(n)(qkv, s.cos, s.sin, i32([0] * n, dev), i32(pos, dev), s.table, s.pages, out, tree=s.ops.TreeRows(i32(base, dev), i32(rope, dev), _masks(masks, dev)))
    s.check(qkv, [0] * n, pos, out, _seen(base, masks), rope)


@pytest.mark.parametrize("rows", [2, 66])
@pytest.mark.parametrize("scale", [1e-7, 1e3, 0.0])
def test_sizes_of_values(dev, scale, rows):
    """Values (and keys) whose sizes differ by many powers of two between positions, all tiny, all large, all zero."""
    s = Setup(dev, 8, 2, [520], 3, scale=scale)
    qkv = s.qkv(rows, q_scale=1.0 if scale < 1 else 1e-2)
    qkv[:, 8 * 128:] *= scale
    qkv[1, 10 * 128:] *= 2.0 ** -12
    out = torch.empty(rows, 1024, device=dev, dtype=BF)
    s.attention(rows)(qkv, s.cos, s.sin, i32([0] * rows, dev), i32(range(520, 520 + rows), dev), s.table, s.pages, out, longest_run=rows)
    half = 2.0 ** -11
    for r in (0, 1, rows - 1):
        p = 520 + r
        k, v = s.held(0, 768)
        want, bound = attend(rotate(qkv[r].view(-1, 128)[:8], s.cos[p], s.sin[p]), k, v, torch.arange(768, device=dev) <= p, half, half)
        # FP16 weights below their normal range: 2^-25 of the largest product, of which there are p + 1
        assert bool(((out[r].view(8, 128).double() - want).abs() <= bound + (p + 1) * 2.0 ** -24 * v[:p + 1].abs().amax()).all())


@pytest.mark.parametrize("q_scale", [40.0, 0.0])
def test_sharp_and_flat_scores(dev, q_scale):
    """Scores of hundreds (one position takes all; references move from chunk to chunk), and all alike."""
    s = Setup(dev, 4, 2, [1300], 6, seed=9)
    qkv, out, pos = s.qkv(3, q_scale=q_scale), torch.empty(3, 512, device=dev, dtype=BF), [1300, 1301, 1302]
    s.attention(3)(qkv, s.cos, s.sin, i32([0] * 3, dev), i32(pos, dev), s.table, s.pages, out)
    s.check(qkv, [0] * 3, pos, out, causal(pos))


def test_strides_shared_pages_and_pages_outside_the_pool(dev):
    s = Setup(dev, 8, 2, [512, 256], 4)
    wide = torch.randn(4, 3000, generator=s.g, device=dev).to(BF)
    qkv = wide[:, 6:6 + 12 * 128]                                            # rows of a wider matrix, 4-byte aligned
    out = torch.full((4, 1100), 9.0, device=dev, dtype=BF)
    table = torch.full((2, 6), 99, dtype=torch.int32, device=dev)            # a table with more columns than are looked at
    table[0, :2], table[0, 2:4] = s.table[0, :2], s.table[0, 2:]
    table[1, 0], table[1, 1:4] = s.table[0, 0], s.table[1, 1:]               # the second sequence shares the first one's first page
    view = table[:, :4]
    seq, pos = [0, 0, 1, 1], [512, 513, 256, 257]
    attn = s.attention(4)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), view, s.pages, out[:, 4:1028])
    assert bool((out[:, :4] == 9.0).all()) and bool((out[:, 1028:] == 9.0).all())
    s.table = view
    s.check(qkv, seq, pos, out[:, 4:1028].contiguous(), causal(pos))
    # a page outside the pool: as if nobody saw its positions
    table[0, 0] = 99
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), view, s.pages, out[:, 4:1028])
    s.check(qkv, seq, pos, out[:, 4:1028].contiguous(), lambda r, p: (p <= pos[r]) & ((p >= 256) if r < 2 else (p >= 0)), rows=[0, 1, 2, 3])


def test_a_captured_step_replayed_on_new_inputs_and_two_streams(dev):
    s = Setup(dev, 10, 2, [700, 90], 4)
    attn, rows = s.attention(2), [0, 1]
    qkv, out = s.qkv(2), torch.empty(2, 1280, device=dev, dtype=BF)
    seq, pos = i32(rows, dev), i32([700, 90], dev)
    go = lambda a, q, o: a(q, s.cos, s.sin, seq, pos, s.table, s.pages, o, longest_run=1)
    go(attn, qkv, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(attn, qkv, out)
    for turn in range(3):
        qkv.copy_(s.qkv(2))
        graph.replay()
        pos.add_(1)
    s.check(qkv, rows, [702, 92], out, causal([702, 92]))
    # two objects on two streams, each with rows of its own sequence
    other, streams, outs, inputs = s.attention(2), [torch.cuda.Stream(dev) for _ in range(2)], [torch.empty(1, 1280, device=dev, dtype=BF) for _ in range(2)], [s.qkv(1) for _ in range(2)]
    torch.cuda.synchronize()
    for a, stream, o, q, r in zip((attn, other), streams, outs, inputs, rows):
        with torch.cuda.stream(stream):
            for _ in range(5):
                a(q, s.cos, s.sin, seq[r:r + 1], pos[r:r + 1], s.table, s.pages, o, longest_run=1)
    torch.cuda.synchronize()
    for r in rows:
        s.check(inputs[r], [r], [int(pos[r])], outs[r], causal([int(pos[r])]))


def test_runs_of_the_wide_kernel_without_anything_to_do(dev):
    """Whole tiles of rows that are left out or see nothing, before, between and behind others."""
    s = Setup(dev, 10, 2, [0, 300, 20, 40], 3)
    seq = [-1] * 70 + [1] * 66 + [-1] * 130 + [2] * 3 + [0] * 64
    pos = [5] * 70 + [300 + i for i in range(66)] + [700] * 130 + [20, 21, 22] + list(range(64))
    rows = len(seq)
    qkv, out = s.qkv(rows), torch.full((rows, 1280), 5.0, device=dev, dtype=BF)
    attn = s.attention(rows)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, longest_run=130)
    keep = [r for r in range(rows) if seq[r] >= 0]
    absent = [r for r in range(rows) if seq[r] < 0]
    assert attn.check_status() == 0 and bool((out[absent] == 5.0).all())
    s.check(qkv, seq, pos, out, causal(pos), rows=[keep[i] for i in (0, 1, 40, 65, 66, 68, 69, 100, 132)])
    # nodes of trees that see nothing: 60 of one, all of another
    seq, pos = [1] * 64 + [3] * 20, [300 + i for i in range(64)] + [40 + i for i in range(20)]
    base, mask = [300] * 2 + [0] * 60 + [300] * 2 + [0] * 20, [[1], [3]] + [[0]] * 60 + [[1 << 62 | 1], [3 << 62 | 1]] + [[0]] * 20
    rows = len(seq)
    qkv, out = s.qkv(rows), torch.full((rows, 1280), 5.0, device=dev, dtype=BF)
    attn = s.attention(rows)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, tree=s.ops.TreeRows(i32(base, dev), i32(pos, dev), _masks([[m if m < 1 << 63 else m - (1 << 64) for m in x] for x in mask], dev)))
    assert attn.check_status() == 0 and bool((out[2:62] == 0).all()) and bool((out[64:] == 0).all())
    s.check(qkv, seq, pos, out, _seen(base, mask), pos, rows=[0, 1, 62, 63])


@pytest.mark.parametrize("rows,before", [(66, 4031), (66, 4032), (70, 9000), (150, 4100), (66, 16400)])
def test_prompt_rows_behind_long_contexts(dev, rows, before):
    """Parts of every size, of which a tile's last may be short; a run by itself has the same bits."""
    s = Setup(dev, 5, 1, [before, 100], -(-(before + rows) // 256), seed=rows)
    seq, pos = [0] * rows + [1] * 64, list(range(before, before + rows)) + list(range(100, 164))
    qkv, out = s.qkv(rows + 64), torch.full((rows + 64, 640), float("nan"), device=dev, dtype=BF)
    attn = s.attention(rows + 64)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out, longest_run=rows)
    assert attn.check_status() == 0
    s.check(qkv, seq, pos, out, causal(pos), rows=[0, rows // 2, rows - 1, rows, rows + 63])
    alone = torch.empty(rows, 640, device=dev, dtype=BF)
    attn(qkv[:rows], s.cos, s.sin, i32(seq[:rows], dev), i32(pos[:rows], dev), s.table, s.pages, alone, longest_run=rows)
    assert torch.equal(alone, out[:rows])


def test_long_contexts_and_many_units_a_cta(dev):
    """Runs of units over several sequences, parts and heads, one and two blocks of columns."""
    lengths = [3000 + 37 * i for i in range(12)]
    for nq, nkv, longest in ((40, 8, 1), (32, 2, 1)):
        s = Setup(dev, nq, nkv, lengths, 14, seed=1)
        qkv, out = s.qkv(12), torch.empty(12, nq * 128, device=dev, dtype=BF)
        s.attention(12)(qkv, s.cos, s.sin, i32(range(12), dev), i32(lengths, dev), s.table, s.pages, out, longest_run=longest)
        s.check(qkv, list(range(12)), lengths, out, causal(lengths), rows=[0, 5, 11])
