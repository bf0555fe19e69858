"""Pages of a cache copied, forked, freed and compacted, against plain bookkeeping on the host (needs a B200)."""
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

FORMATS = ["bf16", "e4m3", "q4"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


class Cache:
    """A stack of layers with bytes of any kind, and its copy on the host as [layers][pages][heads][256 positions][bytes of an entry]."""

    def __init__(self, dev, fmt, layers, pages, heads, seed=0):
        from georefine_b200 import ops

        g = torch.Generator(device=dev).manual_seed(seed)
        self.ops, self.dev, self.fmt = ops, dev, fmt
        self.pages = ops.KVPages.alloc(pages, heads, dev, kv_format=fmt, layers=layers)
        for t in self._tensors():
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
        self.host = self.entries()

    def _tensors(self):
        return [t.view(torch.uint8) for t in (self.pages.k, self.pages.v, self.pages.k_exp, self.pages.v_exp) if t is not None]

    def entries(self):
        """Every byte of the cache, by the entry it belongs to."""
        out = []
        for t in (x.cpu() for x in self._tensors()):
            if self.fmt == "q4":
                flat = t.flatten(3)
                out += [flat[..., :16384].unflatten(-1, (256, 64)).clone(), flat[..., 16384:17408].unflatten(-1, (256, 4)).clone(), flat[..., 17408:].unflatten(-1, (256, 1)).clone()]
            else:
                out.append((t if t.dim() == 5 else t[..., None]).clone())
        return out

    def move(self, src, dst, count=256):
        for x in self.host:
            x[:, dst, :, :count] = x[:, src, :, :count].clone()

    def check(self):
        for a, b in zip(self.entries(), self.host):
            assert torch.equal(a, b)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("layers,heads", [(1, 1), (3, 2), (2, 8)])
def test_copies(dev, fmt, layers, heads):
    c = Cache(dev, fmt, layers, 12, heads)
    src, dst, count = [0, 1, 2, 3, -1, 5, 99, 4], [6, 7, 8, 9, 10, -1, 11, 4], [256, 0, 1, 255, 9, 9, 9, 17]
    c.ops.kv_copy(_i32(src, dev), _i32(dst, dev), c.pages, positions=_i32(count, dev))
    for s, d, n in list(zip(src, dst, count))[:4]:
        c.move(s, d, n)
    c.check()
    c.ops.kv_copy(_i32([0, 0], dev), _i32([10, 11], dev), c.pages)           # one source twice, whole
    c.move(0, 10)
    c.move(0, 11)
    c.check()
    c.ops.kv_copy(_i32([1], dev), _i32([2], dev), c.pages, positions=_i32([1000], dev))          # (more than there are: all)
    c.move(1, 2)
    c.ops.kv_copy(_i32([], dev), _i32([], dev), c.pages)
    c.check()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("empty", [-1, 19])
def test_forks_and_frees(dev, fmt, empty):
    """Lengths of zero, one, a page's border and others; many children of a parent; a table wider than is looked at."""
    c = Cache(dev, fmt, 2, 20, 2, seed=4)
    table = torch.full((9, 6), 77, dtype=torch.int32, device=dev)
    view = table[:, :4]
    view.fill_(empty)
    view[0, :3], view[1, :2] = _i32([3, 0, 7], dev), _i32([5, 2], dev)
    refs = torch.zeros(20, dtype=torch.int32, device=dev)
    refs[[3, 0, 7, 5, 2]] = 1
    forks = [(0, 2, 700, 10), (0, 3, 512, 11), (1, 4, 1, 12), (0, 5, 256, -1), (1, 6, 0, -1), (0, 7, 513, 13), (-1, 8, 5, 14), (0, 99, 5, 14), (0, 8, 5000, 14)]
    host, counts = view.cpu().clone(), refs.cpu().clone()
    for parent, child, length, fresh in forks[:6]:
        whole, rest = divmod(length, 256)
        row = [int(x) for x in host[parent, :whole]] + ([fresh] if rest else [])
        for p in row:
            counts[p] += 1
        host[child] = torch.tensor(row + [empty] * (4 - len(row)))
        if rest:
            c.move(int(host[parent, whole]), fresh, rest)
    c.ops.kv_fork(*(_i32(x, dev) for x in zip(*forks)), view, refs, c.pages, empty=empty)
    assert torch.equal(view.cpu(), host) and torch.equal(refs.cpu(), counts) and bool((table[:, 4:] == 77).all())
    c.check()
    # without a fresh page in the pool: the whole pages alone
    c.ops.kv_fork(_i32([0], dev), _i32([8], dev), _i32([700], dev), _i32([20], dev), view, refs, c.pages, empty=empty)
    assert view[8].tolist() == [3, 0, empty, empty] and refs[[3, 0]].tolist() == [int(counts[3]) + 1, int(counts[0]) + 1]
    c.ops.kv_free(_i32([8], dev), view, refs, empty=empty)
    # some of them freed, one twice, one that holds nothing, slots that are not there
    freed = [2, 5, 2, 6, -1, 55]
    for s in (2, 5):
        for p in host[s].tolist():
            if p != empty:
                counts[p] -= 1
        host[s] = empty
    c.ops.kv_free(_i32(freed, dev), view, refs, empty=empty)
    assert torch.equal(view.cpu(), host) and torch.equal(refs.cpu(), counts)
    c.check()
    for s in (0, 1, 3, 4, 7):
        c.ops.kv_free(_i32([s], dev), view, refs, empty=empty)
    assert int(refs.abs().sum()) == 0 and bool((view == empty).all()) and bool((table[:, 4:] == 77).all())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("pages,share", [(1, 1.0), (1, 0.0), (7, 0.5), (40, 0.5), (64, 0.0), (64, 1.0), (97, 0.2), (97, 0.9)])
def test_compaction(dev, fmt, pages, share):
    rng = random.Random(pages * 100 + int(share * 10))
    c = Cache(dev, fmt, 2, pages, 1, seed=pages)
    held = [p for p in range(pages) if rng.random() < share]
    rng.shuffle(held)
    table = torch.full((5, 30), -1, dtype=torch.int32)
    for i, p in enumerate(held):
        table.view(-1)[i] = p
    if held:
        table[4, -1] = held[0]                                               # one page twice
    table[4, -2] = 1000                                                      # (a number outside the pool stays)
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table.flatten().tolist():
        if 0 <= p < pages:
            refs[p] += 1
    dev_table, dev_refs = table.to(dev), refs.to(dev)
    where, used = torch.full((pages,), 5, dtype=torch.int32, device=dev), torch.full((1,), 5, dtype=torch.int32, device=dev)
    scratch = torch.empty(c.ops.kv_compact_scratch_bytes(c.pages), dtype=torch.uint8, device=dev) if pages % 2 else None
    c.ops.kv_compact(dev_table, dev_refs, c.pages, where, used, scratch=scratch)
    u = len(held)
    sources, targets = [p for p in range(u, pages) if p in set(held)], [p for p in range(u) if p not in set(held)]
    moves = dict(zip(sources, targets))
    want = [moves.get(p, p) if p in set(held) else -1 for p in range(pages)]
    for s, d in moves.items():
        c.move(s, d)
    assert int(used) == u and where.tolist() == want
    assert dev_table.flatten().tolist() == [want[p] if 0 <= p < pages else p for p in table.flatten().tolist()]
    assert dev_refs.tolist() == [sum(1 for q in table.flatten().tolist() if 0 <= q < pages and want[q] == p) for p in range(pages)]
    c.check()
    before = [t.clone() for t in c._tensors()]
    c.ops.kv_compact(dev_table, dev_refs, c.pages, where, used)              # nothing is left to move
    assert where.tolist() == [p if p < u else -1 for p in range(pages)] and all(torch.equal(a, b) for a, b in zip(before, c._tensors()))


def test_a_large_pool_is_planned_in_many_rounds(dev):
    from georefine_b200 import ops

    pages = 5000
    k, v = (torch.zeros(pages, 1, 69, 256, dtype=torch.uint8, device=dev) for _ in range(2))
    k[:, 0, 0, :2] = torch.stack([torch.arange(pages) % 256, torch.arange(pages) // 256], 1).to(torch.uint8).to(dev)
    g = torch.Generator().manual_seed(0)
    refs = (torch.rand(pages, generator=g) < 0.5).int()
    u = int(refs.sum())
    table, where, used = torch.arange(pages, dtype=torch.int32, device=dev)[None].contiguous(), *(torch.empty(n, dtype=torch.int32, device=dev) for n in (pages, 1))
    ops.kv_compact(table, refs.to(dev), ops.KVPages(k, v), where, used)
    held = refs.bool()
    number = torch.arange(pages)
    src, dst = number[held & (number >= u)], number[~held & (number < u)]
    want = torch.where(held, number, -1)
    want[src] = dst
    assert int(used) == u and torch.equal(where.cpu().long(), want)
    at = k[:u, 0, 0, :2].cpu().long()
    origin = torch.empty(u, dtype=torch.long)
    origin[want[held]] = number[held]
    assert torch.equal(at[:, 0] + 256 * at[:, 1], origin)
    assert torch.equal(table[0].cpu().long(), torch.where(held, want, number))


def test_forks_and_compactions_replayed_from_a_graph(dev):
    c = Cache(dev, "q4", 2, 8, 2, seed=8)
    table = torch.full((4, 3), -1, dtype=torch.int32, device=dev)
    table[0, :2] = _i32([6, 2], dev)
    refs = torch.zeros(8, dtype=torch.int32, device=dev)
    refs[[6, 2]] = 1
    args = [_i32(x, dev) for x in ([0, 0], [1, 2], [300, 256], [5, -1])]
    where, used, scratch = torch.empty(8, dtype=torch.int32, device=dev), torch.empty(1, dtype=torch.int32, device=dev), torch.empty(c.ops.kv_compact_scratch_bytes(c.pages), dtype=torch.uint8, device=dev)

    def go():
        c.ops.kv_free(args[1], table, refs)
        c.ops.kv_fork(*args, table, refs, c.pages)

    go()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    for _ in range(3):
        graph.replay()
    c.move(2, 5, 44)
    assert table.tolist() == [[6, 2, -1], [6, 5, -1], [6, -1, -1], [-1, -1, -1]] and refs.tolist() == [0, 0, 1, 0, 0, 1, 3, 0]
    c.check()
    packing = torch.cuda.CUDAGraph()
    with torch.cuda.graph(packing):
        c.ops.kv_compact(table, refs, c.pages, where, used, scratch=scratch)
    for turn in range(2):
        packing.replay()
        assert int(used) == 3 and where.tolist() == ([-1, -1, 2, -1, -1, 0, 1, -1] if turn == 0 else [0, 1, 2, -1, -1, -1, -1, -1])
    assert table.tolist() == [[1, 2, -1], [1, 0, -1], [1, -1, -1], [-1, -1, -1]] and refs.tolist() == [1, 3, 1, 0, 0, 0, 0, 0]
    c.move(5, 0)
    c.move(6, 1)
    c.check()
