"""A 4-bit KV cache: rows in and out, kept paths, byte for byte by the definition in 64 bits (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from q4_reference import GRID, entry, i32, packed  # noqa: E402

BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _inputs(dev, kind, rows, heads, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(rows, heads, 128, generator=g, device=dev)
    if kind == "sizes":              # entries of all sizes, groups of an entry of very different ones
        x *= torch.exp2(torch.randint(-60, 40, (rows, heads, 1), generator=g, device=dev).float())
        x = (x.unflatten(-1, (4, 32)) * torch.exp2(torch.randint(-20, 1, (rows, heads, 4, 1), generator=g, device=dev).float())).flatten(-2)
    elif kind == "ties":             # values on the borders between two codes, groups whose scales lie on borders, zeros of both signs
        x = torch.randint(-15, 16, (rows, heads, 128), generator=g, device=dev) * 0.5
        x *= (16 + torch.randint(0, 32, (rows, heads, 1), generator=g, device=dev)) * 0.5
        x[:, :, 0] = 7 * (33 + 2 * torch.randint(0, 16, (rows, heads), generator=g, device=dev)) * 0.25
        x[:, :, 96:] *= -0.0
    elif kind == "extremes":
        pick = torch.tensor([0.0, -0.0, 1e-38, 9e-41, 3.0e38, -3.0e38, 1.0, 57344.0, 111104.0, 131072.0, 2.0 ** -52, 448.0], device=dev)
        x = pick[torch.randint(0, len(pick), (rows, heads, 128), generator=g, device=dev)]
    return x.to(BF)


def _bytes(pages, which, page, head, at):
    flat = (pages.k if which == 0 else pages.v)[page, head].flatten()
    return flat[64 * at:64 * at + 64], flat[16384 + 4 * at:16384 + 4 * at + 4], flat[17408 + at]


@pytest.mark.parametrize("kind", ["normal", "sizes", "ties", "extremes"])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_entries_are_those_of_the_definition(dev, kind, heads):
    from georefine_b200 import ops

    rows = 70
    k, v = (_inputs(dev, kind, rows, heads, seed) for seed in (1, 2))
    table = i32([[3, 1], [0, 2]][0], dev)[None].repeat(2, 1)
    table[1] = i32([0, 2], dev)
    pages = ops.KVPages.alloc(4, heads, dev, kv_format="q4")
    seq, pos = [r % 2 for r in range(rows)], [230 + r // 2 for r in range(rows)]               # across the border of a page
    ops.kv_write(k, v, i32(seq, dev), i32(pos, dev), table, pages)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv_read(i32(seq, dev), i32(pos, dev), table, pages, ko, vo)
    for which, (x, got) in enumerate(((k, ko), (v, vo))):
        code, scale, byte, value = entry(x)
        assert torch.equal(got.double(), value)
        codes = packed(code)
        for r in range(0, rows, 7):
            page = int(table[seq[r], pos[r] // 256])
            for h in range(heads):
                held = _bytes(pages, which, page, h, pos[r] % 256)
                assert torch.equal(held[0], codes[r, h]) and torch.equal(held[1], scale[r, h]) and int(held[2]) == int(byte[r, h])


def test_a_value_is_off_by_half_a_step_at_most(dev):
    """Half a step: a fourteenth of the group's largest value, by a scale that is off by 2^-5 of itself at most."""
    from georefine_b200 import ops

    x = _inputs(dev, "normal", 256, 4, 5)
    pages = ops.KVPages.alloc(1, 4, dev, kv_format="q4")
    table, seq, pos = torch.zeros(1, 1, dtype=torch.int32, device=dev), i32([0] * 256, dev), i32(range(256), dev)
    ops.kv_write(x, x, seq, pos, table, pages)
    out = torch.empty_like(x)
    ops.kv_read(seq, pos, table, pages, out, out.clone())
    top = x.double().unflatten(-1, (4, 32)).abs().amax(-1, keepdim=True)
    off = (out.double() - x.double()).unflatten(-1, (4, 32)).abs()
    assert bool((off <= top / 14 * (1 + 2.0 ** -5)).all())


def test_not_finite_entries_and_memory_of_zeros(dev):
    from georefine_b200 import ops

    x = torch.ones(4, 2, 128, device=dev, dtype=BF)
    x[0, 0, 5], x[1, 1, 127], x[2, 0, 64] = float("nan"), float("inf"), float("-inf")
    pages = ops.KVPages.alloc(1, 2, dev, kv_format="q4")
    table, seq, pos = torch.zeros(1, 1, dtype=torch.int32, device=dev), i32([0] * 4, dev), i32(range(4), dev)
    ops.kv_write(x, x, seq, pos, table, pages)
    k, v = (torch.empty(5, 2, 128, device=dev, dtype=BF) for _ in range(2))
    ops.kv_read(i32([0] * 5, dev), i32([0, 1, 2, 3, 200], dev), table, pages, k, v)
    bad = [[True, False], [False, True], [True, False], [False, False], [False, False]]
    for got in (k, v):
        assert got.isnan().all(-1).tolist() == bad and got.isnan().any(-1).tolist() == bad
        assert bool((got[4] == 0).all())                                                       # nobody wrote there
        assert bool((got[3] == 7 * 18 / 128).all())                                            # (128 / 7 = 18.3: the scale nearest to a seventh is 18 / 128)
    held = _bytes(pages, 0, 0, 0, 0)
    assert bool((held[0] == 0x88).all()) and bool((held[1] == 64).all()) and int(held[2]) == 255


def test_rows_left_out_strides_and_places_outside(dev):
    from georefine_b200 import ops

    wide = torch.randn(6, 1000, device=dev).to(BF)
    k, v = wide[:, 8:264].unflatten(1, (2, 128)), wide[:, 512:768].unflatten(1, (2, 128))
    table = i32([0, 1, 77], dev)[None]
    pages = ops.KVPages.alloc(2, 2, dev, kv_format="q4")
    seq, pos = i32([0, -1, 0, 0, 1, 0], dev), i32([255, 3, 256, 600, 0, 5000], dev)            # rows 3 to 5: outside the pool, the table's slots, its pages
    ops.kv_write(k, v, seq, pos, table, pages)
    ko, vo = (torch.full((6, 2, 128), 5.0, device=dev, dtype=BF) for _ in range(2))
    ops.kv_read(seq, pos, table, pages, ko, vo)
    for x, got in ((k, ko), (v, vo)):
        assert torch.equal(got[[0, 2]].double(), entry(x[[0, 2]])[3])
        assert bool((got[[1, 3, 4, 5]] == 5).all())
    assert int((pages.k.flatten(2)[:, :, 17408:] != 0).sum()) == 4                             # two entries of two heads


@pytest.mark.parametrize("layers", [1, 3])
def test_kept_paths(dev, layers):
    from georefine_b200 import ops

    g = torch.Generator(device=dev).manual_seed(3)
    raw = [torch.randint(0, 256, (layers, 5, 3, 69, 256), generator=g, device=dev, dtype=torch.uint8) for _ in range(2)]
    pages = ops.KVPages(*raw)
    before = [x.clone() for x in raw]
    table = i32([4, 0], dev)[None].repeat(3, 1)
    table[1], table[2] = i32([2, 3], dev), i32([1, 1], dev)
    base, path, count = [250, 10, 0], [[0, 3, 4, 9], [0, 1, 7, -1], [0, 5, 6, 7]], [4, 3, 4]
    ops.kv_keep(i32([0, 1, -1], dev), i32(base, dev), torch.tensor(path, dtype=torch.int32, device=dev), i32(count, dev), table, pages)
    for x, was in zip(raw, before):
        for s in range(2):
            for i in range(1, count[s]):
                src, dst = base[s] + path[s][i], base[s] + i
                sp, dp = int(table[s, src // 256]), int(table[s, dst // 256])
                src, dst = src % 256, dst % 256
                for lo, width in ((0, 64), (16384, 4), (17408, 1)):
                    a, b = x.flatten(3)[:, dp, :, lo + width * dst:lo + width * (dst + 1)], was.flatten(3)[:, sp, :, lo + width * src:lo + width * (src + 1)]
                    assert torch.equal(a, b)
                    was.flatten(3)[:, dp, :, lo + width * dst:lo + width * (dst + 1)] = b.clone()      # (paths ascend: later sources lie behind)
        assert torch.equal(x, was)


def test_every_scale_and_code_reads_as_it_should(dev):
    """All bytes of a scale with all nibbles, at the ends of the exponents: what kv_read gives is the definition's number."""
    from georefine_b200 import ops

    pages = ops.KVPages.alloc(4, 1, dev, kv_format="q4")
    flat = pages.k.view(4, -1)
    for p, exp in enumerate((0, 87, 130, 149)):
        flat[p, :16384] = (torch.arange(16384, device=dev) * 37 % 256).to(torch.uint8)
        flat[p, 16384:17408] = (torch.arange(1024, device=dev) // 4).to(torch.uint8)          # position i: scale byte i
        flat[p, 17408:] = exp
    pages.v.copy_(pages.k)
    table = torch.arange(4, dtype=torch.int32, device=dev)[None]
    k, v = (torch.empty(1024, 1, 128, device=dev, dtype=BF) for _ in range(2))
    ops.kv_read(i32([0] * 1024, dev), i32(range(1024), dev), table, pages, k, v)
    codes = flat[:, :16384].reshape(1024, 16, 4)
    number = torch.empty(1024, 16, 8, dtype=torch.float64, device=dev)
    for byte, (lo, hi) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        number[..., lo], number[..., hi] = (codes[..., byte] % 16).double() - 8, (codes[..., byte] // 16).double() - 8
    byte = torch.arange(256, device=dev).double().repeat(4)
    scale = torch.where(byte < 16, byte / 8, (16 + byte % 16) * torch.exp2((byte // 16) - 4))
    unit = torch.exp2(torch.tensor([87, 87, 130, 149], device=dev).double() - 127 - 24).repeat_interleave(256)
    assert torch.equal(k.double().view(1024, 128), number.view(1024, 128) * (scale * unit)[:, None]) and torch.equal(k, v)
    assert float(GRID[0]) == 16 and float(GRID[-1]) == 63488
