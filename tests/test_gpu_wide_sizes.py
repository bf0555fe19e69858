"""Entries of very different sizes in one part of a cache, where many rows of a sequence are multiplied together: what a row does not see, or
hardly weighs, takes nothing from the values that it does (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_prompt_rows import _all_rows  # noqa: E402
from test_gpu_tree_attention import BF, Setup, _i32  # noqa: E402


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _context(s, n, key_size, value_size, dev):
    """Positions 0 .. n - 1 of sequence 0."""
    k, v = (size * torch.randn(n, s.nkv, 128, generator=s.g, device=dev) for size in (key_size, value_size))
    return k.to(BF), v.to(BF)


def _store(s, k, v, dev):
    s.ops.kv_write(k, v, _i32([0] * len(k), dev), _i32(range(len(k)), dev), s.table, s.pages)


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("value_size", [1e-4, 1e-7, 1e-8])
@pytest.mark.parametrize("key_size", [1.0, 1e-6])
def test_a_node_that_few_rows_see(dev, fmt, key_size, value_size):
    """One node's key and value are as large as 8 bits hold; only its children see it."""
    n, rows = 300, 40
    s = Setup(dev, fmt, 8, 2, [0], 2)
    _store(s, *_context(s, n, key_size, value_size, dev), dev)
    parents = [-1] + [(i * 5) // 7 for i in range(rows - 1)]
    depth, masks = s.ops.TreeRows.masks(parents)
    qkv = s.qkv(rows, q_scale=1.0 if key_size == 1.0 else 1e3)
    qkv[:, 8 * 128:10 * 128] *= key_size
    qkv[:, 10 * 128:] *= value_size
    qkv[5, 8 * 128:10 * 128] *= 1e-3 / key_size
    qkv[5, 10 * 128:] = (qkv[5, 10 * 128:] / value_size).sign() * 5e4
    out = torch.full((rows, 1024), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, rows, 2, dev, kv_format=fmt)
    rope = torch.tensor([n + d for d in depth], device=dev)
    attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), _i32(range(n, n + rows), dev), s.table, s.pages, out,
         tree=s.ops.TreeRows(_i32([n] * rows, dev), rope.int(), torch.tensor(masks, device=dev)))
    places = torch.arange(512, device=dev)
    bits = torch.tensor([[m[0] >> j & 1 for j in range(64)] for m in masks], device=dev).bool()
    seen = (places < n) | ((places >= n) & (places < n + 64) & bits[:, (places - n).clamp(0, 63)])
    want, bound = _all_rows(s, qkv, rope, 0, seen)
    assert attn.check_status() == 0 and bool(((out.view(rows, 8, 128).double() - want).abs() <= bound).all())
    small = want.abs().amax((1, 2)) < 10 * value_size
    assert 10 < int(small.sum()) < rows


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("rows", [70, 76])
def test_a_position_that_hardly_counts(dev, fmt, rows):
    """A large value whose score is some 60 below the others', beside values of 1e-8, under causal rows."""
    n = 500
    s = Setup(dev, fmt, 5, 1, [0], 3)
    k, v = _context(s, n, 0.05, 1e-8, dev)
    direction = torch.randn(128, generator=s.g, device=dev).sign()
    k[130, 0], v[130, 0] = -8.0 * direction, 5e4
    _store(s, k, v, dev)
    # keys as they are; queries that the rotation leaves along `direction`: turned back by the same angles first
    pos = torch.arange(n, n + rows, device=dev)
    cos, sin = s.cos[pos].double()[:, None, :64], s.sin[pos].double()[:, None, :64]
    q = direction.double().expand(rows, 5, 128)
    q = torch.cat([q[..., :64] * cos + q[..., 64:] * sin, q[..., 64:] * cos - q[..., :64] * sin], dim=2)
    qkv = s.qkv(rows)
    qkv[:, :640] = (0.7 * q).reshape(rows, 640).to(BF)
    qkv[:, 640:768] *= 0.05
    qkv[:, 768:] *= 1e-8
    out = torch.full((rows, 640), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(5, 1, rows, 3, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out, longest_run=rows)
    want, bound = _all_rows(s, qkv, pos, 0, torch.arange(768, device=dev) <= pos[:, None])
    assert float(want.abs().max()) < 1e-6
    assert attn.check_status() == 0 and bool(((out.view(rows, 5, 128).double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("scale", [1e-7, 1e3, 0.0])
def test_sizes_that_differ_between_positions(dev, fmt, scale):
    n, rows = 300, 70
    s = Setup(dev, fmt, 8, 2, [0], 2)
    k, v = _context(s, n, 1.0, 1.0, dev)
    powers = torch.exp2(torch.randint(-20, 3, (n, 1, 1), generator=s.g, device=dev).float())
    _store(s, k, (v * powers * scale).to(BF), dev)
    qkv = s.qkv(rows)
    qkv[:, 10 * 128:] *= scale
    pos = torch.arange(n, n + rows, device=dev)
    out = torch.full((rows, 1024), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, rows, 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out, longest_run=rows)
    want, bound = _all_rows(s, qkv, pos, 0, torch.arange(512, device=dev) <= pos[:, None])
    assert attn.check_status() == 0 and bool(((out.view(rows, 8, 128).double() - want).abs() <= bound).all())


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_nan_and_infinity_among_many_rows(dev, fmt):
    """A key and a value that are not finite: the rows that see them, and those alone."""
    n, rows = 200, 70
    s = Setup(dev, fmt, 8, 2, [0], 2)
    _store(s, *_context(s, n, 1.0, 1.0, dev), dev)
    pos = torch.arange(n, n + rows, device=dev)
    out = torch.empty(rows, 1024, device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, rows, 2, dev, kv_format=fmt)
    for at, value in ((8 * 128 + 5, "nan"), (11 * 128 + 5, "inf")):
        qkv = s.qkv(rows)
        qkv[33, at] = float(value)
        attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out, longest_run=rows)
        bad = (~torch.isfinite(out.float())).view(rows, 2, 4, 128).any(-1).any(-1)
        head = 0 if value == "nan" else 1
        assert bad[:, head].tolist() == [r >= 33 for r in range(rows)] and not bool(bad[:, 1 - head].any())
    # a query that is not finite: its head alone
    qkv = s.qkv(rows)
    qkv[7, 3 * 128] = float("inf")
    attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out, longest_run=rows)
    bad = (~torch.isfinite(out.float())).view(rows, 8, 128).any(-1)
    assert bool(bad[7, 3]) and int(bad.sum()) == 1
