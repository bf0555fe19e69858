"""Rotary positions in every layout, part, scaling and type, against the formula in 64 bits (needs a B200)."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

SCALINGS = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 8.0}, "yarn": {"kind": "yarn", "factor": 16.0, "original": 4096},
            "bands": {"kind": "bands", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _definition(x, positions, rope, backward=False):
    """The formula, and a bound on the kernel's error: the result's rounding (half a step), cosine and sine 2^-22 off (their own rounding, the
    rounded angle, the factor's product), and two roundings of 2^-24 of the sums."""
    inv = torch.tensor(rope.frequencies, dtype=torch.float64, device=x.device)
    angle = positions.double()[:, None] * inv
    c, s = (f(angle)[:, None] * rope.factor for f in (torch.cos, torch.sin))
    s = -s if backward else s
    y, n = x.double(), rope.dim
    a, b = (slice(0, n // 2), slice(n // 2, n)) if rope.layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    p, q, out = y[..., a], y[..., b], y.clone()
    out[..., a], out[..., b] = p * c - q * s, q * c + p * s
    size = torch.zeros_like(y)
    size[..., a] = size[..., b] = (p.abs() + q.abs()) * rope.factor
    # (the product of a position and a frequency of 53 bits is itself off by |position| 2^-52 here, and 2^-34 for the frequency's 64 bits there)
    loose = 2.0 ** -22 + 2.0 ** -23 + positions.abs().double()[:, None, None] * 2.0 ** -51
    return out, torch.finfo(x.dtype).eps / 2 * out.abs() * (size > 0) + loose * size * (1 + torch.finfo(x.dtype).eps) + (size > 0) * torch.finfo(x.dtype).smallest_normal


def _check(x, positions, rope, got, backward=False):
    want, bound = _definition(x, positions, rope, backward)
    assert bool(((got.double() - want).abs() <= bound).all()), float((((got.double() - want).abs() - bound).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,dim,turned", [(1, 2, 2), (3, 64, 64), (6, 80, 20), (5, 96, 48), (9, 128, 128), (2, 128, 64), (4, 256, 6), (1, 7, 4), (2, 1024, 1024), (3, 1000, 998)])
def test_sizes_layouts_and_types(dev, dtype, layout, heads, dim, turned):
    from georefine_b200 import ops

    rope = ops.Rope(turned, 1e4, layout=layout, device=dev)
    g = torch.Generator(device=dev).manual_seed(dim + turned)
    for rows in (1, 37):
        x = torch.randn(rows, heads, dim, generator=g, device=dev).to(dtype)
        positions = torch.randint(0, 5000, (rows,), generator=g, device=dev)
        positions[0] = 0
        for pos in (positions.int(), positions):
            out = torch.empty_like(x)
            assert ops.rotary(x, pos, rope, out=out) is out
            _check(x, positions, rope, out)
            assert torch.equal(out[..., turned:], x[..., turned:])
            assert torch.equal(out[0], x[0])                                 # position 0
        place = x.clone()
        ops.rotary(place, positions.int(), rope)
        assert torch.equal(place, out)
        back = torch.empty_like(x)
        ops.rotary(x, positions, rope, out=back, backward=True)
        _check(x, positions, rope, back, backward=True)


@pytest.mark.parametrize("name", SCALINGS)
def test_scalings_and_far_positions(dev, name):
    """Positions from the far negative to 2^31, where an angle in 32 bits would mean nothing."""
    from georefine_b200 import ops

    rope = ops.Rope(128, 1e6, scaling=SCALINGS[name], device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    positions = torch.tensor([0, 1, -1, 4095, 100000, -99999, 1 << 20, (1 << 31) - 1, -(1 << 31), 12345678], device=dev)
    x = torch.randn(10, 4, 128, generator=g, device=dev)
    out = torch.empty_like(x)
    ops.rotary(x, positions, rope, out=out)
    _check(x, positions, rope, out)
    small = torch.empty_like(x)
    ops.rotary(x, positions.int(), rope, out=small)
    assert torch.equal(small, out)
    assert bool((out[2] - out[1]).abs().max() > 0.1)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_alignments(dev, layout):
    """Heads of rows that are wider than they, odd distances and addresses, a broadcast input; nothing beside the heads is touched."""
    from georefine_b200 import ops

    rope = ops.Rope(64, 1e4, layout=layout, device=dev)
    for start, width, head in ((0, 1024, 96), (1, 1001, 97), (2, 1002, 98), (8, 1024, 104)):
        buffer = torch.randn(6, width, device=dev).to(torch.bfloat16)
        x = torch.as_strided(buffer, (6, 9, 96), (width, head, 1), start)
        was, kept = x.clone(), buffer.clone()
        positions = torch.arange(100, 106, device=dev).int()
        ops.rotary(x, positions, rope)
        _check(was, positions, rope, x)
        torch.as_strided(kept, (6, 9, 96), (width, head, 1), start).copy_(x)
        assert torch.equal(kept, buffer)
    one = torch.randn(1, 1, 96, device=dev)
    out = torch.empty(5, 3, 96, device=dev)
    ops.rotary(one.expand(5, 3, 96), torch.arange(5, device=dev), rope, out=out)
    _check(one.expand(5, 3, 96).contiguous(), torch.arange(5, device=dev), rope, out)
    by_head = torch.randn(3, 7, 96, device=dev)                              # heads outside, rows inside
    got = torch.empty(3, 7, 96, device=dev)
    ops.rotary(by_head.transpose(0, 1), torch.arange(7, device=dev), rope, out=got.transpose(0, 1))
    _check(by_head.transpose(0, 1).contiguous(), torch.arange(7, device=dev), rope, got.transpose(0, 1).contiguous())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("scaling", ["none", "yarn"])
def test_backward_is_the_gradient(dev, layout, scaling):
    """Against differences of the forward pass along random directions, and <R x, y> = <x, R' y>."""
    from georefine_b200 import ops

    rope = ops.Rope(96, 1e4, layout=layout, scaling=SCALINGS[scaling], device=dev)
    g = torch.Generator(device=dev).manual_seed(2)
    x, y, d = (torch.randn(11, 3, 128, generator=g, device=dev) for _ in range(3))
    positions = torch.randint(-3000, 3000, (11,), generator=g, device=dev).int()
    turn = lambda t, **kw: ops.rotary(t, positions, rope, out=torch.empty_like(t), **kw)
    gradient = turn(y, backward=True).double()
    # the loss <R x, y> is linear: its difference along d over a step of 1 is the derivative, to the roundings of 4224 products of two factors of 2^-21
    slope = ((turn(x + d).double() - turn(x).double()) * y.double()).sum()
    size = (d.abs().double() * y.abs().double()).sum() + ((x.abs() + d.abs()) * y.abs()).double().sum()
    assert abs(float(slope - (gradient * d.double()).sum())) <= 8 * 2.0 ** -21 * float(size) * rope.factor
    there = turn(turn(x), backward=True)
    scale = torch.ones(128, device=dev)
    scale[:96] = rope.factor ** 2                 # (dimensions that do not turn are left as they are)
    assert bool(((there - x * scale).abs() <= 2.0 ** -19 * scale * 4 * x.abs().amax()).all())


def test_a_captured_call_and_another_stream(dev):
    from georefine_b200 import ops

    rope = ops.Rope(128, 1e4, device=dev)
    x, positions, out = torch.randn(4, 8, 128, device=dev).to(torch.bfloat16), torch.arange(4, device=dev).int(), torch.empty(4, 8, 128, device=dev, dtype=torch.bfloat16)
    ops.rotary(x, positions, rope, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rotary(x, positions, rope, out=out)
    for _ in range(2):
        x.normal_()
        positions.add_(1000)
        graph.replay()
    _check(x, positions, rope, out)
    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        other = ops.rotary(x, positions, rope, out=torch.empty_like(x))
    stream.synchronize()
    assert torch.equal(other, out)


def test_the_attention_s_tables_and_the_rotation_agree(dev):
    """`Rope.tables` are the cosines and sines of the call, rounded to BF16."""
    from georefine_b200 import ops

    rope = ops.Rope(128, 1e6, scaling=SCALINGS["yarn"], device=dev)
    cos, sin = rope.tables(3000)
    x = torch.zeros(3000, 1, 128, device=dev)
    x[..., :64] = 1.0
    got = ops.rotary(x, torch.arange(3000, device=dev), rope)
    for table, part in ((cos, got[:, 0, :64]), (sin, got[:, 0, 64:])):
        assert torch.equal(table[:, :64], table[:, 64:])
        assert bool(((table[:, :64].double() - part.double()).abs() <= 2.0 ** -8 * part.abs().double() + 2.0 ** -20).all())
    assert math.isclose(rope.factor, 0.1 * math.log(16) + 1)
