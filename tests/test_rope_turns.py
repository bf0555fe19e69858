"""Fractions of a turn that rotary positions are held in: the nearest multiple of 2^-64 to the formula's, so that an angle is off by
2^-65 of a turn a position.  By whole powers of what is held, which need neither exponentials nor logarithms.  No GPU."""
from decimal import Decimal, localcontext

import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import ops  # noqa: E402

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


def _ends(turns):
    """Frequencies, in radians, between which the exact one lies when ``turns`` is the nearest number of units of 2^-64."""
    t = Decimal(turns % (1 << 64))
    return (t - Decimal("0.5000001")) * 2 * PI / (1 << 64), (t + Decimal("0.5000001")) * 2 * PI / (1 << 64)


@pytest.mark.parametrize("dim,theta", [(2, 1e4), (10, 1e4), (64, 1e4), (80, 1e4), (96, 1e6), (128, 1e4), (128, 5e5), (128, 1e6), (128, 12345.678), (256, 1e7)])
@pytest.mark.parametrize("linear", [None, 3.0, 32.0])
def test_plain_and_linear(dim, theta, linear):
    rope = ops.Rope(dim, theta, scaling=None if linear is None else {"kind": "linear", "factor": linear}, device="cpu")
    with localcontext() as c:
        c.prec = 80
        for i, turns in enumerate(rope.turns.tolist()):
            lo, hi = (f * Decimal(linear or 1) for f in _ends(turns))
            assert lo ** dim <= 1 / Decimal(theta) ** (2 * i) <= hi ** dim, (i, turns)


@pytest.mark.parametrize("dim,theta,factor", [(64, 1e4, 8.0), (128, 1e6, 4.0), (96, 1e4, 2.5)])
def test_a_larger_base(dim, theta, factor):
    """f^dim = (theta factor^(dim / (dim - 2)))^(-2 i), both sides to the power dim - 2."""
    rope = ops.Rope(dim, theta, scaling={"kind": "ntk", "factor": factor}, device="cpu")
    with localcontext() as c:
        c.prec = 80
        for i, turns in enumerate(rope.turns.tolist()):
            lo, hi = _ends(turns)
            want = 1 / (Decimal(theta) ** (dim - 2) * Decimal(factor) ** dim) ** (2 * i)
            assert lo ** (dim * (dim - 2)) <= want <= hi ** (dim * (dim - 2)), (i, turns)


@pytest.mark.parametrize("kind", ["yarn", "bands"])
def test_ramps(kind):
    """Between the plain pair's frequency and the slow one's at the share that the formula gives, worked out in 60 digits."""
    dim, theta, factor, original = 128, 1e6, 16.0, 4096.0
    more = {"yarn": {}, "bands": {"low": 1.0, "high": 4.0}}[kind]
    rope = ops.Rope(dim, theta, scaling={"kind": kind, "factor": factor, "original": original, **more}, device="cpu")
    with localcontext() as c:
        c.prec = 60
        plain = [(-Decimal(theta).ln() * 2 * i / dim).exp() for i in range(dim // 2)]
        if kind == "yarn":
            number = lambda turns: Decimal(dim) / 2 * (Decimal(original) / (2 * PI * turns)).ln() / Decimal(theta).ln()
            lo, hi = int(number(32)), int(number(1)) + 1           # (both positive, and no whole numbers)
            slow = [min(max(Decimal(i - lo) / (hi - lo), Decimal(0)), Decimal(1)) for i in range(dim // 2)]
            assert sum(0 < s < 1 for s in slow) > 5
        else:
            slow = [1 - min(max((Decimal(original) * f / (2 * PI) - 1) / 3, Decimal(0)), Decimal(1)) for f in plain]
            assert sum(0 < s < 1 for s in slow) > 2
        for f, s, turns in zip(plain, slow, rope.turns.tolist()):
            lo, hi = _ends(turns)
            assert lo <= f * (1 - s) + f * s / Decimal(factor) <= hi
        for f, s, got in zip(plain, slow, rope.frequencies):
            assert abs(Decimal(got) / (f * (1 - s) + f * s / Decimal(factor)) - 1) < Decimal(2) ** -52


def test_more_than_a_turn_a_position():
    with localcontext() as c:
        c.prec = 60
        turns = ops.Rope(2, 1e4, scaling={"kind": "linear", "factor": 2.0 ** -40}, device="cpu").turns.item()
        want = Decimal(2) ** 40 / (2 * PI)
        assert abs(Decimal(turns % (1 << 64)) - (want - int(want)) * (1 << 64)) <= Decimal("0.5000001")
