"""How far a 4-bit entry's values may be from what was stored, by the definition.  No GPU."""
import pytest

torch = pytest.importorskip("torch")

from q4_bounds import bound, inputs  # noqa: E402
from q4_reference import entry  # noqa: E402


@pytest.mark.parametrize("seed", range(4))
def test_values_of_any_entry(seed):
    x = inputs("cpu", 4000, seed)
    off = (entry(x)[3] - x.double()).abs()
    assert bool((off <= bound(x)).all())
    groups = x.double().unflatten(-1, (4, 32))
    g, a = groups.abs().amax(-1), groups.abs().amax((-2, -1))[:, None]
    share = off.unflatten(-1, (4, 32)).amax(-1) / g
    usual = (a < 1e5) & (a > 2.0 ** -40)
    assert float(share[(g >= a * 2.0 ** -11) & usual].max()) <= 1 / 14 * (1 + 2.0 ** -5)
    # a fourteenth of the group does not bound the groups that are smaller: 16 units are their smallest scale, and half of it is more than a / 57344
    assert float(share[(g < a * 2.0 ** -12) & usual].max()) > 0.2 and float(share[(g < a * 2.0 ** -16) & usual].min()) == 1.0


def test_values_beyond_the_largest_power():
    x = torch.tensor([1.0, 111104.0, 131072.0, -3.0e38] * 32, dtype=torch.bfloat16)
    value = entry(x)[3]
    assert value[1::4].eq(111104.0).all() and value[2::4].eq(111104.0).all() and value[3::4].eq(-111104.0).all()
