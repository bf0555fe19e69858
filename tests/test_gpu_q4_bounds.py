"""How far values that went through a 4-bit cache may be from what was stored, groups of any size (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from q4_bounds import bound, inputs  # noqa: E402
from q4_reference import i32  # noqa: E402


def test_rows_in_and_out():
    from georefine_b200 import ops

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    dev, n = torch.device("cuda:0"), 1024
    k, v = (inputs(dev, n * 3, seed).view(n, 3, 128) for seed in (1, 2))
    pages = ops.KVPages.alloc(4, 3, dev, kv_format="q4")
    table, seq, pos = i32([2, 0, 3, 1], dev)[None], i32([0] * n, dev), i32(range(n), dev)
    ops.kv_write(k, v, seq, pos, table, pages)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    ops.kv_read(seq, pos, table, pages, ko, vo)
    for x, got in ((k, ko), (v, vo)):
        assert bool(((got.double() - x.double()).abs() <= bound(x)).all())
