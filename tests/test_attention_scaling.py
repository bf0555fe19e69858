"""What the attention of causal rows and draft trees refuses of its scores' scale, without a GPU."""
import ctypes

import pytest

pytest.importorskip("torch")

from georefine_b200 import _native  # noqa: E402

P = 1 << 20           # stands for device memory: aligned, never touched


@pytest.mark.parametrize("scaling", [0.0, -0.0, -0.088, float("inf"), float("nan")])
def test_a_scale_that_is_not_positive(scaling):
    """The wide kernel takes a row's maximum before it multiplies: only a positive scale keeps the order."""
    s = _native.TreeStep()
    pages = _native.KvPages(k=P, v=P, k_exp=P, v_exp=P, layers=1, pages=4, nkv=2, format=1)
    table = _native.KvTable(table=P, ld=4, slots=2, max_pages=4)
    for name, value in dict(qkv=P, ldq=1536, cos_table=P, sin_table=P, rope_rows=1024, row_seq=P, row_pos=P, scratch=P, scratch_bytes=1 << 40, out=P, ldo=1024, rows=0, nq=8,
                            head_dim=128, scaling=0.1, pages=pages, table=table).items():
        setattr(s, name, value)
    assert _native.lib().grb_attn_tree(ctypes.byref(s), None) == 0          # (no rows: nothing is launched)
    s.scaling = scaling
    assert _native.lib().grb_attn_tree(ctypes.byref(s), None) == 1
