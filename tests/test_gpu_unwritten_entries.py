"""Positions of a cache that nobody wrote: zeros where a row sees them, anything where it does not (needs a B200)."""
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


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("q_scale", [1.5, 12.0])
def test_empty_pages_that_a_row_sees_hold_zeros(dev, fmt, rows, q_scale):
    """Trees behind 300 positions of which 40 were written: the others are keys and values of zero, each of weight 1."""
    s = Setup(dev, fmt, 8, 2, [0], 2)
    for t in (s.pages.k, s.pages.v, s.pages.k_exp, s.pages.v_exp):
        if t is not None:
            t.view(torch.uint8).zero_()
    k, v = (torch.randn(40, 2, 128, generator=s.g, device=dev).to(BF) for _ in range(2))
    s.ops.kv_write(k, v, _i32([0] * 40, dev), _i32(range(0, 280, 7), dev), s.table, s.pages)
    qkv = s.qkv(rows, q_scale=q_scale)
    pos = torch.arange(300, 300 + rows, device=dev)
    out = torch.full((rows, 1024), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(8, 2, rows, 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out,
         tree=s.ops.TreeRows(_i32([300] * rows, dev), pos.int(), torch.tensor([[(1 << (i + 1)) - 1] for i in range(rows)], device=dev)))
    want, bound = _all_rows(s, qkv, pos, 0, torch.arange(512, device=dev) <= pos[:, None])
    off = ((out.view(rows, 8, 128).double() - want).abs() / bound).amax()
    assert attn.check_status() == 0 and float(off) <= 1


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
def test_causal_rows_with_places_between_them_that_hold_anything(dev, fmt):
    """Rows of one call at positions far apart: a row's answer is that of the positions up to its own."""
    s = Setup(dev, fmt, 4, 1, [20], 2)                 # (the places behind 20 hold NaN)
    qkv = s.qkv(3)
    out = torch.full((3, 512), float("nan"), device=dev, dtype=BF)
    attn = s.ops.TreeAttention(4, 1, 3, 2, dev, kv_format=fmt)
    pos = [20, 21, 100]
    attn(qkv, s.cos, s.sin, _i32([0] * 3, dev), _i32(pos, dev), s.table, s.pages, out)
    s.check(qkv[:2], [0, 0], pos[:2], out[:2], lambda r, p: p <= pos[r])
    assert bool(out[2].isnan().all())                  # (it sees the places that nobody wrote)
