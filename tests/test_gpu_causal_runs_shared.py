"""Long runs of causal rows beside other rows: what shares the call changes no bit of theirs (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_tree_attention import Setup, _causal, _i32  # noqa: E402


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("longest", [None, 100])
@pytest.mark.parametrize("beside", [1, 28, 100])
def test_a_run_of_100_rows_alone_and_beside_others(dev, fmt, longest, beside):
    s = Setup(dev, fmt, 10, 2, [150, 40], 2)
    seq, pos = [0] * 100 + [1] * beside, list(range(150, 250)) + list(range(40, 40 + beside))
    qkv = s.qkv(len(seq))
    out, solo = torch.empty(len(seq), 1280, device=dev, dtype=torch.bfloat16), torch.empty(100, 1280, device=dev, dtype=torch.bfloat16)
    attn = s.ops.TreeAttention(10, 2, len(seq), 2, dev, kv_format=fmt)
    attn(qkv, s.cos, s.sin, _i32(seq, dev), _i32(pos, dev), s.table, s.pages, out, longest_run=longest)
    for table in (s.table, s.table[:1]):
        attn(qkv[:100], s.cos, s.sin, _i32(seq[:100], dev), _i32(pos[:100], dev), table, s.pages, solo.zero_(), longest_run=longest)
        assert attn.check_status() == 0 and torch.equal(solo, out[:100])
    keep = [0, 1, 63, 98, 99, 100]
    s.check(qkv[keep], [seq[i] for i in keep], [pos[i] for i in keep], out[keep], _causal([pos[i] for i in keep]))
