"""Few rows behind long 4-bit contexts, whose parts are more than the lanes that merge them, against the definition in 64 bits (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from q4_reference import Setup, causal, i32  # noqa: E402

BF = torch.bfloat16


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.mark.parametrize("nq,nkv", [(5, 1), (4, 2), (16, 1)])
def test_rows_of_32_parts_and_more(dev, nq, nkv):
    """The 32nd part's last position, the 33rd's first, chains across that border, 64 parts and 65."""
    lengths, per = [16382, 16384, 16380, 20001, 32767, 32768], [2, 1, 9, 3, 1, 1]
    s = Setup(dev, nq, nkv, lengths, 130)
    seq = [i for i, n in enumerate(per) for _ in range(n)]
    pos = [lengths[i] + j for i, n in enumerate(per) for j in range(n)]
    rows = len(seq)
    qkv, out = s.qkv(rows), torch.full((rows, nq * 128), float("nan"), device=dev, dtype=BF)
    attn = s.attention(rows)
    attn(qkv, s.cos, s.sin, i32(seq, dev), i32(pos, dev), s.table, s.pages, out)
    s.check(qkv, seq, pos, out, causal(pos))
    solo = torch.empty(1, nq * 128, device=dev, dtype=BF)
    for r in (0, 1, 2, 5, 14, 16):
        attn(qkv[r:r + 1], s.cos, s.sin, i32(seq[r:r + 1], dev), i32(pos[r:r + 1], dev), s.table, s.pages, solo, longest_run=1)
        assert torch.equal(solo[0], out[r])
    assert attn.check_status() == 0


def test_a_position_of_weight_in_any_part_counts(dev):
    """One key, in one part after another, takes nearly all of the weight (a score of 28 where the others' are below 1, exp(27) / 33000): its value, whole
    numbers that an entry holds as they are, is the answer."""
    s = Setup(dev, 4, 1, [33000], 130, scale=0.01)
    attn, qkv = s.attention(1), s.qkv(1)
    qkv[:, :512] = 0
    qkv[:, :512].view(4, 128)[:, 63] = 8.0        # (the slowest pair: turned by 0.04 at the row's position)
    k, v = torch.zeros(1, 1, 128, device=dev, dtype=BF), torch.zeros(1, 1, 128, device=dev, dtype=BF)
    k[0, 0, 63], v[0, 0] = 40.0, torch.arange(128, device=dev) % 15 - 7
    for at in (5, 511, 512, 8000, 16383, 16384, 16900, 24000, 32767, 32768, 32999):
        place = i32([0], dev), i32([at], dev), s.table, s.pages
        before = [torch.empty(1, 1, 128, device=dev, dtype=BF) for _ in range(2)]
        s.ops.kv_read(*place, *before)
        s.ops.kv_write(k, v, *place)
        out = torch.empty(1, 512, device=dev, dtype=BF)
        attn(qkv, s.cos, s.sin, i32([0], dev), i32([33000], dev), s.table, s.pages, out)
        s.check(qkv, [0], [33000], out, causal([33000]))
        assert bool(((out.view(4, 128).float() - v[0].float()).abs() < 0.25).all())
        s.ops.kv_write(*before, *place)
    assert attn.check_status() == 0
