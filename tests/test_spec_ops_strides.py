"""Distances between rows that the operators of speculative serving are given, without a GPU: what is launched is recorded, and tensors whose
rows overlap (expanded ones, whose rows are all the same memory) are turned away - their rows would be walked past their end."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, ops, sampling  # noqa: E402

BF, I32 = torch.bfloat16, torch.int32
CPU = torch.device("cpu")


@pytest.fixture
def launched(monkeypatch):
    calls = []
    monkeypatch.setattr(ops, "_launch", lambda device, name, *args: calls.append((name, args)))
    return calls


def _pages(kv_heads=2):
    p = object.__new__(ops.KVPages)              # (as on a device: addresses are recorded, not followed)
    p.device, p.stacked, p.kv_heads, p.pages, p.format = CPU, False, kv_heads, 4, "bf16"
    p._fields = (1 << 20, 1 << 20, 0, 0, 0, 0, 1, 4, kv_heads, 0)
    p._packed = _native.KV_PAGES.pack(*p._fields)
    return p


def _overlapping(t):
    """Views of t's shape whose rows are one row, or begin inside the row before."""
    yield t[:1].expand(t.shape)
    yield t.flatten().as_strided(t.shape, (t[0].numel() // 2,) + t.stride()[1:])


def test_overlapping_rows_are_refused(launched):
    rows, table, seq = 4, torch.zeros(2, 4, dtype=I32), torch.zeros(4, dtype=I32)
    kv = torch.zeros(rows, 2, 128, dtype=BF)
    for call, first in ((lambda k, v: ops.kv_write(k, v, seq, seq, table, _pages()), "keys"), (lambda k, v: ops.kv_read(seq, seq, table, _pages(), k, v), "keys")):
        call(kv, kv)
        for bad in _overlapping(kv):
            with pytest.raises(ValueError, match="keys.*overlap"):
                call(bad, kv)
            with pytest.raises(ValueError, match="values.*overlap"):
                call(kv, bad)
    path = torch.zeros(rows, 6, dtype=I32)
    ops.kv_keep(seq, seq, path, seq, table, _pages())
    for bad in _overlapping(path):
        with pytest.raises(ValueError, match="path.*overlap"):
            ops.kv_keep(seq, seq, bad, seq, table, _pages())
    attn = ops.TreeAttention(4, 2, 8, 4, "cpu")
    qkv, out, cos = torch.zeros(rows, 1024, dtype=BF), torch.zeros(rows, 512, dtype=BF), torch.zeros(64, 128, dtype=BF)
    go = lambda qkv=qkv, out=out, tree=None: attn(qkv, cos, cos, seq, seq, table, _pages(), out, tree=tree)
    go()
    for bad in _overlapping(qkv):
        with pytest.raises(ValueError, match="qkv.*overlap"):
            go(qkv=bad)
    for bad in _overlapping(out):
        with pytest.raises(ValueError, match="out.*overlap"):
            go(out=bad)
    for words in (1, 3):
        mask = torch.ones(rows, words, dtype=torch.int64)
        go(tree=ops.TreeRows(seq, seq, mask))
        with pytest.raises(ValueError, match="mask.*overlap"):
            ops.TreeRows(seq, seq, mask[:1].expand(rows, words))
    v = sampling.DraftVerifier(8, 2, 4, "cpu")
    u, starts = torch.zeros(rows), torch.tensor([0, 2, 4], dtype=I32)
    logits, q = torch.zeros(rows, 10), torch.zeros(rows, 10)
    check = lambda logits=logits, q=q: v(logits, seq, starts, u, torch.zeros(2), draft_probs=q)
    check()
    for bad in _overlapping(logits):
        with pytest.raises(ValueError, match="logits.*overlap"):
            check(logits=bad)
        with pytest.raises(ValueError, match="draft_probs.*overlap"):
            check(q=bad)
    assert [name for name, _ in launched] == ["grb_kv_write", "grb_kv_read", "grb_kv_keep"] + ["grb_attn_tree"] * 3 + ["grb_verify_drafts"]


def test_the_distances_that_are_passed_on(launched):
    """Rows of a wider matrix keep its distance; a single row has none, whatever its stride says."""
    seq, table = torch.zeros(3, dtype=I32), torch.zeros(2, 9, dtype=I32)[:, :4]
    wide = torch.zeros(3, 5, 128, dtype=BF)
    ops.kv_write(wide[:, :2], wide[:, 3:], seq, seq, table, _pages())
    _, (pages, table_at, _, _, _, ldk, _, ldv, rows) = launched.pop()
    assert (ldk, ldv, rows) == (640, 640, 3) and _native.KV_TABLE.unpack(table_at)[1:] == (9, 2, 4)
    one = torch.zeros(256, dtype=BF).as_strided((1, 2, 128), (0, 128, 1))
    ops.kv_write(one, one, seq[:1], seq[:1], torch.zeros(4, dtype=I32).expand(1, 4), _pages())
    _, (pages, table_at, _, _, _, ldk, _, ldv, rows) = launched.pop()
    assert (ldk, ldv, rows) == (256, 256, 1) and _native.KV_TABLE.unpack(table_at)[1:] == (4, 1, 4)
    attn = ops.TreeAttention(4, 2, 8, 4, "cpu")
    qkv, out, cos, mask = torch.zeros(3, 2000, dtype=BF)[:, 6:1030], torch.zeros(3, 600, dtype=BF)[:, :512], torch.zeros(64, 128, dtype=BF), torch.ones(3, 4, dtype=torch.int64)
    attn(qkv, cos, cos, seq, seq, table, _pages(), out, tree=ops.TreeRows(seq, seq, mask[:, :2]))
    step = _native.TreeStep.from_buffer_copy(launched.pop()[1][0])
    assert (step.ldq, step.ldo, step.ldm, step.mask_words, step.table.ld, step.rows) == (2000, 600, 4, 2, 9, 3)
    v = sampling.DraftVerifier(8, 2, 4, "cpu")
    v(torch.zeros(3, 20)[:, :10], seq, torch.tensor([0, 3], dtype=I32), torch.zeros(3), torch.zeros(1), draft_probs=torch.zeros(3, 12)[:, 1:11])
    step = _native.VerifyStep.from_buffer_copy(launched.pop()[1][0])
    assert (step.ldl, step.ldq, step.rows, step.vocab) == (20, 12, 3, 10)
    assert not launched


def test_a_page_table_that_is_a_vector(launched):
    attn = ops.TreeAttention(4, 2, 8, 4, "cpu")
    seq = torch.zeros(2, dtype=I32)
    with pytest.raises(ValueError, match="page table"):
        attn(torch.zeros(2, 1024, dtype=BF), torch.zeros(64, 128, dtype=BF), torch.zeros(64, 128, dtype=BF), seq, seq, torch.zeros(4, dtype=I32), _pages(), torch.zeros(2, 512, dtype=BF))
    assert not launched
