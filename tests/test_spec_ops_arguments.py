"""Refusals of the operators of speculative serving, without a GPU: every call here is turned away before anything is launched."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, ops, sampling  # noqa: E402

ARGUMENT, UNSUPPORTED, WORKSPACE = 1, 2, 3
P = 1 << 20           # stands for device memory: aligned, never touched


def _pages(**kw):
    d = dict(k=P, v=P, k_exp=P, v_exp=P, layer_stride=0, exp_stride=0, layers=1, pages=4, nkv=2, format=1)
    d.update(kw)
    return _native.KvPages(**d)


def _table(**kw):
    d = dict(table=P, ld=4, slots=2, max_pages=4)
    d.update(kw)
    return _native.KvTable(**d)


BAD_PAGES = [(dict(k=None), ARGUMENT), (dict(v=None), ARGUMENT), (dict(k_exp=None), ARGUMENT), (dict(format=0), ARGUMENT), (dict(format=2), UNSUPPORTED),
             (dict(layers=0), ARGUMENT), (dict(pages=0), ARGUMENT), (dict(nkv=0), ARGUMENT), (dict(k=P + 8), ARGUMENT), (dict(v_exp=P + 4), ARGUMENT),
             (dict(layers=2, layer_stride=100), ARGUMENT), (dict(layers=2, layer_stride=4 * 2 * 256 * 128, exp_stride=1), ARGUMENT), (dict(pages=1 << 30), UNSUPPORTED),
             (dict(nkv=5000), UNSUPPORTED)]
BAD_TABLES = [(dict(table=None), ARGUMENT), (dict(slots=0), ARGUMENT), (dict(max_pages=0), ARGUMENT), (dict(ld=3), ARGUMENT), (dict(max_pages=1 << 24, ld=1 << 24), UNSUPPORTED)]


@pytest.mark.parametrize("name", ["grb_kv_write", "grb_kv_read"])
def test_rows(name):
    call = getattr(_native.lib(), name)
    go = lambda pages=None, table=None, seq=P, pos=P, k=P, ldk=256, v=P, ldv=256, rows=3: call(pages or _pages(), table or _table(), seq, pos, k, ldk, v, ldv, rows, None)
    for kw, status in BAD_PAGES:
        assert go(pages=_pages(**kw)) == status, kw
    for kw, status in BAD_TABLES:
        assert go(table=_table(**kw)) == status, kw
    for kw in (dict(seq=None), dict(pos=None), dict(k=None), dict(v=None), dict(ldk=255), dict(ldv=128), dict(ldk=258), dict(k=P + 2)):
        assert go(**kw) == ARGUMENT, kw
    assert call(None, _table(), P, P, P, 256, P, 256, 3, None) == ARGUMENT
    assert go(rows=0) == 0                        # nothing to do, and nothing launched


def test_keep():
    call = _native.lib().grb_kv_keep
    go = lambda pages=None, table=None, seqs=P, base=P, path=P, ldp=4, count=P, n=2, width=4: call(pages or _pages(), table or _table(), seqs, base, path, ldp, count, n, width, None)
    for kw, status in BAD_PAGES:
        assert go(pages=_pages(**kw)) == status, kw
    for kw in (dict(seqs=None), dict(base=None), dict(path=None), dict(count=None), dict(ldp=3)):
        assert go(**kw) == ARGUMENT, kw
    assert go(n=70000) == UNSUPPORTED
    assert go(n=0) == 0 and go(width=1) == 0


def _tree(**kw):
    s = _native.TreeStep()
    d = dict(qkv=P, ldq=1536, cos_table=P, sin_table=P, rope_rows=1024, row_seq=P, row_pos=P, scratch=P, scratch_bytes=1 << 40, out=P, ldo=1024, rows=3, nq=8, head_dim=128,
             scaling=0.1, pages=_pages(), table=_table())
    d.update(kw)
    for name, value in d.items():
        setattr(s, name, value)
    return s


def test_attention():
    call = _native.lib().grb_attn_tree
    tree = dict(row_base=P, row_rope=P, row_mask=P, ldm=1, mask_words=1)
    for kw, status in ([(dict([(n, None)]), ARGUMENT) for n in ("qkv", "cos_table", "sin_table", "row_seq", "row_pos", "scratch", "out")] +
                       [(dict(nq=0), ARGUMENT), (dict(nq=7), ARGUMENT), (dict(nq=64, ldq=1 << 20, ldo=1 << 20), UNSUPPORTED), (dict(head_dim=64), ARGUMENT), (dict(rope_rows=0), ARGUMENT),
                        (dict(rows=4097), UNSUPPORTED), (dict(ldq=1535), ARGUMENT), (dict(ldq=1537), ARGUMENT), (dict(ldo=1000), ARGUMENT), (dict(out=P + 4), ARGUMENT),
                        (dict(qkv=P + 2), ARGUMENT), (dict(scratch=P + 8), ARGUMENT), (dict(scratch_bytes=1000), WORKSPACE),
                        (dict(tree, row_rope=None), ARGUMENT), (dict(tree, row_mask=None), ARGUMENT), (dict(tree, mask_words=0), ARGUMENT), (dict(tree, mask_words=5, ldm=5), UNSUPPORTED),
                        (dict(tree, ldm=0), ARGUMENT), (dict(tree, row_mask=P + 4), ARGUMENT)] +
                       [(dict(pages=_pages(**k)), st) for k, st in BAD_PAGES] + [(dict(table=_table(**k)), st) for k, st in BAD_TABLES]):
        assert call(_tree(**kw), None) == status, kw
    assert call(None, None) == ARGUMENT
    assert call(_tree(rows=0), None) == 0
    size = _native.lib().grb_attn_tree_scratch_bytes
    assert size(1, 8, 4, 1) > 0 and size(4096, 8, 4, 0) > size(1, 8, 4, 0)
    assert size(0, 8, 4, 1) == size(4097, 8, 4, 1) == size(1, 0, 4, 1) == size(1, 8, 0, 1) == size(1, 8, 4, 2) == 0


def test_verification():
    call = _native.lib().grb_verify_drafts

    def step(**kw):
        s = _native.VerifyStep()
        d = dict(logits=P, ldl=1000, tokens=P, starts=P, u_keep=P, u_draw=P, stats=P, out_tokens=P, out_rows=P, out_count=P, rows=6, seqs=2, vocab=1000, width=6, temperature=1.0)
        d.update(kw)
        for name, value in d.items():
            setattr(s, name, value)
        return s

    for kw, status in ([(dict([(n, None)]), ARGUMENT) for n in ("logits", "tokens", "starts", "u_keep", "u_draw", "stats", "out_tokens", "out_rows", "out_count")] +
                       [(dict(vocab=0), ARGUMENT), (dict(width=0), ARGUMENT), (dict(ldl=999), ARGUMENT), (dict(temperature=0.0), ARGUMENT), (dict(temperature=-1.0), ARGUMENT),
                        (dict(temperature=float("nan")), ARGUMENT), (dict(temperature=float("inf")), ARGUMENT), (dict(dtype=2), ARGUMENT), (dict(stats=P + 8), ARGUMENT),
                        (dict(draft_probs=P, ldq=1000, parent=P), ARGUMENT), (dict(draft_probs=P, ldq=999), ARGUMENT), (dict(vocab=600000, ldl=600000), UNSUPPORTED),
                        (dict(width=257), UNSUPPORTED), (dict(rows=70000), UNSUPPORTED), (dict(seqs=70000), UNSUPPORTED), (dict(rows=0), ARGUMENT)]):
        assert call(step(**kw), None) == status, kw
    assert call(None, None) == ARGUMENT and call(step(seqs=0), None) == 0


def test_python_refusals_before_the_library_is_called():
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVPages.alloc(2, 2, "cpu")
    with pytest.raises(ValueError, match="format"):
        ops.KVPages.alloc(2, 2, "cpu", kv_format="int4")
    with pytest.raises(ValueError, match="256, 128"):
        ops.KVPages(torch.zeros(2, 2, 256, 64), torch.zeros(2, 2, 256, 64))
    for args in ((5, 2), (34, 2), (0, 1)):
        with pytest.raises(ValueError, match="heads"):
            ops.TreeAttention(*args, 4, 4, "cpu")
    for rows, pages in ((0, 4), (4097, 4), (4, 0)):
        with pytest.raises(ValueError, match="rows"):
            ops.TreeAttention(4, 2, rows, pages, "cpu")
    with pytest.raises(ValueError, match="format"):
        ops.TreeAttention(4, 2, 4, 4, "cpu", kv_format="fp8")
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)
    with pytest.raises(ValueError, match="mask"):
        ops.TreeRows(i32(3), i32(3), torch.zeros(3, 5, dtype=torch.int64))
    with pytest.raises(ValueError, match="mask"):
        ops.TreeRows(i32(3), i32(3), torch.zeros(3, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="rope"):
        ops.TreeRows(i32(3), i32(2), torch.zeros(3, 1, dtype=torch.int64))
    for args in ((0, 1, 4), (4, 0, 4), (4, 1, 0), (4, 1, 257)):
        with pytest.raises(ValueError):
            sampling.DraftVerifier(*args, "cpu")
    v = sampling.DraftVerifier(8, 2, 4, "cpu")
    f32 = lambda *n: torch.zeros(*n, dtype=torch.float32)
    good = dict(logits=f32(6, 10), tokens=i32(6), starts=i32(3), u_keep=f32(6), u_draw=f32(2))
    call = lambda temperature=1.0, parent=None, draft_probs=None, **kw: v(*{**good, **kw}.values(), temperature=temperature, parent=parent, draft_probs=draft_probs)
    for bad in (dict(logits=f32(9, 10)), dict(logits=f32(6, 10).double()), dict(logits=f32(10, 6).T), dict(starts=i32(4)), dict(starts=i32(0)), dict(tokens=i32(5)),
                dict(tokens=torch.zeros(6, dtype=torch.int64)), dict(u_keep=f32(5)), dict(u_draw=f32(3)), dict(u_keep=f32(12)[::2]), dict(temperature=0.0), dict(parent=i32(5)),
                dict(parent=i32(6), draft_probs=f32(6, 10)), dict(draft_probs=f32(6, 11)), dict(draft_probs=f32(6, 10).to(torch.bfloat16))):
        with pytest.raises(ValueError):
            call(**bad)
    tokens, rows, count = call(starts=i32(1), u_draw=f32(0))          # no sequences: nothing to do
    assert tokens.shape == rows.shape == (0, 4) and count.shape == (0,)


def test_masks_of_a_tree():
    depth, masks = ops.TreeRows.masks([-1, 0, 0, 1, 3])
    assert depth == [0, 1, 1, 2, 3] and masks == [[1], [3], [5], [11], [27]]
    depth, masks = ops.TreeRows.masks([-1] + list(range(64)))         # a chain of 65 nodes: two words, the first full
    assert depth == list(range(65)) and masks[63] == [-1, 0] and masks[64] == [-1, 1] and masks[0] == [1, 0]
    with pytest.raises(ValueError, match="parent"):
        ops.TreeRows.masks([-1, 1])
    with pytest.raises(ValueError, match="words"):
        ops.TreeRows.masks([-1] * 65, words=1)
    with pytest.raises(ValueError, match="words"):
        ops.TreeRows.masks([-1] * 257)


def test_structures_packed_in_one_go_are_the_c_structures():
    import struct

    for packed, c in ((_native.KV_PAGES, _native.KvPages), (_native.KV_TABLE, _native.KvTable), (_native.TREE_STEP, _native.TreeStep), (_native.VERIFY_STEP, _native.VerifyStep)):
        assert packed.size == ctypes.sizeof(c)

        def flat(s):
            for name, kind in s._fields_:
                value = getattr(s, name)
                yield from flat(value) if isinstance(value, ctypes.Structure) else [value or 0]

        values = [0.5 if code in "fd" else i + 1 for i, code in enumerate(packed.format.replace("4x", "")[1:])]
        assert list(flat(c.from_buffer_copy(packed.pack(*values)))) == values
