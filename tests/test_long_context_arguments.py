"""Refusals of the 4-bit cache, of rotary positions and of page operators, without a GPU: every call here is turned away, or has nothing to
do, before anything is launched."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, ops  # noqa: E402

ARGUMENT, UNSUPPORTED, WORKSPACE = 1, 2, 3
P = 1 << 20           # stands for device memory: aligned, never touched
BLOCK = 17664


def _pages(**kw):
    return _native.KvPages(**{**dict(k=P, v=P, layers=1, pages=4, nkv=2, format=4), **kw})


def _table(**kw):
    return _native.KvTable(**{**dict(table=P, ld=4, slots=2, max_pages=4), **kw})


BAD_PAGES = [(dict(k=None), ARGUMENT), (dict(v=None), ARGUMENT), (dict(k_exp=P), ARGUMENT), (dict(k_exp=P, v_exp=P), ARGUMENT), (dict(format=3), UNSUPPORTED), (dict(format=5), UNSUPPORTED),
             (dict(layers=0), ARGUMENT), (dict(pages=0), ARGUMENT), (dict(nkv=0), ARGUMENT), (dict(k=P + 8), ARGUMENT), (dict(v=P + 4), ARGUMENT),
             (dict(layers=2, layer_stride=4 * 2 * BLOCK - 16), ARGUMENT), (dict(layers=2, layer_stride=4 * 2 * BLOCK + 8), ARGUMENT), (dict(pages=1 << 30), UNSUPPORTED), (dict(nkv=5000), UNSUPPORTED)]
BAD_TABLES = [(dict(table=None), ARGUMENT), (dict(slots=0), ARGUMENT), (dict(max_pages=0), ARGUMENT), (dict(ld=3), ARGUMENT), (dict(max_pages=1 << 24, ld=1 << 24), UNSUPPORTED)]


def test_4_bit_pages_and_tables():
    lib = _native.lib()
    rows = lambda pages, table, n=3: lib.grb_kv_write(pages, table, P, P, P, 256, P, 256, n, None)
    keep = lambda pages, table, n=2: lib.grb_kv_keep(pages, table, P, P, P, 4, P, n, 4, None)
    for kw, status in BAD_PAGES:
        for call in (rows, keep):
            assert call(_pages(**kw), _table()) == status, kw
        assert lib.grb_kv_copy(_pages(**kw), P, P, None, 3, None) == status, kw
    for kw, status in BAD_TABLES:
        for call in (rows, keep):
            assert call(_pages(), _table(**kw)) == status, kw
    assert rows(_pages(layers=2, layer_stride=4 * 2 * BLOCK), _table(), 0) == 0 and keep(_pages(), _table(), 0) == 0


def _step(**kw):
    s = _native.TreeStep()
    d = dict(qkv=P, ldq=1536, cos_table=P, sin_table=P, rope_rows=1024, row_seq=P, row_pos=P, scratch=P, scratch_bytes=1 << 40, out=P, ldo=1024, rows=3, nq=8, head_dim=128, scaling=0.1,
             pages=_pages(), table=_table())
    for name, value in {**d, **kw}.items():
        setattr(s, name, value)
    return s


def test_attention_over_4_bit_pages():
    lib = _native.lib()
    for kw, status in BAD_PAGES:
        assert lib.grb_attn_tree(_step(pages=_pages(**kw)), None) == status, kw
    size = lib.grb_attn_tree_scratch_bytes
    need = size(3, 8, 4, 4)
    assert lib.grb_attn_tree(_step(scratch_bytes=need - 1), None) == WORKSPACE and lib.grb_attn_tree(_step(rows=0), None) == 0
    assert 0 < need < size(3, 8, 4, 1) and size(3, 8, 5, 4) > size(3, 8, 4, 4) and size(3, 8, 4, 3) == size(3, 8, 4, 5) == 0


def _rotary(**kw):
    s = _native.RotaryStep()
    d = dict(x=P, ldx=1024, ldx_head=128, out=P, ldo=1024, ldo_head=128, positions=P, turns=P, rows=3, heads=8, dim=128, turned=64, factor=1.0)
    for name, value in {**d, **kw}.items():
        setattr(s, name, value)
    return s


def test_rotary_arguments():
    call = _native.lib().grb_rotary
    for kw, status in ([(dict([(n, None)]), ARGUMENT) for n in ("x", "out", "positions", "turns")] +
                       [(dict(dtype=3), ARGUMENT), (dict(layout=2), ARGUMENT), (dict(positions_64=2), ARGUMENT), (dict(backward=2), ARGUMENT), (dict(heads=0), ARGUMENT), (dict(turned=0), ARGUMENT),
                        (dict(turned=63), ARGUMENT), (dict(turned=130), ARGUMENT), (dict(dim=1026, turned=64, ldo_head=1026, ldo=1 << 20), UNSUPPORTED), (dict(heads=70000), UNSUPPORTED),
                        (dict(x=P + 1), ARGUMENT), (dict(out=P + 1), ARGUMENT), (dict(x=P + 2, dtype=1), ARGUMENT), (dict(turns=P + 4), ARGUMENT), (dict(positions=P + 2), ARGUMENT),
                        (dict(positions=P + 4, positions_64=1), ARGUMENT), (dict(ldo_head=127), ARGUMENT), (dict(ldo=1023), ARGUMENT), (dict(ldo=0), ARGUMENT), (dict(ldo_head=0), ARGUMENT),
                        (dict(ldx=-1), ARGUMENT), (dict(ldx_head=-1), ARGUMENT), (dict(ldo=128, ldo_head=383), ARGUMENT)]):
        assert call(_rotary(**kw), None) == status, kw
    assert call(None, None) == ARGUMENT and call(_rotary(rows=0), None) == 0
    for kw in (dict(ldx=2048), dict(ldx_head=256), dict(ldo=2048), dict(rows=1, ldo_head=256)):      # in place, and elsewhere
        assert call(_rotary(**kw), None) == ARGUMENT
    assert call(_rotary(rows=0, ldo=128, ldo_head=384), None) == 0           # rows inside, heads outside
    assert _native.ROTARY_STEP.size == ctypes.sizeof(_native.RotaryStep)
    values = P, 7, 8, 2 * P, 9, 10, 3 * P, 4 * P, 1, 2, 3, 4, 1, 2, 1, 0, 0.5
    s = _native.RotaryStep.from_buffer_copy(_native.ROTARY_STEP.pack(*values))
    assert tuple(getattr(s, n) for n, _ in s._fields_) == values


def test_page_operators():
    lib = _native.lib()
    assert lib.grb_kv_copy(_pages(), None, P, None, 3, None) == lib.grb_kv_copy(_pages(), P, None, None, 3, None) == ARGUMENT and lib.grb_kv_copy(_pages(), P, P, None, 0, None) == 0
    fork = lambda pages=None, table=None, n=3, **kw: lib.grb_kv_fork(pages or _pages(), table or _table(), *({**dict(parents=P, children=P, lengths=P, fresh=P, refs=P), **kw}.values()), -1, n, None)
    free = lambda table=None, slots=P, refs=P, pages=4, n=3: lib.grb_kv_free(table or _table(), slots, refs, pages, -1, n, None)
    size = lib.grb_kv_compact_scratch_bytes(4)
    compact = lambda pages=None, table=None, bytes=size, **kw: lib.grb_kv_compact(pages or _pages(), table or _table(), *({**dict(refs=P, where=P, used=P, scratch=P), **kw}.values()), bytes, None)
    for name in ("parents", "children", "lengths", "fresh", "refs"):
        assert fork(**{name: None}) == ARGUMENT
    for name in ("refs", "where", "used", "scratch"):
        assert compact(**{name: None}) == ARGUMENT
    assert compact(scratch=P + 8) == ARGUMENT and compact(bytes=size - 1) == WORKSPACE and size >= 16 + 8 * 4
    assert free(slots=None) == free(refs=None) == free(pages=0) == ARGUMENT
    for kw, status in BAD_TABLES:
        assert fork(table=_table(**kw)) == free(table=_table(**kw)) == compact(table=_table(**kw)) == status
    for kw, status in BAD_PAGES:
        assert fork(pages=_pages(**kw)) == compact(pages=_pages(**kw)) == status
    assert fork(n=0) == free(n=0) == 0


class _Here:
    """Stands for a tensor on a GPU where only its description is looked at."""

    def __new__(cls, *shape, dtype=torch.int32):
        return torch.empty(*shape, dtype=dtype, device="meta")


def test_python_refusals_before_the_library_is_called():
    with pytest.raises(ValueError, match="CUDA"):
        ops.KVPages.alloc(2, 2, "cpu", kv_format="q4")
    with pytest.raises(ValueError, match="69, 256"):
        ops.KVPages(torch.zeros(2, 2, 256, 128, dtype=torch.uint8), torch.zeros(2, 2, 256, 128, dtype=torch.uint8))
    with pytest.raises(ValueError, match="format"):
        ops.KVPages.alloc(2, 2, "cpu", kv_format="q5")
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_free(torch.zeros(1, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="layout"):
        ops.Rope(64, layout="neighbours", device="cpu")
    rope = ops.Rope(64, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        ops.rotary(torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), rope)
    with pytest.raises(ValueError, match="128 dimensions"):
        rope.tables(10)


class _Pages:
    device, pages, _packed = torch.device("meta"), 4, b""


@pytest.mark.parametrize("call", [
    lambda: ops.kv_copy(_Here(3), _Here(2), _Pages), lambda: ops.kv_copy(_Here(3), _Here(3, dtype=torch.int64), _Pages), lambda: ops.kv_copy(_Here(3), _Here(3), _Pages, positions=_Here(3, 1)),
    lambda: ops.kv_copy(torch.zeros(3, dtype=torch.int32), _Here(3), _Pages),
    lambda: ops.kv_fork(_Here(2), _Here(2), _Here(1), _Here(2), _Here(3, 4), _Here(4), _Pages), lambda: ops.kv_fork(_Here(2), _Here(2), _Here(2), _Here(2), _Here(3, 4), _Here(5), _Pages),
    lambda: ops.kv_fork(_Here(2), _Here(2), _Here(2), _Here(2), _Here(12), _Here(4), _Pages), lambda: ops.kv_fork(_Here(2), _Here(2), _Here(2), _Here(2), _Here(3, 4), _Here(4), _Pages, empty=1 << 31),
    lambda: ops.kv_compact(_Here(3, 4), _Here(4), _Pages, _Here(3), _Here(1)), lambda: ops.kv_compact(_Here(3, 4), _Here(4), _Pages, _Here(4), _Here(2)),
    lambda: ops.kv_compact(_Here(3, 4)[:, ::2], _Here(4), _Pages, _Here(4), _Here(1)), lambda: ops.kv_compact(_Here(3, 4), _Here(4), _Pages, _Here(4), _Here(1), scratch=_Here(64)),
])
def test_page_vectors_of_the_wrong_kind(call):
    with pytest.raises(ValueError):
        call()


def test_frequencies_by_their_formulas():
    for dim, theta in ((2, 1e4), (64, 1e4), (96, 1e6), (128, 5e5)):
        plain = [theta ** (-2 * i / dim) for i in range(dim // 2)]
        got, factor = ops.rope_frequencies(dim, theta)
        assert factor == 1.0 and all(math.isclose(a, b, rel_tol=1e-14) for a, b in zip(got, plain))
        got, factor = ops.rope_frequencies(dim, theta, {"kind": "linear", "factor": 8.0})
        assert factor == 1.0 and all(math.isclose(a, b / 8, rel_tol=1e-14) for a, b in zip(got, plain))
        got, _ = ops.rope_frequencies(dim, theta, {"kind": "ntk", "factor": 8.0})
        assert math.isclose(got[0], plain[0]) and (dim == 2 or math.isclose(got[-1], plain[-1] / 8, rel_tol=1e-12))      # fastest as it was, slowest by the factor
        for kind, extra in (("yarn", {}), ("bands", {"low": 1.0, "high": 4.0})):
            got, factor = ops.rope_frequencies(dim, theta, {"kind": kind, "factor": 8.0, "original": 4096, **extra})
            turns = [4096 * f / (2 * math.pi) for f in plain]
            for f, p, t in zip(got, plain, turns):
                assert p / 8 * (1 - 1e-12) <= f <= p * (1 + 1e-12)
                if kind == "bands":
                    share = min(max((t - 1) / 3, 0.0), 1.0)
                    assert math.isclose(f, p / 8 * (1 - share) + p * share, rel_tol=1e-12)
                elif t >= 32 * theta ** (2 / dim):         # a pair's number or more beyond the ramp's end
                    assert math.isclose(f, p, rel_tol=1e-12)
                elif t <= theta ** (-2 / dim):
                    assert math.isclose(f, p / 8, rel_tol=1e-12)
            assert math.isclose(factor, 0.1 * math.log(8) + 1 if kind == "yarn" else 1.0)
    assert ops.rope_frequencies(64, 1e4, {"kind": "yarn", "factor": 8.0, "original": 4096, "attention": 1.25})[1] == 1.25
    for bad in (dict(dim=0), dict(dim=3), dict(theta=0.0), dict(theta=math.inf), dict(scaling={"factor": 2.0}), dict(scaling={"kind": "twice"}), dict(scaling={"kind": "linear"}),
                dict(scaling={"kind": "linear", "factor": 0.0}), dict(scaling={"kind": "linear", "factor": 2.0, "original": 5}), dict(scaling={"kind": "yarn", "factor": 2.0}),
                dict(scaling={"kind": "yarn", "factor": 2.0, "original": 4096, "fast": 1.0, "slow": 1.0}), dict(scaling={"kind": "bands", "factor": 2.0, "original": 4096, "low": 4.0, "high": 4.0})):
        with pytest.raises(ValueError):
            ops.rope_frequencies(**{**dict(dim=64, theta=1e4), **bad})


def test_turns_are_fractions_of_a_turn():
    rope = ops.Rope(128, 1e6, device="cpu")
    for f, t in zip(rope.frequencies, rope.turns.tolist()):
        assert abs((t % (1 << 64)) / 2 ** 64 - f / (2 * math.pi)) <= 2.0 ** -53 * f + 2.0 ** -65        # (a fraction is kept in units of 2^-64)
    assert ops.Rope(2, 1e4, scaling={"kind": "linear", "factor": 0.125}, device="cpu").turns.dtype == torch.int64        # (8 radians: more than a turn)
    assert abs((ops.Rope(2, 1e4, scaling={"kind": "linear", "factor": 0.125}, device="cpu").turns.item() % (1 << 64)) / 2 ** 64 - (8 / (2 * math.pi) - 1)) < 1e-15


def test_decoder_configurations():
    from georefine_b200 import serve

    cfg = serve.DecoderConfig(rope_scaling={"kind": "linear", "factor": 2.0}, rope_dim=64, rope_layout="interleaved")
    assert cfg.rope_options == {"kind": "linear", "factor": 2.0} and hash(cfg) is not None and serve.DecoderConfig().rope_options is None
    assert serve.DecoderConfig(rope_scaling=cfg.rope_scaling, rope_dim=64, rope_layout="interleaved") == cfg
    for bad in (dict(rope_layout="pairs"), dict(rope_dim=0), dict(rope_dim=130), dict(rope_dim=63), dict(rope_scaling={"kind": "linear"}), dict(rope_scaling={"kind": "more", "factor": 2.0})):
        with pytest.raises(ValueError):
            serve.DecoderConfig(**bad)


BASE = dict(hidden_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=128, intermediate_size=1024, vocab_size=1000, rope_theta=5000.0,
            max_position_embeddings=8192)


@pytest.mark.parametrize("given,fields", [
    ({}, {}), (dict(rope_scaling=None), {}), (dict(rope_scaling={"rope_type": "default"}), {}), (dict(partial_rotary_factor=0.5), dict(rope_dim=64)), (dict(partial_rotary_factor=1.0), {}),
    (dict(rope_scaling={"type": "linear", "factor": 4.0}), dict(rope_options={"kind": "linear", "factor": 4.0})),
    (dict(rope_scaling={"rope_type": "yarn", "type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}),
     dict(rope_options={"kind": "yarn", "factor": 4.0, "original": 2048.0, "fast": 32.0, "slow": 1.0, "attention": None})),
    (dict(rope_scaling={"rope_type": "yarn", "factor": 4.0, "beta_fast": 16, "beta_slow": 2, "attention_factor": 1.5}),
     dict(rope_options={"kind": "yarn", "factor": 4.0, "original": 8192.0, "fast": 16.0, "slow": 2.0, "attention": 1.5})),
    (dict(rope_scaling={"rope_type": "by bands", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 4096}),
     dict(rope_options={"kind": "bands", "factor": 8.0, "original": 4096.0, "low": 1.0, "high": 4.0})),
    (dict(rope_parameters={"rope_theta": 7000.0, "rope_type": "default", "partial_rotary_factor": 0.25}, rope_theta=None), dict(rope_theta=7000.0, rope_dim=32)),
])
def test_a_checkpoint_s_rotary_positions(given, fields):
    from georefine_b200 import checkpoint

    config = {k: v for k, v in {**BASE, **given}.items() if v is not None}
    cfg = checkpoint.decoder_config(config)
    want = {**dict(rope_theta=5000.0, rope_dim=None, rope_options=None, rope_layout="half"), **fields}
    assert {k: getattr(cfg, k) for k in want} == want


@pytest.mark.parametrize("scaling", [{"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "linear"}, {"rope_type": "yarn", "factor": 2.0, "mscale": 0.7}, {"rope_type": "linear", "factor": "many"},
                                     {"full_attention": {"rope_type": "default"}}])
def test_a_checkpoint_s_rotary_positions_that_are_not_known(scaling):
    from georefine_b200 import checkpoint
    from georefine_b200.serving import ContextServingError

    with pytest.raises(ContextServingError):
        checkpoint.decoder_config({**BASE, "rope_scaling": scaling})
