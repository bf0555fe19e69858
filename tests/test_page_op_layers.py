"""Stacks of 8-bit pages whose layers' exponents lie any distance apart: what moves whole pages takes pieces of 16 bytes and refuses other
distances, before anything is launched; what goes by entries takes them all.  No GPU."""
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import _native, ops  # noqa: E402

ARGUMENT = 1
P = 1 << 20           # stands for device memory: aligned, never touched
EXPS = 4 * 2 * 256    # exponents of a layer


def _pages(**kw):
    return _native.KvPages(**{**dict(k=P, v=P, k_exp=P, v_exp=P, layers=2, layer_stride=EXPS * 128, exp_stride=EXPS, pages=4, nkv=2, format=1), **kw})


def _calls(pages):
    """Status of each operator on whole pages (copies and forks of none; a compaction whose scratch is too small, which is refused behind the pages)."""
    lib, table = _native.lib(), _native.KvTable(table=P, ld=4, slots=2, max_pages=4)
    return (lib.grb_kv_copy(pages, P, P, None, 0, None), lib.grb_kv_fork(pages, table, P, P, P, P, P, -1, 0, None),
            lib.grb_kv_compact(pages, table, P, P, P, P, lib.grb_kv_compact_scratch_bytes(4) - 1, None))


@pytest.mark.parametrize("more", [1, 2, 4, 8, 24, 100])
def test_exponents_off_the_16_byte_grid_are_refused(more):
    assert _calls(_pages(exp_stride=EXPS + more)) == (ARGUMENT, ARGUMENT, ARGUMENT)


@pytest.mark.parametrize("kw", [dict(), dict(exp_stride=EXPS + 16), dict(exp_stride=4 * EXPS), dict(layers=1, exp_stride=EXPS + 1), dict(layers=1, exp_stride=0)])
def test_exponents_on_it_are_taken(kw):
    assert _calls(_pages(**kw)) == (0, 0, 3)


def test_rows_and_kept_paths_take_any_distance():
    lib, table = _native.lib(), _native.KvTable(table=P, ld=4, slots=2, max_pages=4)
    for more in (0, 1, 8):
        pages = _pages(exp_stride=EXPS + more)
        assert lib.grb_kv_write(pages, table, P, P, P, 256, P, 256, 0, None) == lib.grb_kv_keep(pages, table, P, P, P, 4, P, 0, 4, None) == 0


class _Stack:
    """Stands for ``KVPages`` where only its description is looked at."""

    device, pages, kv_heads, stacked, format, _packed = torch.device("meta"), 4, 2, True, "e4m3", b""

    def __init__(self, layers, distance):
        self.k_exp = torch.empty(layers * distance, dtype=torch.uint8, device="meta").as_strided((layers, 4, 2, 256), (distance, 512, 256, 1))


@pytest.mark.parametrize("distance", [EXPS + 1, EXPS + 8])
def test_the_python_calls_say_so(distance):
    i32 = lambda *shape: torch.empty(*shape, dtype=torch.int32, device="meta")
    pages = _Stack(2, distance)
    for call in (lambda: ops.kv_copy(i32(3), i32(3), pages), lambda: ops.kv_fork(i32(2), i32(2), i32(2), i32(2), i32(3, 4), i32(4), pages),
                 lambda: ops.kv_compact(i32(3, 4), i32(4), pages, i32(4), i32(1), scratch=torch.empty(64, dtype=torch.uint8, device="meta"))):
        with pytest.raises(ValueError, match="16 bytes"):
            call()
