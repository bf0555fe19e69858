"""Whole pages copied, forked and compacted in stacks whose layers lie apart: every layer moves, and nothing between the layers does (needs a B200)."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

LAYERS, PAGES, HEADS = 3, 10, 2


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _i32(v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


class Stack:
    """Bytes of any kind, layers ``gap`` elements further apart than they are long (exponents: 16 or 48 bytes), and what they are to become."""

    def __init__(self, dev, fmt, gap):
        from georefine_b200 import ops

        g = torch.Generator(device=dev).manual_seed(gap)
        shape = (69, 256) if fmt == "q4" else (256, 128)
        size = 2 if fmt == "bf16" else 1
        self.buffers, self.views = [], []

        def layers(shape, gap):
            own = 1
            for n in shape:
                own *= n
            flat = torch.randint(0, 256, (LAYERS * (own + gap),), generator=g, device=dev, dtype=torch.uint8)
            strides = [1]
            for n in reversed(shape[1:]):
                strides.insert(0, strides[0] * n)
            self.buffers.append(flat)
            self.views.append(flat.as_strided((LAYERS, *shape), (own + gap, *strides)))
            return self.views[-1]

        codes = [layers((PAGES, HEADS, shape[0], shape[1] * size), gap * size) for _ in range(2)]
        exps = [layers((PAGES, HEADS, 256), 48 if gap > 16 else 16) for _ in range(2)] if fmt == "e4m3" else []
        kind = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "q4": torch.uint8}[fmt]
        self.pages = ops.KVPages(*(t.view(kind) for t in codes), *exps)
        self.want = [b.clone() for b in self.buffers]
        self.moved = [w.as_strided(v.shape, v.stride()) for w, v in zip(self.want, self.views)]
        self.fmt = fmt

    def move(self, src, dst, count=256):
        for x in self.moved:
            if self.fmt == "q4":
                for lo, width in ((0, 64), (16384, 4), (17408, 1)):
                    for h in range(HEADS):
                        a = x.view(LAYERS, PAGES, HEADS, -1)[:, :, h, lo:lo + width * count]
                        a[:, dst] = a[:, src].clone()
            else:
                x[:, dst, :, :count] = x[:, src, :, :count].clone()

    def check(self):
        assert all(torch.equal(a, b) for a, b in zip(self.buffers, self.want))


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "q4"])
@pytest.mark.parametrize("gap", [16, 4096])
def test_layers_that_lie_apart(dev, fmt, gap):
    from georefine_b200 import ops

    s = Stack(dev, fmt, gap)
    ops.kv_copy(_i32([0, 3], dev), _i32([4, 5], dev), s.pages, positions=_i32([77, 256], dev))
    s.move(0, 4, 77)
    s.move(3, 5)
    s.check()
    table = _i32([8, 2, -1, -1, -1, -1], dev).view(3, 2)[:2].contiguous()
    refs = torch.zeros(PAGES, dtype=torch.int32, device=dev)
    refs[[8, 2]] = 1
    ops.kv_fork(_i32([0], dev), _i32([1], dev), _i32([256 + 19], dev), _i32([9], dev), table, refs, s.pages)
    s.move(2, 9, 19)
    s.check()
    assert table.tolist() == [[8, 2], [8, 9]] and refs[[8, 2, 9]].tolist() == [2, 1, 1]
    where, used = _i32([0] * PAGES, dev), _i32([0], dev)
    ops.kv_compact(table, refs, s.pages, where, used)
    s.move(8, 0)
    s.move(9, 1)
    s.check()
    assert table.tolist() == [[0, 2], [0, 1]] and used.item() == 3 and refs.tolist() == [2, 1, 1] + [0] * (PAGES - 3)
