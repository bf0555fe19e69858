"""Runs of many causal rows of one sequence, as prompts make them, and tree rows that see alike, over a BF16 or an 8-bit cache: every
length from 64 to 128 rows, against the definition in 64 bits (needs a B200).

A tile of such a run takes 128 / (query heads per kv head) rows, so the lengths leave last tiles of every number of rows, one among
them, and the positions end anywhere in a step of 64."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from spec_reference import attend  # noqa: E402
from test_gpu_tree_attention import Setup, _i32  # noqa: E402

BF = torch.bfloat16
HALF = {"bf16": 2.0 ** -16, "e4m3": 2.0 ** -11}      # half a step of the queries and weights that are multiplied (BF16: in two terms)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _all_rows(s, qkv, turn, slot, seen):
    """``spec_reference.attend`` for all rows of one sequence at once: (wanted, bound), each [rows, nq, 128]; seen [rows, positions]."""
    rows, nq, group, half = qkv.shape[0], s.nq, s.nq // s.nkv, HALF[s.fmt]
    x, h = qkv.view(rows, -1, 128)[:, :nq].double(), 64
    cos, sin = s.cos[turn].double()[:, None], s.sin[turn].double()[:, None]
    q = torch.cat([x[..., :h] * cos[..., :h] - x[..., h:] * sin[..., :h], x[..., h:] * cos[..., h:] + x[..., :h] * sin[..., h:]], dim=2)
    some = seen.any(1)
    k, v = (torch.where(seen.any(0)[:, None, None], t, 0.0).repeat_interleave(group, dim=1) for t in s.held(slot, seen.shape[1]))
    score = (torch.einsum("rhd,phd->rhp", q, k) / math.sqrt(128)).masked_fill(~seen[:, None], -math.inf)
    most = torch.einsum("rhd,phd->rhp", q.abs(), k.abs()).masked_fill(~seen[:, None], 0.0).amax(2) / math.sqrt(128)
    w = torch.softmax(score, dim=2).masked_fill(~some[:, None, None], 0.0)
    want, size = torch.einsum("rhp,phd->rhd", w, v), torch.einsum("rhp,phd->rhd", w, v.abs())
    inner = (torch.expm1(2 * half * most)[..., None] + 2 * half + 2.0 ** -14) * size
    return want, inner + 2.0 ** -8 * (want.abs() + inner) + 1e-30


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("nq,nkv", [(1, 1), (2, 1), (4, 1), (10, 2), (7, 1), (8, 1), (16, 1)])
def test_runs_of_every_length(dev, fmt, nq, nkv):
    s = Setup(dev, fmt, nq, nkv, [0], 2)
    attn = s.ops.TreeAttention(nq, nkv, 128, 2, dev, kv_format=fmt)
    places = torch.arange(512, device=dev)
    # (the first run is a prompt; the others follow cached positions, or come again over what the runs before stored)
    for n in range(64, 129):
        for first in (0, n * 37 % 200 + 1, 320 - n) if n > 64 else (0, 64):
            pos = torch.arange(first, first + n, device=dev)
            qkv = s.qkv(n)
            out = torch.full((n, nq * 128), float("nan"), device=dev, dtype=BF)
            if first and not bool(torch.isfinite(s.held(0, first)[0]).all()):
                k = torch.randn(first, nkv, 128, generator=s.g, device=dev).to(BF)
                s.ops.kv_write(k, k.flip(0), _i32([0] * first, dev), _i32(range(first), dev), s.table, s.pages)
            attn(qkv, s.cos, s.sin, _i32([0] * n, dev), pos.int(), s.table, s.pages, out, longest_run=n)
            want, bound = _all_rows(s, qkv, pos, 0, places <= pos[:, None])
            off = ((out.view(n, nq, 128).double() - want).abs() / bound).amax((1, 2))
            assert bool((off <= 1).all()), (n, first, off.max().item(), int(off.argmax()))
    assert attn.check_status() == 0


@pytest.mark.parametrize("fmt", ["e4m3", "bf16"])
@pytest.mark.parametrize("base", [1, 63, 64, 100, 300])
@pytest.mark.parametrize("rows", [17, 40])
def test_tree_rows_that_see_alike(dev, fmt, base, rows):
    """Rows whose masks are empty see their base alone; rows with one and the same node see up to the same place."""
    s = Setup(dev, fmt, 4, 1, [base], 2)
    attn = s.ops.TreeAttention(4, 1, rows, 2, dev, kv_format=fmt)
    places, pos = torch.arange(512, device=dev), torch.arange(base, base + rows, device=dev)
    for node in (None, 0, 9):
        qkv = s.qkv(rows)
        out = torch.full((rows, 512), float("nan"), device=dev, dtype=BF)
        mask = torch.full((rows, 1), 0 if node is None else 1 << node, dtype=torch.int64, device=dev)
        attn(qkv, s.cos, s.sin, _i32([0] * rows, dev), pos.int(), s.table, s.pages, out, tree=s.ops.TreeRows(_i32([base] * rows, dev), pos.int(), mask))
        seen = places < base
        if node is not None:
            seen = seen | (places == base + node)
        want, bound = _all_rows(s, qkv, pos, 0, seen.expand(rows, -1))
        assert bool(((out.view(rows, 4, 128).double() - want).abs() <= bound).all()), node
    assert attn.check_status() == 0


@pytest.mark.parametrize("tokens", [76, 101, 126, 128, 204, 384 + 76])
def test_a_prompt_s_last_token(dev, tokens):
    """The engine over an 8-bit cache, five query heads a KV head: the attention that the first answer is drawn from."""
    from georefine_b200 import ops, serve
    from spec_reference import rotate

    cfg = serve.DecoderConfig(hidden=512, layers=1, heads=10, kv_heads=2, head_dim=128, ffn=512, vocab=512)
    d = serve.BatchDecoder(serve.DecoderWeights.synthetic(cfg, dev, seed=5, max_m=128), max_rows=128, max_slots=2, max_context=1024, device=dev, kv_format="e4m3")
    prompt = torch.randint(0, cfg.vocab, (tokens,), generator=torch.Generator().manual_seed(tokens)).tolist()
    slot = serve.Batcher(d).admit(prompt)
    at = [r for r in range(d.qkv.shape[0]) if int(d.row_pos[r]) == tokens - 1 and int(d.row_seq[r]) == slot][-1]
    k, v = (torch.empty(tokens, 2, 128, device=dev, dtype=BF) for _ in range(2))
    ops.kv_read(_i32([slot] * tokens, dev), _i32(range(tokens), dev), d.page_table, d.pages.layer(0), k, v)
    q = rotate(d.qkv[at].view(-1, 128)[:10], d.cos[tokens - 1], d.sin[tokens - 1])
    want, bound = attend(q, k.double(), v.double(), torch.ones(tokens, dtype=torch.bool, device=dev), HALF["e4m3"], HALF["e4m3"])
    assert bool(((d.ctx[at].view(10, 128).double() - want).abs() <= bound).all())
