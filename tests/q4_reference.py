"""4-bit cache entries by their definition, in 64 bits, and a cache with rows for the tests of what reads it."""
import torch

from spec_reference import attend, rotate

BF = torch.bfloat16
GRID = torch.tensor([(16 + m) * 2.0 ** k for k in range(12) for m in range(16)], dtype=torch.float64)      # what a scale may be


def _nearest(values, want):
    """Index of the value nearest to `want` (ties to the even index)."""
    want = want.clamp(max=float(values[-1]))       # (differences to numbers far beyond the last value are all alike in 64 bits)
    hi = torch.searchsorted(values, want.contiguous()).clamp(max=values.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = (values[hi] - want).abs(), (want - values[lo]).abs()
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def entry(x):
    """Vectors [..., 128] -> what an entry holds of them: (whole numbers, scale bytes [..., 4], exponent bytes, values)."""
    x = x.double()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    top = x.abs().amax(-1)
    e = torch.full_like(top, -40.0)
    for power in range(-39, 23):                   # floor(log2(top / 7)) + 9 >= power
        e = torch.where(top >= 7 * 2.0 ** (power - 9), torch.full_like(e, power), e)
    unit = torch.exp2(e - 24)[..., None]
    groups = x.unflatten(-1, (4, 32))
    at = _nearest(GRID.to(x.device), groups.abs().amax(-1) / 7 / unit)
    step = (GRID.to(x.device)[at] * unit)[..., None]
    code = torch.round(groups / step).clamp(-7, 7)
    value = (code * step).flatten(-2)
    nan = torch.where(fine[..., None], value, torch.nan)
    byte = torch.where(fine, e + 127, torch.full_like(e, 255.0)).to(torch.uint8)
    return code.flatten(-2), (at + 64).to(torch.uint8), byte, nan


def packed(code):
    """Whole numbers [..., 128] as an entry's 64 bytes, nibble by nibble."""
    out = torch.zeros(*code.shape[:-1], 64, dtype=torch.int32, device=code.device)
    for d in range(128):
        word, i = divmod(d, 8)
        nibble = i // 2 + 4 * (i % 2)
        out[..., 4 * word + nibble // 2] |= (code[..., d].int() + 8) << (4 * (nibble % 2))
    return out.to(torch.uint8)


def i32(v, dev):
    return torch.tensor(list(v), dtype=torch.int32, device=dev)


class Setup:
    """Sequences with cached positions in scattered pages, whose other places hold what memory that nobody wrote may hold."""

    def __init__(self, dev, nq, nkv, lengths, per_slot, seed=0, scale=1.0, fmt="q4"):
        from georefine_b200 import ops

        self.dev, self.nq, self.nkv, self.ops, self.fmt = dev, nq, nkv, ops, fmt
        self.g = torch.Generator(device=dev).manual_seed(1000 * nq + nkv + seed)
        slots = len(lengths)
        self.table = torch.randperm(slots * per_slot, generator=self.g, device=dev).reshape(slots, per_slot).int()
        self.pages = ops.KVPages.alloc(slots * per_slot, nkv, dev, kv_format=fmt)
        for t in (self.pages.k, self.pages.v):
            t.view(torch.uint8).fill_(0xFF)
        self.cos, self.sin = ops.rope_tables(per_slot * 256, device=dev)
        for slot, n in enumerate(lengths):
            if n:
                k, v = (scale * torch.randn(n, nkv, 128, generator=self.g, device=dev) * torch.exp(0.7 * torch.randn(n, 1, 1, generator=self.g, device=dev)) for _ in range(2))
                ops.kv_write(k.to(BF), v.to(BF), i32([slot] * n, dev), i32(range(n), dev), self.table, self.pages)

    def qkv(self, rows, q_scale=1.5):
        x = torch.randn(rows, (self.nq + 2 * self.nkv) * 128, generator=self.g, device=self.dev)
        x[:, :self.nq * 128] *= q_scale
        return x.to(BF)

    def attention(self, rows):
        return self.ops.TreeAttention(self.nq, self.nkv, rows, self.table.shape[1], self.dev, kv_format=self.fmt)

    def held(self, slot, n):
        """Keys and values of positions 0 .. n - 1 as the cache holds them."""
        k, v = (torch.full((n, self.nkv, 128), 7.0, device=self.dev, dtype=BF) for _ in range(2))
        self.ops.kv_read(i32([slot] * n, self.dev), i32(range(n), self.dev), self.table, self.pages, k, v)
        return k.double(), v.double()

    def check(self, qkv, seq, pos, out, seen, rope=None, rows=None):
        """Rows against the definition over what the cache holds after the call; ``seen(row, positions)`` -> bool tensor.  Queries and weights are
        rounded to FP16, half a step of which is 2^-11 of the number - but 2^-25 below 2^-14.  A weight is held as w 2^e over the largest such
        product's 2^-7 or less (e: the exponent of the position's value entry), the entry as v 2^-e <= 7 x 31 x 2^11 x 2^-24 < 0.0266; and 2^e <= 2^9 / 7 of the entry's
        largest component.  So a weight that small is off by 2^-25 2^-7 x 2^9 / 7 x 0.0266 < 2^-31 of the largest component seen, at each of the positions
        seen: it shows where a component is zero at every position of weight."""
        half = 2.0 ** -11
        for r in range(len(seq)) if rows is None else rows:
            s, p = seq[r], pos[r]
            if s < 0:
                continue
            turn = p if rope is None else rope[r]
            x = qkv[r].view(-1, 128)
            q = rotate(x[:self.nq], self.cos[turn], self.sin[turn])
            k_new, v_new = rotate(x[self.nq:self.nq + self.nkv], self.cos[turn], self.sin[turn]), x[self.nq + self.nkv:].double()
            n = self.table.shape[1] * 256
            k, v = self.held(s, n)
            if self.fmt == "q4":
                # (products of BF16 numbers are exact in 32 bits, and their sum is rounded once before the codes are chosen)
                assert torch.equal(k[p], entry(k_new.float())[3]) and torch.equal(v[p], entry(v_new)[3])
            sees = seen(r, torch.arange(n, device=self.dev))
            want, bound = attend(q, k, v, sees, half, half)
            if bool(sees.any()):
                bound = bound + int(sees.sum()) * 2.0 ** -31 * v[sees].abs().amax()
            got = out[r].view(self.nq, 128).double()
            assert bool(((got - want).abs() <= bound).all()), (r, float(((got - want).abs() / bound).max()))


def causal(pos):
    return lambda r, p: p <= pos[r]
