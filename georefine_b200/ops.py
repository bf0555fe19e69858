"""The kernels of a batched decode step other than the linears, as calls on torch tensors.

Thin wrappers over the C ABI (``grb_rmsnorm_bf16``, ``grb_silu_mul_bf16``, ``grb_argmax_bf16``,
``grb_attn_decode_bf16``; kernels in ``csrc/decode_ops.cuh``): every call writes into a tensor the caller provides, on
the current stream, without allocating or synchronising, so a whole step can be captured in a CUDA graph.  They take the
place of the reference's step kernels (``glc_serve/fastdec_kernels.cu:83-110,324-488``) for a plain grouped-query
decoder with head dimension 128.

``KVPages``, ``kv_write``, ``kv_read``, ``kv_keep`` and ``TreeAttention`` are speculative serving over a cache in BF16, 8 or 4 bits
(``csrc/kv_cache.cuh``, ``csrc/tree_attention.cuh``, ``csrc/tree_q4.cuh``); ``Rope`` and ``rotary`` are rotary positions in every layout and scaling
(``csrc/rotary.cuh``); ``kv_copy``, ``kv_fork``, ``kv_free`` and ``kv_compact`` are pages shared and moved (``csrc/kv_pages.cuh``).  The
reference has no counterparts.
"""
from __future__ import annotations

import ctypes
import decimal
import math
from decimal import Decimal

from . import _native

PAGE = 256        # positions per KV page
PART = 128        # positions per attention CTA pass: two parts per page
HEAD_DIM = 128


def _stream(t):
    import torch

    return torch.cuda.current_stream(t.device).cuda_stream


def rmsnorm(h, weight, out, *, delta=None, eps=1e-6, unit_offset=False):
    """out = bf16(h * rsqrt(mean(h^2) + eps) * weight); with ``delta`` the residual add h = bf16(h + delta) happens first
    and is written back into ``h``.  ``unit_offset``: the weight is stored as an offset from one."""
    rows, hidden = h.shape
    st = _native.lib().grb_rmsnorm_bf16(h.data_ptr(), h.stride(0), None if delta is None else delta.data_ptr(),
                                        0 if delta is None else delta.stride(0), weight.data_ptr(), out.data_ptr(), out.stride(0),
                                        rows, hidden, float(eps), int(bool(unit_offset)), _stream(h))
    _native.check(st, "grb_rmsnorm_bf16")


def silu_mul(gate_up, out):
    """out[r, i] = bf16(bf16(silu(gate_up[r, i])) * gate_up[r, f + i]) with f = out.shape[1]."""
    rows, f = out.shape
    st = _native.lib().grb_silu_mul_bf16(gate_up.data_ptr(), gate_up.stride(0), out.data_ptr(), out.stride(0), rows, f, _stream(out))
    _native.check(st, "grb_silu_mul_bf16")


def argmax(logits, out):
    """out[r] (int32) = index of the first maximum of row r."""
    rows, vocab = logits.shape
    st = _native.lib().grb_argmax_bf16(logits.data_ptr(), logits.stride(0), rows, vocab, out.data_ptr(), _stream(logits))
    _native.check(st, "grb_argmax_bf16")


def rope_tables(positions: int, theta: float = 1e6, device="cuda:0"):
    """BF16 cos / sin tables [positions, 128] in the rotate-half convention (the second half repeats the first)."""
    import torch

    inv = 1.0 / (theta ** (torch.arange(0, HEAD_DIM, 2, dtype=torch.float32) / HEAD_DIM))
    angle = torch.arange(positions, dtype=torch.float32)[:, None] * inv[None, :]
    angle = torch.cat([angle, angle], dim=1)
    return angle.cos().to(torch.bfloat16).to(device), angle.sin().to(torch.bfloat16).to(device)


class PagedAttention:
    """Scratch and geometry of the attention call for up to ``max_rows`` rows per step and ``max_pages`` pages per
    sequence; ``__call__`` runs rotary embedding + KV append + decode attention for one layer."""

    def __init__(self, nq: int, nkv: int, max_rows: int, max_pages: int, device):
        import torch

        if nq % nkv or nq // nkv not in (1, 2, 4, 5, 8):
            raise ValueError("query heads per kv head must be 1, 2, 4, 5 or 8")
        self.nq, self.nkv, self.max_rows, self.max_pages = nq, nkv, max_rows, max_pages
        self.q = torch.empty(max_rows, nq, HEAD_DIM, device=device, dtype=torch.bfloat16)
        self.max_parts = max_pages * (PAGE // PART)
        self.part_acc = torch.empty(max_rows, nq, self.max_parts, HEAD_DIM, device=device, dtype=torch.float32)
        self.part_ml = torch.empty(max_rows, nq, self.max_parts, 2, device=device, dtype=torch.float32)
        self.scratch_bytes = sum(t.numel() * t.element_size() for t in (self.q, self.part_acc, self.part_ml))

    def __call__(self, qkv, cos, sin, row_seq, row_pos, page_table, k_pages, v_pages, out, *, max_splits=None):
        rows = qkv.shape[0]
        if rows > self.max_rows:
            raise ValueError("more rows than the attention scratch was sized for")
        step = _native.AttnStep()
        step.qkv, step.ldq = qkv.data_ptr(), qkv.stride(0)
        step.cos_table, step.sin_table = cos.data_ptr(), sin.data_ptr()
        step.row_seq, step.row_pos, step.page_table = row_seq.data_ptr(), row_pos.data_ptr(), page_table.data_ptr()
        step.max_pages = page_table.shape[1]
        step.k_pages, step.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
        step.q, step.part_acc, step.part_ml, step.out = self.q.data_ptr(), self.part_acc.data_ptr(), self.part_ml.data_ptr(), out.data_ptr()
        step.rows, step.nq, step.nkv, step.head_dim = rows, self.nq, self.nkv, HEAD_DIM
        # parts (128 positions each) launched per (row group, kv head) = the stride of the partial buffers in this call;
        # rows shorter than that leave their surplus CTAs at once.  A caller that knows every row is short passes fewer.
        step.max_splits = min(self.max_parts, page_table.shape[1] * (PAGE // PART)) if max_splits is None else int(max_splits)
        if not 1 <= step.max_splits <= self.max_parts:
            raise ValueError("max_splits outside the scratch that was allocated")
        step.scaling = 1.0 / math.sqrt(HEAD_DIM)
        st = _native.lib().grb_attn_decode_bf16(ctypes.byref(step), _stream(qkv))
        _native.check(st, "grb_attn_decode_bf16")


# ---- a cache in BF16, 8 or 4 bits, and attention of causal rows and draft trees over it --------------------------------

KV_FORMATS = ("bf16", "e4m3")                       # of 128 numbers an entry
KV_CODES = {"bf16": 0, "e4m3": 1, "q4": 4}          # all formats, and their numbers in the C interface
Q4_ROWS = 69          # rows of 256 bytes of a 4-bit page of one head; bytes of an entry
MASK_WORDS = 4        # of 64 nodes: the largest tree a row's mask describes
TREE_ROWS = 4096      # rows of one call


def _on(t, device, dtype, what, shape=None):
    """Refuses a tensor that the kernels would read wrongly."""
    if t.device != device or t.dtype != dtype:
        raise ValueError(f"{what}: {t.dtype} on {t.device}, not {dtype} on {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, not {shape}")


def _vector(t, device, what, n=None):
    """A contiguous int32 vector's address."""
    import torch

    if t.dim() != 1 or (n is not None and t.shape[0] != n) or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous vector{'' if n is None else f' of {n}'} is wanted")
    _on(t, device, torch.int32, what)
    return t.data_ptr()


def _ld(t, width, what):
    """Elements from one row (of ``width``) to the next.  Rows that overlap - an expanded tensor's are all the same memory - would be
    walked past its end; a single row has no distance to keep."""
    ld = t.stride(0)
    if ld < width:
        if t.shape[0] > 1:
            raise ValueError(f"{what}: rows overlap (they start {ld} elements apart and are {width} long)")
        return width
    return ld


def _launch(device, name, *args):
    """The call on the device's current stream; a device that is not the current one is made so meanwhile."""
    import torch

    index = device.index
    if index == torch._C._cuda_getDevice():
        status = _native.packed(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = _native.packed(name)(*args, torch._C._cuda_getCurrentRawStream(index))
    if status:
        _native.check(status, name)


class KVPages:
    """Keys and values of one layer, [pages, kv heads, 256, 128], or of a stack of layers ([layers, pages, ...], layers may be
    strided): BF16, or ``float8_e4m3fn`` codes with an exponent byte per entry (128 values of one head at one position) in
    ``k_exp`` and ``v_exp``, [pages, kv heads, 256].  In 4 bits (``"q4"``: 69 bytes for an entry of 256) pages are ``uint8`` [pages, kv heads,
    69, 256] and hold codes, scales and exponents together.  Where whole pages are copied, layers of exponents lie a multiple of 16 bytes
    apart.  The formats are in ``csrc/kv_cache.cuh``.  An object holds no copies."""

    def __init__(self, k, v, k_exp=None, v_exp=None):
        import torch

        if k.dim() not in (4, 5) or tuple(k.shape[-2:]) != ((Q4_ROWS, PAGE) if k.dtype == torch.uint8 else (PAGE, HEAD_DIM)):
            raise ValueError("pages are [pages, kv heads, 256, 128] (4 bits: [pages, kv heads, 69, 256]), or that with the layers in front")
        if k.device.type != "cuda":
            raise ValueError("pages live on a CUDA device")
        self.format = {torch.bfloat16: "bf16", torch.float8_e4m3fn: "e4m3", torch.uint8: "q4"}.get(k.dtype)
        if self.format is None:
            raise ValueError(f"pages are BF16, e4m3 or bytes of 4-bit pages, not {k.dtype}")
        _on(v, k.device, k.dtype, "values", tuple(k.shape))
        if (k_exp is None) != (self.format != "e4m3") or (v_exp is None) != (self.format != "e4m3"):
            raise ValueError("exponents go with e4m3 pages, and with those alone")
        for t, what in ((k, "keys"), (v, "values"), (k_exp, "exponents of keys"), (v_exp, "exponents of values")):
            if t is None:
                continue
            if t is not k and t is not v:
                _on(t, k.device, torch.uint8, what, tuple(k.shape[:-1]))
            if not (t if k.dim() == 4 else t[0]).is_contiguous():
                raise ValueError(f"{what}: the pages of a layer have to be contiguous")
        if k.dim() == 5 and k.shape[0] > 1 and (k.stride(0) != v.stride(0) or (k_exp is not None and k_exp.stride(0) != v_exp.stride(0))):
            raise ValueError("keys and values: layers are equally far apart")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.device, self.stacked = k.device, k.dim() == 5
        self.pages, self.kv_heads = k.shape[-4], k.shape[-3]
        stride = (k.stride(0), 0 if k_exp is None else k_exp.stride(0)) if self.stacked else (0, 0)
        # (fields of the C structure)
        self._fields = (k.data_ptr(), v.data_ptr(), 0 if k_exp is None else k_exp.data_ptr(), 0 if v_exp is None else v_exp.data_ptr(), *stride,
                        k.shape[0] if self.stacked else 1, self.pages, self.kv_heads, KV_CODES[self.format])
        self._packed = _native.KV_PAGES.pack(*self._fields)

    @classmethod
    def alloc(cls, pages: int, kv_heads: int, device, *, kv_format="bf16", layers=None):
        """Empty pages (zeros)."""
        import torch

        if kv_format not in KV_CODES:
            raise ValueError(f"the cache's format is one of {tuple(KV_CODES)}")
        shape = (() if layers is None else (int(layers),)) + (int(pages), int(kv_heads), PAGE, HEAD_DIM)
        if kv_format == "q4":
            return cls(*(torch.zeros(*shape[:-2], Q4_ROWS, PAGE, device=device, dtype=torch.uint8) for _ in range(2)))
        if kv_format == "bf16":
            return cls(*(torch.zeros(shape, device=device, dtype=torch.bfloat16) for _ in range(2)))
        return cls(*(torch.zeros(shape, device=device, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)),
                   *(torch.zeros(shape[:-1], device=device, dtype=torch.uint8) for _ in range(2)))

    def layer(self, i: int) -> "KVPages":
        """One layer of a stack."""
        pick = lambda t: None if t is None else t[i]
        return KVPages(pick(self.k), pick(self.v), pick(self.k_exp), pick(self.v_exp))

    @property
    def entry_bytes(self) -> int:
        """Bytes of the cache per position, key or value head."""
        return {"bf16": 2 * HEAD_DIM, "e4m3": HEAD_DIM + 1, "q4": Q4_ROWS}[self.format]


def _table(page_table, device):
    """Fields of the C structure of a page table."""
    import torch

    slots, pages = page_table.shape if page_table.dim() == 2 else (0, 0)
    if not slots or not pages or page_table.stride(1) != 1:
        raise ValueError("the page table is [slots, pages], its rows contiguous")
    _on(page_table, device, torch.int32, "page table")
    return page_table.data_ptr(), _ld(page_table, pages, "page table"), slots, pages


def _kv_rows(name, k, v, row_seq, row_pos, page_table, pages):
    import torch

    if pages.stacked:
        raise ValueError("rows go to one layer: give pages.layer(i)")
    rows, device, width = row_seq.shape[0], pages.device, pages.kv_heads * HEAD_DIM
    shape = (rows, pages.kv_heads, HEAD_DIM)
    for t, what in ((k, "keys"), (v, "values")):
        _on(t, device, torch.bfloat16, what, shape)
        if rows and not (t.is_contiguous() or (t.stride(2) == 1 and t.stride(1) == HEAD_DIM)):
            raise ValueError(f"{what}: the heads of a row have to lie side by side")
    args = _native.KV_TABLE.pack(*_table(page_table, device)), _vector(row_seq, device, "row_seq"), _vector(row_pos, device, "row_pos", rows)
    ldk, ldv = _ld(k, width, "keys"), _ld(v, width, "values")
    if rows:
        _launch(device, name, pages._packed, *args, k.data_ptr(), ldk, v.data_ptr(), ldv, rows)


def kv_write(k, v, row_seq, row_pos, page_table, pages):
    """Stores rows of keys and values ([rows, kv heads, 128] BF16, as they are: rotated already) at positions ``row_pos`` of the
    sequences in slots ``row_seq``, quantised when the pages are.  Rows of slot -1 are left out; no two rows name the same place."""
    _kv_rows("grb_kv_write", k, v, row_seq, row_pos, page_table, pages)


def kv_read(row_seq, row_pos, page_table, pages, k_out, v_out):
    """Reads entries back as BF16 rows (exactly what they stand for).  Rows of slot -1 leave their outputs as they were."""
    _kv_rows("grb_kv_read", k_out, v_out, row_seq, row_pos, page_table, pages)


def kv_keep(slots, base, path, count, page_table, pages):
    """What verified draft trees keep, in every layer of ``pages``: of sequence i, the entries at ``base[i] + path[i, j]`` go to
    ``base[i] + j`` for j = 1 .. ``count[i]`` - 1.  ``path`` and ``count`` are the ``rows`` and ``count`` of
    ``sampling.DraftVerifier`` (paths ascend).  A slot of -1 is left out."""
    import torch

    n = slots.shape[0]
    if path.dim() != 2 or path.shape[0] != n or (path.shape[1] > 1 and path.stride(1) != 1):
        raise ValueError("path is [sequences, nodes], its rows contiguous")
    _on(path, pages.device, torch.int32, "path")
    device = pages.device
    args = _native.KV_TABLE.pack(*_table(page_table, device)), _vector(slots, device, "slots"), _vector(base, device, "base", n)
    kept, ldp = _vector(count, device, "count", n), _ld(path, path.shape[1], "path")
    if n and path.shape[1]:
        _launch(device, "grb_kv_keep", pages._packed, *args, path.data_ptr(), ldp, kept, n, path.shape[1])


# ---- pages as a whole -------------------------------------------------------------------------------------------------------


def _refs(refs, pages):
    return _vector(refs, pages.device, "refs", pages.pages)


def _empty(empty):
    if not -(1 << 31) <= empty < 1 << 31:
        raise ValueError("empty is a number of 32 bits")
    return int(empty)


def _whole_pages(pages):
    """Refuses exponents that cannot be moved in pieces of 16 bytes."""
    if pages.k_exp is not None and pages.stacked and pages.k_exp.shape[0] > 1 and pages.k_exp.stride(0) % 16:
        raise ValueError("exponents of keys and values: where whole pages are copied, layers lie a multiple of 16 bytes apart")


def kv_copy(src, dst, pages, *, positions=None):
    """Entries of page ``src[i]`` to page ``dst[i]`` (int32 vectors), keys and values, in every layer of ``pages``: all 256, or the first
    ``positions[i]``.  A page of -1 is left out; no page is a destination twice, or a source and a destination."""
    n, device = src.shape[0], pages.device
    args = _vector(src, device, "src"), _vector(dst, device, "dst", n), 0 if positions is None else _vector(positions, device, "positions", n)
    _whole_pages(pages)
    if n:
        _launch(device, "grb_kv_copy", pages._packed, *args, n)


def kv_fork(parents, children, lengths, fresh, page_table, refs, pages, *, empty=-1):
    """Sequences that begin as others: slot ``children[i]`` gets the first ``lengths[i]`` positions of slot ``parents[i]``.  Whole pages are
    shared, and are not to be written to while they are; the positions behind them are copied to page ``fresh[i]``, in every layer.
    ``refs`` (int32 [pages]) counts the places of the table that name a page and goes up for every page the child gets; the places behind
    its pages hold ``empty``.  What the child's slot held before is not given back (``kv_free`` it first).  A parent may have many children; no
    slot is a child twice, or a parent and a child, and no fresh page is in use.  Forks of slot -1 are left out."""
    n, device = parents.shape[0], pages.device
    args = _native.KV_TABLE.pack(*_table(page_table, device)), _vector(parents, device, "parents"), *(
        _vector(t, device, what, n) for t, what in ((children, "children"), (lengths, "lengths"), (fresh, "fresh"))), _refs(refs, pages), _empty(empty)
    _whole_pages(pages)
    if n:
        _launch(device, "grb_kv_fork", pages._packed, *args, n)


def kv_free(slots, page_table, refs, *, empty=-1):
    """Gives the pages of the sequences in ``slots`` back: their places in the table become ``empty``, and the counts in ``refs`` go down;
    a page is free when its count is 0.  Slots of -1 are left out."""
    device, n = refs.device, slots.shape[0]
    if device.type != "cuda":
        raise ValueError("refs live on a CUDA device")
    args = _native.KV_TABLE.pack(*_table(page_table, device)), _vector(slots, device, "slots"), _vector(refs, device, "refs")
    if n and refs.shape[0]:
        _launch(device, "grb_kv_free", *args, refs.shape[0], _empty(empty), n)


def kv_compact(page_table, refs, pages, where, used, *, scratch=None):
    """Moves the pages in use (``refs`` above 0) to the front of the pool, entries, counts and the places that name them: with u in use, the i-th
    at u or behind goes to the i-th free one before u.  ``where`` (int32 [pages]) receives each page's new number, -1 for pages that are not
    in use, and ``used`` (int32 [1]) u.  ``scratch``: uint8, ``kv_compact_scratch_bytes`` of it; allocated by the call if not given."""
    import torch

    device = pages.device
    args = _native.KV_TABLE.pack(*_table(page_table, device)), _refs(refs, pages), _vector(where, device, "where", pages.pages), _vector(used, device, "used", 1)
    size = kv_compact_scratch_bytes(pages)
    if scratch is None:
        with torch.cuda.device(device):
            scratch = torch.empty(size, device=device, dtype=torch.uint8)
    _on(scratch, device, torch.uint8, "scratch")
    if not scratch.is_contiguous():
        raise ValueError("scratch has to be contiguous")
    _whole_pages(pages)
    _launch(device, "grb_kv_compact", pages._packed, *args, scratch.data_ptr(), scratch.numel())


def kv_compact_scratch_bytes(pages) -> int:
    return _native.lib().grb_kv_compact_scratch_bytes(pages.pages)


# ---- rotary positions ---------------------------------------------------------------------------------------------------


ROPE_LAYOUTS = ("half", "interleaved")
_ROPE_KEYS = {"linear": ("factor",), "ntk": ("factor",), "yarn": ("factor", "original"), "bands": ("factor", "original", "low", "high")}
_ROPE_MORE = {"yarn": {"fast": 32.0, "slow": 1.0, "attention": None}}
_ROPE_DIGITS = decimal.Context(prec=40)
_PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def rope_frequencies(dim: int, theta: float = 1e4, scaling=None):
    """Radians a position of the dim / 2 pairs (Python floats), theta^(-2 i / dim) scaled for contexts longer than the trained one, and the
    factor on both components of a turned pair.  ``scaling`` is None or a dict:
      kind "linear", factor: every pair slower by the factor (positions interpolated);
      kind "ntk", factor: theta factor^(dim / (dim - 2)), under which the slowest pair is slower by the factor and the fastest as it was;
      kind "yarn", factor, original (the trained context), fast=32, slow=1, attention=None: pairs that turn ``fast`` times or more within the
        trained context stay, those that turn ``slow`` times or fewer are slower by the factor, between the pairs' numbers it is a ramp; both
        components are multiplied by ``attention``, where it is None 0.1 ln(factor) + 1, and 1 for a factor below one (Peng et al., 2023);
      kind "bands", factor, original, low, high: the same with the ramp over the turns themselves, between ``low`` and ``high``, and no factor."""
    frequencies, factor = _rope_frequencies(dim, theta, scaling)
    return [float(f) for f in frequencies], factor


def _rope_frequencies(dim, theta, scaling):
    """``rope_frequencies`` to 36 digits or more: a position of millions multiplies what its frequency is off by."""
    if dim < 2 or dim % 2:
        raise ValueError("the turned dimensions are an even number of two or more")
    if not 0 < theta < float("inf"):
        raise ValueError("theta is positive")
    given = dict(scaling or {"kind": None})
    kind = given.pop("kind", None)
    if kind is not None:
        if kind not in _ROPE_KEYS:
            raise ValueError(f"the scaling's kind is one of {tuple(_ROPE_KEYS)}")
        given = {**_ROPE_MORE.get(kind, {}), **given}
        if set(given) != {*_ROPE_KEYS[kind], *_ROPE_MORE.get(kind, {})}:
            raise ValueError(f"scaling {kind!r} takes {(*_ROPE_KEYS[kind], *_ROPE_MORE.get(kind, {}))}")
        if any(v is None or not 0 < v < float("inf") for name, v in given.items() if v is not None or name != "attention"):
            raise ValueError("the numbers of a scaling are positive")
    elif given:
        raise ValueError("a scaling has a kind")
    if kind == "yarn" and (theta == 1 or given["fast"] <= given["slow"]):
        raise ValueError("yarn needs a theta other than 1 and fast above slow")
    if kind == "bands" and given["low"] >= given["high"]:
        raise ValueError("low lies below high")
    with decimal.localcontext(_ROPE_DIGITS):
        number = {name: None if v is None else Decimal(float(v)) for name, v in given.items()}
        base, factor, attention = Decimal(float(theta)).ln(), number.get("factor"), 1.0
        if kind == "ntk" and dim > 2:
            base += factor.ln() * dim / (dim - 2)
        ratio, inv = (base * -2 / dim).exp(), [Decimal(1)]
        while 2 * len(inv) < dim:
            inv.append(inv[-1] * ratio)           # (off by 10^-39 a pair)
        if kind == "linear":
            inv = [f / factor for f in inv]
        elif kind == "yarn":
            pair = lambda turns: (number["original"] / (2 * _PI * turns)).ln() / base * dim / 2
            lo, hi = max(math.floor(pair(number["fast"])), 0), min(math.ceil(pair(number["slow"])), dim - 1)
            width = max(Decimal(hi - lo), Decimal("0.001"))
            slow = [min(max((i - lo) / width, 0), 1) for i in range(dim // 2)]
            inv = [f / factor * s + f * (1 - s) for f, s in zip(inv, slow)]
            attention = 0.1 * math.log(max(given["factor"], 1.0)) + 1 if given["attention"] is None else float(given["attention"])
        elif kind == "bands":
            turns, width = number["original"] / (2 * _PI), number["high"] - number["low"]
            keep = [min(max((f * turns - number["low"]) / width, 0), 1) for f in inv]
            inv = [f / factor * (1 - k) + f * k for f, k in zip(inv, keep)]
        if max(inv) >= 1 << 60:                   # (whose fraction of a turn would not be known to 2^-64)
            raise ValueError("a position turns a pair by less than 2^60 radians")
    return inv, attention


class Rope:
    """Rotary positions of the first ``dim`` dimensions of a head: pairs (i, i + dim / 2) (``layout`` "half") or (2 i, 2 i + 1)
    ("interleaved"), frequencies by ``theta`` and ``scaling`` (``rope_frequencies``), held on the device as the nearest 64-bit fractions of a turn."""

    def __init__(self, dim: int, theta: float = 1e4, *, layout="half", scaling=None, device="cuda:0"):
        import torch

        if layout not in ROPE_LAYOUTS:
            raise ValueError(f"the layout is one of {ROPE_LAYOUTS}")
        self.dim, self.layout = int(dim), layout
        frequencies, self.factor = _rope_frequencies(self.dim, theta, scaling)
        self.frequencies = [float(f) for f in frequencies]
        with decimal.localcontext(_ROPE_DIGITS):
            units = (1 << 64) / (2 * _PI)         # of a radian
            turns = [round(f * units) % (1 << 64) for f in frequencies]
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64).to(device)
        self.device = self.turns.device

    def tables(self, positions: int):
        """BF16 cos / sin tables [positions, 128] as the attention takes them, with the factor: for all 128 dimensions in halves."""
        import torch

        if self.dim != HEAD_DIM or self.layout != "half":
            raise ValueError("the attention's tables are of 128 dimensions in halves")
        angle = torch.arange(positions, dtype=torch.float64)[:, None] * torch.tensor(self.frequencies, dtype=torch.float64)
        angle = torch.cat([angle, angle], dim=1)
        return tuple((f(angle) * self.factor).to(torch.bfloat16).to(self.device) for f in (torch.cos, torch.sin))


def rotary(x, positions, rope, *, out=None, backward=False):
    """Turns the first ``rope.dim`` dimensions of every head of ``x`` ([rows, heads, head dim] BF16, FP16 or FP32; rows and heads may be any distance apart) by
    ``positions`` (int32 or int64 [rows]), into ``out`` - memory apart from that of ``x``, from its first to its last element - or, without it, in place.  An angle is off by 2^-32 of a turn at most, and 2^-65 of one for
    every position (2^-25 at 2^40); a value is rounded once.  ``backward``: turned the other way - the gradient of the call, given that of its result, and where ``rope.factor`` is 1 its inverse."""
    import torch

    device = rope.device
    out = x if out is None else out
    kinds = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
    if x.dim() != 3 or x.dtype not in kinds or x.device != device or device.type != "cuda":
        raise ValueError("x is BF16, FP16 or FP32 [rows, heads, head dim] on the rope's device, a CUDA device")
    rows, heads, dim = x.shape
    if rope.dim > dim:
        raise ValueError(f"{rope.dim} dimensions are turned, a head has {dim}")
    _on(out, device, x.dtype, "out", x.shape)
    if positions.dim() != 1 or positions.shape[0] != rows or not positions.is_contiguous() or positions.device != device or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions: a contiguous int32 or int64 vector of {rows} is wanted")
    if not rows or not heads:
        return out
    for t, what in ((x, "x"), (out, "out")):
        if dim > 1 and t.stride(2) != 1:
            raise ValueError(f"{what}: the dimensions of a head have to be contiguous")
    if out is not x:
        span = [(t.data_ptr(), t.data_ptr() + t.element_size() * (t.stride(0) * (rows - 1) + t.stride(1) * (heads - 1) + dim)) for t in (x, out)]
        if span[0][0] < span[1][1] and span[1][0] < span[0][1] and (x.data_ptr() != out.data_ptr() or x.stride() != out.stride()):
            raise ValueError("x and out overlap: give the same tensor, or tensors apart")
    wide = positions.dtype == torch.int64
    step = _native.ROTARY_STEP.pack(x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1), positions.data_ptr(), rope.turns.data_ptr(),
                                    rows, heads, dim, rope.dim, ROPE_LAYOUTS.index(rope.layout), kinds[x.dtype], wide, bool(backward), rope.factor)
    _launch(device, "grb_rotary", step)
    return out


class TreeRows:
    """What makes rows nodes of draft trees: ``base`` (int32 [rows]): positions below it are seen by the row; ``rope`` (int32
    [rows]): the row's rotary position, base + its depth; ``mask`` (int64 [rows, words], 1 to 4 words): bit j of word w says
    that the row sees position base + 64 w + j.  A node's entry is stored at its ``row_pos``, mostly base + its number."""

    def __init__(self, base, rope, mask):
        import torch

        rows = base.shape[0]
        if mask.dim() != 2 or mask.shape[0] != rows or not 1 <= mask.shape[1] <= MASK_WORDS or (mask.shape[1] > 1 and mask.stride(1) != 1):
            raise ValueError(f"mask is [rows, 1 to {MASK_WORDS} words], its rows contiguous")
        _on(mask, base.device, torch.int64, "mask")
        _vector(base, base.device, "base", rows)
        _vector(rope, base.device, "rope", rows)
        self.rows, self.device = rows, base.device
        self.base, self.rope, self.mask = base, rope, mask
        # (fields of the C structure)
        self._fields = base.data_ptr(), rope.data_ptr(), mask.data_ptr(), _ld(mask, mask.shape[1], "mask"), mask.shape[1]

    @staticmethod
    def masks(parents, words=None):
        """Depths and masks (Python integers, ``words`` of 64 bits each) of a tree given by its nodes' parents (-1: a root),
        parents before children: every node sees its ancestors and itself."""
        depth, seen = [], []
        for i, p in enumerate(parents):
            if not -1 <= p < i:
                raise ValueError("a node's parent comes before it")
            depth.append(0 if p < 0 else depth[p] + 1)
            seen.append((1 << i) | (0 if p < 0 else seen[p]))
        words = words or max(1, -(-len(parents) // 64))
        if len(parents) > 64 * words or words > MASK_WORDS:
            raise ValueError(f"{len(parents)} nodes do not fit {min(words, MASK_WORDS)} words")
        signed = lambda m: m - (1 << 64) if m >> 63 else m
        return depth, [[signed(m >> (64 * w) & ((1 << 64) - 1)) for w in range(words)] for m in seen]


class TreeAttention:
    """Attention over a cache in BF16, 8 or 4 bits, for causal rows and for nodes of draft trees: scratch and geometry for up to
    ``max_rows`` rows a call and ``max_pages`` pages a sequence; ``__call__`` runs rotary embedding, append and attention for one
    layer.  Up to 16 query heads per kv head.  Calls that may run at the same time need an object each: they share its scratch."""

    def __init__(self, nq: int, nkv: int, max_rows: int, max_pages: int, device, *, kv_format="bf16"):
        import torch

        if kv_format not in KV_CODES:
            raise ValueError(f"the cache's format is one of {tuple(KV_CODES)}")
        if nq < 1 or nkv < 1 or nq % nkv or nq // nkv > 16:
            raise ValueError("query heads per kv head: a whole number up to 16")
        if not 1 <= max_rows <= TREE_ROWS or max_pages < 1:
            raise ValueError(f"1 to {TREE_ROWS} rows and at least one page")
        self.nq, self.nkv, self.max_rows, self.max_pages, self.format = nq, nkv, int(max_rows), int(max_pages), kv_format
        self.scratch_bytes = _native.lib().grb_attn_tree_scratch_bytes(self.max_rows, nq, self.max_pages, KV_CODES[kv_format])
        self.scratch = torch.empty(self.scratch_bytes, device=device, dtype=torch.uint8)
        self.scratch[:16].zero_()
        self.status = self.scratch[:4].view(torch.int32)
        self.device = self.scratch.device
        self._bf16, self._scaling, self._width = torch.bfloat16, 1.0 / math.sqrt(HEAD_DIM), ((nq + 2 * nkv) * HEAD_DIM, nq * HEAD_DIM)

    def check_status(self) -> int:
        """GRB_STATUS_* bits of the calls since the last check (0: their outputs can be trusted).  Synchronises."""
        bits = int(self.status.item())
        self.status.zero_()
        return bits

    def __call__(self, qkv, cos, sin, row_seq, row_pos, page_table, pages, out, *, tree=None, longest_run=None):
        """``qkv`` (BF16 [rows, (nq + 2 nkv) 128]) -> ``out`` (BF16 [rows, nq 128]).  Keys (rotated) and values are stored at
        ``row_pos`` of the sequences in slots ``row_seq`` before any row reads.  Without ``tree`` row r sees positions up to its
        own; with ``TreeRows`` what they say, a row that sees nothing giving zeros.  Rows of slot -1 are left out; no two rows name the
        same place.
        ``longest_run``: how many rows of one sequence follow one another, at most, where the caller knows it; runs of 64 causal rows
        or of more than 32 tree rows and heads are multiplied together (without it: tree rows are, causal rows are taken as steps
        of decoding - a prompt's rows are as right, and slower)."""
        device, bf, (wide, narrow) = self.device, self._bf16, self._width
        rows = qkv.shape[0]
        if rows > self.max_rows or (page_table.dim() == 2 and page_table.shape[1] > self.max_pages):
            raise ValueError("more rows or pages than the scratch was sized for")
        if pages.format != self.format or pages.stacked or pages.kv_heads != self.nkv or pages.device != device:
            raise ValueError("pages of one layer, in this object's format, heads and device")
        _on(qkv, device, bf, "qkv", (rows, wide))
        _on(out, device, bf, "out", (rows, narrow))
        _on(cos, device, bf, "cos")
        _on(sin, device, bf, "sin", cos.shape)
        if cos.dim() != 2 or cos.shape[1] != HEAD_DIM or not cos.is_contiguous() or not sin.is_contiguous():
            raise ValueError("rotary tables are contiguous [positions, 128]")
        if longest_run is not None and longest_run < 1:
            raise ValueError("longest_run is at least 1")
        if not rows:
            return
        if qkv.stride(1) != 1 or out.stride(1) != 1:
            raise ValueError("rows of qkv and out have to be contiguous")
        nodes = (0, 0, 0, 0, 0)
        if tree is not None:
            if tree.rows != rows or tree.device != device:
                raise ValueError("tree rows: one for each row, on the same device")
            nodes = tree._fields
        step = _native.TREE_STEP.pack(
            qkv.data_ptr(), _ld(qkv, wide, "qkv"), cos.data_ptr(), sin.data_ptr(), cos.shape[0], _vector(row_seq, device, "row_seq", rows),
            _vector(row_pos, device, "row_pos", rows), *nodes, *pages._fields, *_table(page_table, device), self.scratch.data_ptr(), self.scratch_bytes,
            out.data_ptr(), _ld(out, narrow, "out"), rows, self.nq, HEAD_DIM, self._scaling, longest_run or 0)
        _launch(device, "grb_attn_tree", step)
