"""Operators of serving long contexts from a 4-bit KV cache, as cases that can be timed: a cache that is quantised to 4 bits as
it is written and read back, attention of decode rows, prompt chunks and draft trees over it, rotary positions in every layout
and scaling, and the pages of a cache forked, freed and compacted.

Ranges.  Heads: those of the benchmark's decoder and of its 2- and 4-way tensor-parallel shards, and of a 4096-wide model.
Cache rows: 1 to 2048 tokens of 1 to 16 sequences.  Attention: 1 to 128 sequences with 1 to 32768 positions, 1 to 8 causal rows each,
prompt chunks of 64 to 384 rows, or 2 to 64 tree nodes each.  Rotary positions: 1 to 8192 rows of 1 to 56 heads of 64 to 256
dimensions, all or part of them turned, both layouts, three types, positions to a million.  Pages: 1 to 16 sequences forked into 1 to 8 branches,
pools of 8 to 512 pages compacted, 1 to 64 layers, all formats.  Pages are scattered and sequences are ragged everywhere.

A 4-bit entry is 128 values of one key or value head at one position, in four groups of 32.  With a = max |x| of the entry, its
exponent is e = clamp(floor(log2(a / 7)) + 9, -40, 22), kept as the byte e + 127.  A group's scale is the number nearest to max |x| / 7 / 2^(e - 24),
max over the group, among (16 + m) 2^k with m = 0 .. 15, k = 0 .. 11 (ties to even m), kept as the byte 64 + 16 k + m.  A value's code is the
whole number nearest to x / (scale 2^(e - 24)) (ties to even) in -7 .. 7, kept as a nibble, code + 8; it stands for code * scale * 2^(e - 24).
A byte below 16 is the scale byte / 8, so that memory of zeros reads as zeros.
A page of one head is 69 rows of 256 bytes: the codes of its 256 positions (64 bytes each), their scales (4 bytes each), their exponents.
The eight codes of dimensions 8 w .. 8 w + 7 share four bytes: (0, 2), (4, 6), (1, 3), (5, 7), the first of each pair in the lower nibble.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DIM, PAGE = 128, 256
ENTRY = 69                                          # bytes of a 4-bit entry; rows of 256 bytes of a page
SCALES, EXPONENTS = 64 * PAGE, 68 * PAGE            # where a page's scales and exponents begin
SHAPES = ((40, 8), (20, 4), (10, 2), (32, 8))       # query and KV heads: the benchmark's decoder, its shards, a smaller model
ORDER = (0, 2, 4, 6, 1, 3, 5, 7)                    # dimensions of eight in the order of their nibbles
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a prompt's last chunk stored in the 4-bit cache and read back: latency of the two calls
        {"name": "write_384", "op": "write", "seqs": 1, "tokens": 384, "kv_heads": 8},
        # sixteen sequences taken over from another cache
        {"name": "write_16x2048", "op": "write", "seqs": 16, "tokens": 2048, "kv_heads": 8},
        # one interactive sequence's decode step
        {"name": "step_1", "op": "attend", "seqs": 1, "rows": 1, "context": 2048, "heads": 40, "kv_heads": 8},
        # a full batch's decode step
        {"name": "step_128", "op": "attend", "seqs": 128, "rows": 1, "context": 2048, "heads": 40, "kv_heads": 8},
        # a decode step of a few long documents
        {"name": "step_8_long", "op": "attend", "seqs": 8, "rows": 1, "context": 32768, "heads": 40, "kv_heads": 8},
        # a chunk of a prompt behind what has been taken in
        {"name": "prompt_384", "op": "attend", "seqs": 1, "rows": 384, "context": 8000, "heads": 40, "kv_heads": 8},
        # wide draft trees of a batch over long contexts: as much arithmetic as traffic
        {"name": "tree_16x64", "op": "tree", "seqs": 16, "nodes": 64, "context": 8192, "heads": 40, "kv_heads": 8},
        # queries and keys of one decode step, half of a head's dimensions turned, neighbours paired
        {"name": "rotary_1", "op": "rotary", "rows": 1, "heads": 48, "dim": 128, "turned": 64, "layout": "interleaved", "dtype": "bf16", "scaling": "none", "far": 2048},
        # queries and keys of a long prompt far behind the trained context
        {"name": "rotary_8192", "op": "rotary", "rows": 8192, "heads": 48, "dim": 128, "turned": 128, "layout": "half", "dtype": "bf16", "scaling": "yarn", "far": 1000000},
        # one sequence's two continuations, in a stack cut to 4 layers; and eight of each of a batch, in all 64
        {"name": "fork_1x2", "op": "fork", "seqs": 1, "branches": 2, "context": 1000, "layers": 4, "kv_heads": 8, "format": "q4"},
        {"name": "fork_8x8", "op": "fork", "seqs": 8, "branches": 8, "context": 2048, "layers": 64, "kv_heads": 8, "format": "q4"},
        # a pool of which half the sequences have ended, in all 64 layers
        {"name": "compact_64", "op": "compact", "pool": 128, "layers": 64, "kv_heads": 8, "format": "q4"},
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "attend", "attend", "prompt", "tree", "rotary", "rotary", "fork", "compact"))
    heads, kv_heads = rng.choice(SHAPES)
    kind = rng.choice(("q4", "q4", "bf16", "e4m3"))
    if op == "write":
        return {"op": op, "seqs": _spread(rng, 1, 16), "tokens": _spread(rng, 1, 2048), "kv_heads": kv_heads}
    if op == "attend":
        context = _spread(rng, 1, 32768)
        return {"op": op, "seqs": _spread(rng, 1, min(128, 262144 // context)), "rows": rng.randint(1, 8), "context": context, "heads": heads, "kv_heads": kv_heads}
    if op == "prompt":
        return {"op": "attend", "seqs": rng.randint(1, 2), "rows": _spread(rng, 64, 384), "context": _spread(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads}
    if op == "tree":
        context = _spread(rng, 1, 8192)
        return {"op": op, "seqs": _spread(rng, 1, min(64, 131072 // context)), "nodes": _spread(rng, 2, 64), "context": context, "heads": heads, "kv_heads": kv_heads}
    if op == "rotary":
        dim = rng.choice((64, 80, 96, 128, 128, 256))
        return {"op": op, "rows": _spread(rng, 1, 8192), "heads": rng.randint(1, 56) if dim <= 128 else rng.randint(1, 24), "dim": dim,
                "turned": rng.choice((dim, dim, dim // 2, dim // 4)), "layout": rng.choice(("half", "interleaved")),
                "dtype": rng.choice(("bf16", "bf16", "fp16", "fp32")), "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands")), "far": _spread(rng, 16, 1000000)}
    most = 8192 * ENTRY // _per_entry({"format": kind})      # pages of all layers
    if op == "fork":
        seqs, branches = rng.randint(1, 16), rng.randint(1, 8)
        return {"op": op, "seqs": seqs, "branches": branches, "context": _spread(rng, 1, 2048), "layers": _spread(rng, 1, min(64, most // (seqs * (8 + branches)))),
                "kv_heads": kv_heads, "format": kind}
    layers = _spread(rng, 1, 64)
    return {"op": op, "pool": _spread(rng, 8, min(512, most // layers)), "layers": layers, "kv_heads": kv_heads, "format": kind}


def _share(i, most, least=0.5):
    """The i-th of a ragged series of lengths between least * most and most."""
    return max(1, int(most * (1 - (1 - least) * ((i * 0.6180339887) % 1.0))))


def _lengths(case):
    """Cached positions of every sequence before the call."""
    return [_share(i, case["context"]) for i in range(case["seqs"])]


def _held_pages(case):
    """Pages in use of a pool to be compacted, as a list of truth values: about half, more of them low."""
    pool = case["pool"]
    return [(i * 0.6180339887) % 1.0 < 0.7 - 0.4 * i / pool for i in range(pool)]


def _per_entry(case):
    return {"q4": ENTRY, "e4m3": DIM + 1, "bf16": 2 * DIM}[case["format"]]


def work(case):
    op = case["op"]
    if op == "write":
        n = case["seqs"] * case["tokens"] * case["kv_heads"] * 2
        return {"bytes": n * 2 * (2 * DIM + ENTRY), "flops": 0}
    if op in ("attend", "tree"):
        rows, heads, kv = case["rows"] if op == "attend" else case["nodes"], case["heads"], case["kv_heads"]
        seen = sum(n * rows + (rows * (rows + 1) // 2 if op == "attend" else rows) for n in _lengths(case))
        return {"bytes": 2 * kv * sum(n + rows for n in _lengths(case)) * ENTRY + rows * case["seqs"] * 2 * DIM * (2 * heads + 2 * kv), "flops": 4 * DIM * heads * seen}
    if op == "rotary":
        n = case["rows"] * case["heads"]
        return {"bytes": n * case["dim"] * 2 * TYPES[case["dtype"]].itemsize + 4 * case["rows"], "flops": 3 * n * case["turned"]}
    if op == "fork":
        rest = sum(n % PAGE for n in _lengths(case))          # positions of the last pages: read once for all branches, written for each
        return {"bytes": rest * (1 + case["branches"]) * 2 * case["kv_heads"] * _per_entry(case) * case["layers"], "flops": 0}
    held = _held_pages(case)
    return {"bytes": 2 * sum(held[sum(held):]) * PAGE * 2 * case["kv_heads"] * _per_entry(case) * case["layers"], "flops": 0}


# ---- the plain forms ----------------------------------------------------------------------------------------------------


def _power(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _scale(byte):
    """What a scale's byte stands for."""
    byte = byte.int()
    return torch.where(byte < 16, byte.float() / 8, (16 + (byte & 15)).float() * _power((byte >> 4) - 4))


def _quantise(x):
    """FP32 vectors [..., 128] -> packed codes [..., 64], scale bytes [..., 4], exponent bytes [...].  In 64 bits: quotients next to a
    border."""
    x = x.double()
    top = x.abs().amax(-1) / 7
    e = torch.where(top > 0, torch.frexp(top)[1] + 8, -40).clamp(-40, 22)            # top = m 2^k with m in [0.5, 1): floor(log2) = k - 1
    unit = _power(e).double()[..., None] * 2.0 ** -24
    groups = x.unflatten(-1, (4, 32))
    want = (groups.abs().amax(-1) / 7 / unit).clamp(16, 31 * 2048)
    k = (torch.frexp(want)[1] - 5).clamp(0, 11)                                      # want / 2^k in [16, 32)
    m = torch.round(want / _power(k).double()).int()
    byte = (48 + 16 * k + m).clamp(max=255)                                          # (m = 32: the first of the next k)
    code = torch.round(groups / (_scale(byte).double() * unit)[..., None]).clamp(-7, 7).to(torch.int32).flatten(-2)
    nibble = (code + 8).unflatten(-1, (16, 8))[..., ORDER].unflatten(-1, (4, 2))
    return (nibble[..., 0] | (nibble[..., 1] << 4)).flatten(-2).to(torch.uint8), byte.to(torch.uint8), (e + 127).to(torch.uint8)


def _values(codes, scales, exponents):
    """FP32 vectors [..., 128] of packed codes [..., 64], scale bytes [..., 4] and exponent bytes [...]."""
    nibble = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).unflatten(-1, (16, 8))
    back = [ORDER.index(i) for i in range(8)]
    code = nibble[..., back].flatten(-2).float() - 8
    return (code.unflatten(-1, (4, 32)) * _scale(scales)[..., None]).flatten(-2) * (_power(exponents.int().clamp(min=87) - 127) * 2.0 ** -24)[..., None]


def _parts(pages):
    """Views of 4-bit pages [..., 69, 256]: codes [..., 256, 64], scales [..., 256, 4], exponents [..., 256]."""
    flat = pages.flatten(-2)
    return flat[..., :SCALES].unflatten(-1, (PAGE, 64)), flat[..., SCALES:EXPONENTS].unflatten(-1, (PAGE, 4)), flat[..., EXPONENTS:]


def _stored(state, which):
    """All sequences' keys or values as FP32 [seqs, positions, kv heads, 128], through the page table."""
    return _values(*_parts(state[which][state["page_table"].long()])).transpose(2, 3).flatten(1, 2)


def _places(s):
    return s["page_table"].long()[s["row_seq"].long(), s["row_pos"].long() // PAGE], s["row_pos"].long() % PAGE


def _store(s, which, x):
    """Puts FP32 rows [rows, kv heads, 128] where the rows' sequences and positions say."""
    page, at = _places(s)
    for view, part in zip(_parts(s[which]), _quantise(x)):
        view[page, :, at] = part


def _rotate(x, cos, sin):
    """Rotate-half: FP32 [rows, heads, 128] by tables [rows, 128]."""
    half = DIM // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    return x * cos[:, None].float() + turned * sin[:, None].float()


def _write_plain(s):
    page, at = _places(s)
    out = []
    for which in ("k", "v"):
        _store(s, which, s[which + "_in"].float())
        out.append(_values(*(view[page, :, at] for view in _parts(s[which]))).to(torch.bfloat16))
    return out


def _attention_plain(s):
    """Appends the rows' keys and values, then every row attends to what it may see."""
    nq, nkv, n, per = s["heads"], s["kv_heads"], s["seqs"], s["per_seq"]
    qkv = s["qkv"].float().view(n * per, nq + 2 * nkv, DIM)
    rope = (s["row_pos"] if s["mask"] is None else s["rope"]).long()
    cos, sin = s["cos"][rope], s["sin"][rope]
    q = _rotate(qkv[:, :nq], cos, sin)
    _store(s, "k", _rotate(qkv[:, nq:nq + nkv], cos, sin))
    _store(s, "v", qkv[:, nq + nkv:])
    k, v = _stored(s, "k"), _stored(s, "v")
    position = torch.arange(k.shape[1], device=k.device)
    if s["mask"] is None:
        seen = position <= s["row_pos"].long().view(n, per, 1)
    else:
        node = position - s["base"].long().view(n, per, 1)
        bit = (s["mask"].view(n, per, 1) >> node.clamp(0, 63)) & 1
        seen = (node < 0) | ((node < 64) & (bit == 1))
    score = torch.einsum("nrgid,npgd->ngirp", q.view(n, per, nkv, nq // nkv, DIM), k) / math.sqrt(DIM)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.einsum("ngirp,npgd->nrgid", weight / weight.sum(-1, keepdim=True), v)
    return out.reshape(n * per, nq * DIM).to(torch.bfloat16)


def _frequencies(case):
    """Radians a position of every turned pair, in 64 bits, and the factor on both components."""
    theta, scaling, turned = 1e6, SCALINGS[case["scaling"]], case["turned"]
    i = torch.arange(turned // 2, dtype=torch.float64, device=DEVICE)
    factor, kind = scaling.get("factor", 1.0), scaling.get("kind")
    if kind == "ntk":                              # a larger base, under which the slowest pair is slowed by the factor
        theta = theta * factor ** (turned / (turned - 2)) if turned > 2 else theta
    inv = theta ** (-2 * i / turned)
    if kind == "linear":
        return inv / factor, 1.0
    if kind == "yarn":                             # pairs that turn often within the trained context keep their speed, slow ones are slowed
        index = lambda turns: turned / 2 * math.log(scaling["original"] / (2 * math.pi * turns)) / math.log(theta)
        lo, hi = max(math.floor(index(scaling["fast"])), 0), min(math.ceil(index(scaling["slow"])), turned - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return inv / factor * slow + inv * (1 - slow), 0.1 * math.log(factor) + 1
    if kind == "bands":                            # the same by the number of turns within the trained context
        turns = scaling["original"] * inv / (2 * math.pi)
        keep = ((turns - scaling["low"]) / (scaling["high"] - scaling["low"])).clamp(0, 1)
        return inv / factor * (1 - keep) + inv * keep, 1.0
    return inv, 1.0


SCALINGS = {"none": {}, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 8.0},
            "yarn": {"kind": "yarn", "factor": 32.0, "original": 32768, "fast": 32.0, "slow": 1.0},
            "bands": {"kind": "bands", "factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}


def _rotary_plain(s):
    """Turns the first dimensions of every head: pairs (i, i + turned / 2), or (2 i, 2 i + 1).  Angles in 64 bits: far positions."""
    angle = s["positions"].double()[:, None] * s["inv"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))
    x, n = s["x"].float(), s["turned"]
    if s["layout"] == "half":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., n:]], dim=-1).to(s["x"].dtype)


def _free_plain(table, refs, slots):
    """Takes the slots' pages away: the pages' counts go down, the places become -1."""
    pages = table[slots.long()].flatten().long()
    refs.scatter_add_(0, pages.clamp(min=0), -(pages >= 0).int())
    table[slots.long()] = -1


def _fork_plain(s):
    """Children get their parents' pages: whole ones are shared and counted, of the last one a fresh page gets the positions in use."""
    table, refs, lengths = s["page_table"], s["refs"], s["lengths"].long()
    _free_plain(table, refs, s["children"])
    rows = table[s["parents"].long()]
    place = torch.arange(table.shape[1], device=table.device)
    whole = place < (lengths // PAGE)[:, None]
    last = (place == (lengths // PAGE)[:, None]) & (lengths % PAGE > 0)[:, None]
    rows = torch.where(whole, rows, torch.where(last, s["fresh"][:, None], -1))
    source = table[s["parents"].long()].gather(1, (lengths // PAGE).clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    table[s["children"].long()] = rows
    refs.scatter_add_(0, rows.flatten().long().clamp(min=0), (rows >= 0).flatten().int())
    used = torch.arange(PAGE, device=table.device) < (lengths % PAGE)[:, None]
    fork, at = used.nonzero(as_tuple=True)
    source, target = source[fork], s["fresh"].long()[fork]
    for which in ("k", "v"):
        for x in ([s[which]] if s["format"] == "bf16" else [s[which].view(torch.uint8), s[which + "_exp"]] if s["format"] == "e4m3" else _parts(s[which])):
            x[:, target, :, at] = x[:, source, :, at]


def _compact_plain(s):
    """The i-th page in use, of those behind as many as there are in use, goes to the i-th free one before them."""
    table, refs = s["page_table"], s["refs"]
    table.copy_(s["table_before"])
    refs.copy_(s["refs_before"])
    held = refs > 0
    used = held.sum()
    number = torch.arange(refs.shape[0], device=refs.device)
    source, target = (held & (number >= used)).nonzero()[:, 0], (~held & (number < used)).nonzero()[:, 0]
    where = torch.where(held, number, -1)
    where[source] = target
    for which in ("k", "v"):
        for x in (s[which], s[which + "_exp"]):
            if x is not None:
                x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
                x[:, target] = x[:, source]
    refs[target] = refs[source]
    refs[source] = 0
    table.copy_(torch.where(table >= 0, where[table.clamp(min=0).long()], -1))
    return where.int(), used.int()[None]


# ---- inputs -------------------------------------------------------------------------------------------------------------


def _vectors(g, *shape):
    """Keys or values as a cache meets them: normal, some channels larger, positions of different size."""
    x = torch.randn(*shape, generator=g, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEVICE))
    return x * torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=g, device=DEVICE))


def _pages(x):
    """Vectors [pages, kv heads, 256, 128] as 4-bit pages [pages, kv heads, 69, 256]."""
    pages = torch.empty(*x.shape[:2], ENTRY, PAGE, device=DEVICE, dtype=torch.uint8)
    for lo in range(0, x.shape[0], 256):                       # (64 bits of all pages at once would take four times their FP32 size)
        for view, part in zip(_parts(pages[lo:lo + 256]), _quantise(x[lo:lo + 256])):
            view.copy_(part)
    return pages


def _page_table(g, lengths, empty=0):
    """Pages for the given lengths, scattered over the pool; `empty` in the places behind a sequence's pages."""
    need = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device=DEVICE)
    table = torch.full((len(need), max(need)), empty, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].int()
        at += n
    return table, sum(need)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, generator=g, device=DEVICE, dtype=torch.uint8)


def _parents(nodes, pick):
    """A draft tree: node 0 is the pending token; every other node hangs below an earlier one, the first few levels wide."""
    parents = [-1]
    for i in range(1, nodes):
        low = (i - 1) // 3
        parents.append(low + int(pick[i] * (i - low)))
    return parents


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 17)
    return {"write": _prepare_write, "attend": _prepare_attention, "tree": _prepare_attention, "rotary": _prepare_rotary, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["op"]](case, g)


def _prepare_write(case, g):
    n, nkv = case["tokens"], case["kv_heads"]
    s = {"op": "write"}
    s["page_table"], pages = _page_table(g, [n] * case["seqs"])
    s["k"], s["v"] = (torch.zeros(pages, nkv, ENTRY, PAGE, device=DEVICE, dtype=torch.uint8) for _ in range(2))
    rows = case["seqs"] * n
    s["row_seq"] = torch.arange(case["seqs"], device=DEVICE).repeat_interleave(n).int()
    s["row_pos"] = torch.arange(n, device=DEVICE).repeat(case["seqs"]).int()
    s["k_in"], s["v_in"] = (_vectors(g, rows, nkv, DIM).to(torch.bfloat16) for _ in range(2))
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"])
        s["k_out"], s["v_out"] = torch.empty_like(s["k_in"]), torch.empty_like(s["v_in"])
    return s


def _prepare_attention(case, g):
    nq, nkv, n = case["heads"], case["kv_heads"], case["seqs"]
    tree = case["op"] == "tree"
    per = case["nodes"] if tree else case["rows"]
    lengths = _lengths(case)
    s = {"op": case["op"], "heads": nq, "kv_heads": nkv, "seqs": n, "per_seq": per, "mask": None}
    s["page_table"], pages = _page_table(g, [length + per for length in lengths])
    s["k"], s["v"] = (_pages(_vectors(g, pages, nkv, PAGE, DIM)) for _ in range(2))
    inv = 1e6 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device=DEVICE) / DIM)
    angle = torch.arange(max(lengths) + per, dtype=torch.float64, device=DEVICE)[:, None] * inv
    angle = torch.cat([angle, angle], dim=1)
    s["cos"], s["sin"] = angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)
    s["row_seq"] = torch.arange(n, device=DEVICE).repeat_interleave(per).int()
    s["row_pos"] = _ints([length + j for length in lengths for j in range(per)])
    s["qkv"] = torch.cat([1.5 * torch.randn(n * per, nq * DIM, generator=g, device=DEVICE), _vectors(g, n * per, 2 * nkv, DIM).flatten(1)], dim=1).to(torch.bfloat16)
    if tree:
        pick = torch.rand(n, per, generator=g, device=DEVICE).tolist()
        rope, mask = [], []
        for length, p in zip(lengths, pick):
            depth, seen = [], []
            for i, up in enumerate(_parents(per, p)):
                depth.append(0 if up < 0 else depth[up] + 1)
                seen.append((1 << i) | (0 if up < 0 else seen[up]))
            rope += [length + d for d in depth]
            mask += [m - (1 << 64) if m >> 63 else m for m in seen]
        s["rope"], s["base"] = _ints(rope), _ints([length for length in lengths for _ in range(per)])
        s["mask"] = torch.tensor(mask, dtype=torch.int64, device=DEVICE)[:, None]
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"])
        s["attention"] = ops.TreeAttention(nq, nkv, n * per, s["page_table"].shape[1], DEVICE, kv_format="q4")
        s["tree"] = ops.TreeRows(s["base"], s["rope"], s["mask"]) if tree else None
        s["out"] = torch.empty(n * per, nq * DIM, device=DEVICE, dtype=torch.bfloat16)
    return s


def _prepare_rotary(case, g):
    rows, far = case["rows"], case["far"]
    s = {"op": "rotary", "turned": case["turned"], "layout": case["layout"]}
    s["x"] = _vectors(g, rows, case["heads"], case["dim"]).to(TYPES[case["dtype"]])
    first = int(torch.randint(0, max(1, far - rows + 1), (1,), generator=g, device=DEVICE))
    s["positions"] = torch.arange(first, first + rows, device=DEVICE).int()
    if own:
        from georefine_b200 import ops

        s["rope"] = ops.Rope(case["turned"], 1e6, layout=case["layout"], scaling=SCALINGS[case["scaling"]] or None, device=DEVICE)
        s["out"] = torch.empty_like(s["x"])
    else:
        s["inv"], s["factor"] = _frequencies(case)
    return s


def _prepare_pages(case, g, pages):
    """A stack of layers with bytes of any kind in its pages: what is moved is not looked at."""
    s = {"op": case["op"], "format": case["format"], "k_exp": None, "v_exp": None}
    shape = (case["layers"], pages, case["kv_heads"])
    for w in ("k", "v"):
        if case["format"] == "q4":
            s[w] = _bytes(g, *shape, ENTRY, PAGE)
        elif case["format"] == "e4m3":
            s[w], s[w + "_exp"] = _bytes(g, *shape, PAGE, DIM).bitwise_and_(0xF7).view(torch.float8_e4m3fn), _bytes(g, *shape, PAGE).clamp_(max=134)
        else:
            s[w] = torch.randint(-16000, 16000, (*shape, PAGE, DIM), generator=g, device=DEVICE, dtype=torch.int16).view(torch.bfloat16)
    return s


def _prepare_fork(case, g):
    lengths, branches = _lengths(case), case["branches"]
    table, held = _page_table(g, lengths, empty=-1)
    forks = case["seqs"] * branches
    s = _prepare_pages(case, g, held + forks)
    s["lengths"] = _ints([n for n in lengths for _ in range(branches)])
    s["parents"] = torch.arange(case["seqs"], device=DEVICE).repeat_interleave(branches).int()
    s["children"] = torch.arange(forks, device=DEVICE).int() + case["seqs"]
    s["fresh"] = (held + torch.randperm(forks, generator=g, device=DEVICE)).int()
    s["page_table"] = torch.cat([table, torch.full((forks, table.shape[1]), -1, dtype=torch.int32, device=DEVICE)])
    s["refs"] = torch.zeros(held + forks, dtype=torch.int32, device=DEVICE)
    s["refs"][:held] = 1
    # the branches of the turn before, which a pass drops: half of them hold their fresh page
    s["page_table"][case["seqs"]::2, 0] = s["fresh"][::2]
    s["refs"][s["fresh"][::2].long()] = 1
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"], s["k_exp"], s["v_exp"])
    return s


def _prepare_compact(case, g):
    held = torch.tensor(_held_pages(case), device=DEVICE)
    s = _prepare_pages(case, g, case["pool"])
    order = held.nonzero()[:, 0]
    order = order[torch.randperm(order.shape[0], generator=g, device=DEVICE)].int()
    width = 8
    table = torch.full((-(-order.shape[0] // width) + 2, width), -1, dtype=torch.int32, device=DEVICE)      # (two slots are free)
    table.view(-1)[:order.shape[0]] = order
    table[-2, :2] = table[0, :2]                                                                             # (and one shares a prefix)
    s["table_before"], s["page_table"] = table, table.clone()
    s["refs_before"] = torch.zeros(case["pool"], dtype=torch.int32, device=DEVICE).scatter_add_(0, table.flatten().clamp(min=0).long(), (table >= 0).flatten().int())
    s["refs"] = s["refs_before"].clone()
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["where"], s["used"] = torch.empty(case["pool"], dtype=torch.int32, device=DEVICE), torch.empty(1, dtype=torch.int32, device=DEVICE)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------


def _buffers(s):
    return {w: s[w] for w in ("k", "v", "k_exp", "v_exp") if s.get(w) is not None}


def run(state):
    s, op = state, state["op"]
    if own:
        from georefine_b200 import ops
    if op == "write":
        if own:
            ops.kv_write(s["k_in"], s["v_in"], s["row_seq"], s["row_pos"], s["page_table"], s["pages"])
            ops.kv_read(s["row_seq"], s["row_pos"], s["page_table"], s["pages"], s["k_out"], s["v_out"])
            k, v = s["k_out"], s["v_out"]
        else:
            k, v = _write_plain(s)
        return {"k_read": k, "v_read": v, **_buffers(s)}
    if op in ("attend", "tree"):
        if own:
            s["attention"](s["qkv"], s["cos"], s["sin"], s["row_seq"], s["row_pos"], s["page_table"], s["pages"], s["out"], tree=s["tree"], longest_run=s["per_seq"])
            out = s["out"]
        else:
            out = _attention_plain(s)
        return {"out": out, **_buffers(s)}
    if op == "rotary":
        if own:
            ops.rotary(s["x"], s["positions"], s["rope"], out=s["out"])
            return {"out": s["out"]}
        return {"out": _rotary_plain(s)}
    if op == "fork":
        if own:
            ops.kv_free(s["children"], s["page_table"], s["refs"])
            ops.kv_fork(s["parents"], s["children"], s["lengths"], s["fresh"], s["page_table"], s["refs"], s["pages"])
        else:
            _fork_plain(s)
        return {"page_table": s["page_table"], "refs": s["refs"], **_buffers(s)}
    if own:
        s["page_table"].copy_(s["table_before"])
        s["refs"].copy_(s["refs_before"])
        ops.kv_compact(s["page_table"], s["refs"], s["pages"], s["where"], s["used"])
        where, used = s["where"], s["used"]
    else:
        where, used = _compact_plain(s)
    return {"page_table": s["page_table"], "refs": s["refs"], "where": where, "used": used, **_buffers(s)}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _nearest(x):
    """What a 4-bit entry holds of vectors x in 64 bits, by the definition, scale by scale."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -40.0)
    for power in range(-39, 23):                              # the largest power with 7 * 2^(power - 9) <= top
        e = torch.where(top >= 7.0 * 2.0 ** (power - 9), torch.full_like(e, power), e)
    unit = torch.exp2(e - 24)
    grid = torch.tensor([(16 + m) * 2.0 ** k for k in range(12) for m in range(16)], dtype=torch.float64, device=x.device)
    held = torch.empty_like(x)
    for g in range(4):
        y = x[..., 32 * g:32 * g + 32] / unit
        want = y.abs().amax(-1, keepdim=True) / 7
        at = torch.searchsorted(grid, want.contiguous()).clamp(max=191)
        above, below = grid[at], grid[(at - 1).clamp(min=0)]
        up = (above - want < want - below) | ((above - want == want - below) & (at % 2 == 0))
        scale = torch.where(up | (at == 0), above, below)
        whole = torch.floor(y / scale)
        part = y / scale - whole
        whole = torch.where((part > 0.5) | ((part == 0.5) & (whole % 2 != 0)), whole + 1, whole)
        held[..., 32 * g:32 * g + 32] = whole.clamp(-7, 7) * scale * unit
    return held


def _entries(pages, head, place):
    """Entries of one head at places (page, position) of 4-bit pages, in 64 bits: dimension by dimension."""
    page, at = place
    flat = pages[:, head].flatten(1)[page]
    codes = flat.gather(1, 64 * at[:, None] + torch.arange(64, device=at.device)).view(-1, 16, 4)
    scales = flat.gather(1, SCALES + 4 * at[:, None] + torch.arange(4, device=at.device)).double()
    scales = torch.where(scales < 16, scales / 8, (16 + scales % 16) * torch.exp2(torch.floor(scales / 16) - 4))
    unit = torch.exp2(flat.gather(1, EXPONENTS + at[:, None]).double().clamp(min=87) - 127 - 24)
    out = torch.empty(at.shape[0], 16, 8, dtype=torch.float64, device=at.device)
    for byte, (low, high) in enumerate(((0, 2), (4, 6), (1, 3), (5, 7))):
        out[..., low], out[..., high] = (codes[..., byte] % 16).double() - 8, (codes[..., byte] // 16).double() - 8
    return (out.view(-1, 4, 32) * scales[..., None]).flatten(1) * unit


def exact(case, seed):
    op = case["op"]
    if op in ("fork", "compact"):                              # whole numbers, and entries moved as they are
        return None
    s = prepare(case, seed)
    if op == "write":
        return {"k_read": _nearest(s["k_in"].double()), "v_read": _nearest(s["v_in"].double()), "k": None, "v": None}
    if op == "rotary":
        inv, factor = _frequencies(case)
        angle = s["positions"].double()[:, None] * inv
        turn = torch.polar(torch.full_like(angle, factor), angle)[:, None]
        x, n = s["x"].double(), case["turned"]
        out = x.clone()
        a, b = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
        turned = torch.complex(x[..., a], x[..., b]) * turn
        out[..., a], out[..., b] = turned.real, turned.imag
        return {"out": out}
    nq, nkv, n, per = s["heads"], s["kv_heads"], s["seqs"], s["per_seq"]
    half, out = DIM // 2, torch.empty(n * per, nq, DIM, dtype=torch.float64, device=DEVICE)
    pos, rope = s["row_pos"].long(), (s["row_pos"] if s["mask"] is None else s["rope"]).long()
    qkv = s["qkv"].double().view(n * per, -1, DIM)
    cos, sin = s["cos"].double()[rope][:, None], s["sin"].double()[rope][:, None]
    first, second = qkv[:, :nq + nkv, :half], qkv[:, :nq + nkv, half:]
    turned = torch.cat([first * cos[..., :half] - second * sin[..., :half], second * cos[..., half:] + first * sin[..., half:]], dim=-1)
    # (the sum is rounded to 32 bits before it is held: the definition's input is an FP32 vector)
    new = {"k": _nearest(turned[:, nq:].float().double()), "v": _nearest(qkv[:, nq + nkv:])}
    lengths, at = _lengths(case), 0
    for i in range(n):
        rows, total = slice(at, at + per), lengths[i] + per
        places = torch.arange(total, device=DEVICE)
        where = s["page_table"][i].long()[places // PAGE], places % PAGE
        if s["mask"] is None:
            seen = places <= pos[rows][:, None]
        else:
            masks = [m & ((1 << 64) - 1) for m in s["mask"][rows, 0].tolist()]
            bits = torch.tensor([[m >> j & 1 for j in range(per)] for m in masks], device=DEVICE).bool()
            seen = torch.cat([torch.ones(per, lengths[i], device=DEVICE, dtype=torch.bool), bits], dim=1)
        for h in range(nkv):
            held = {}
            for w in ("k", "v"):
                held[w] = _entries(s[w], h, where)
                held[w][pos[rows]] = new[w][rows, h]
            group = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            score = torch.matmul(turned[rows, group].transpose(0, 1), held["k"].T) / math.sqrt(DIM)
            out[rows, group] = torch.matmul(torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1), held["v"]).transpose(0, 1)
        at += per
    return {"out": out.view(n * per, nq * DIM), "k": None, "v": None}
