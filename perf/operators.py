"""Operators of speculative serving over an 8-bit KV cache, as cases that can be timed: a cache that is quantised as it is
written and read back, attention of causal rows over it, attention of the nodes of draft trees over a cache, verification
of drafted tokens from given random numbers, and keeping an accepted path in the cache.

Ranges.  Heads: those of the benchmark's decoder and of its 2- and 4-way tensor-parallel shards, and of a 4096-wide model.
Cache rows: 1 to 2048 tokens of 1 to 16 sequences.  Attention: 1 to 128 sequences with 1 to 16384 positions, 1 to 8 causal rows
or 2 to 64 tree nodes each.  Verification: 1 to 128 sequences of 1 to 26 rows, vocabularies of 1001 to 152064 tokens,
BF16 and FP32 logits.  Kept paths: 1 to 128 sequences, 1 to 64 layers.  Pages are scattered and sequences are ragged everywhere.

An entry of an 8-bit cache is 128 values of one key or value head at one position: with a = max |x|, the exponent is
e = clamp(ceil(log2(a / 448)), -40, 7), a code is the e4m3 number nearest to x / 2^e (ties to even, at most 448), and it
stands for code * 2^e.  The exponent is kept as the byte e + 127.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
DIM, PAGE = 128, 256
VOCAB = 152064
SHAPES = ((40, 8), (20, 4), (10, 2), (32, 8))   # query and KV heads: the benchmark's decoder, its shards, a smaller model


def listed():
    return [
        # a prompt's last chunk stored in the 8-bit cache and read back: latency of the two calls
        {"name": "cache_384", "op": "cache", "seqs": 1, "tokens": 384, "kv_heads": 8},
        # sixteen sequences taken over from another cache
        {"name": "cache_16x2048", "op": "cache", "seqs": 16, "tokens": 2048, "kv_heads": 8},
        # one interactive sequence's decode step
        {"name": "step_1", "op": "attend", "seqs": 1, "rows": 1, "context": 2048, "heads": 40, "kv_heads": 8},
        # a full batch's decode step
        {"name": "step_128", "op": "attend", "seqs": 128, "rows": 1, "context": 2048, "heads": 40, "kv_heads": 8},
        # one sequence's draft tree after a BF16 prompt
        {"name": "tree_1x16", "op": "tree", "seqs": 1, "nodes": 16, "context": 1000, "heads": 40, "kv_heads": 8, "format": "bf16"},
        # wide trees of a batch over long 8-bit contexts: as much arithmetic as traffic
        {"name": "tree_16x64", "op": "tree", "seqs": 16, "nodes": 64, "context": 8192, "heads": 40, "kv_heads": 8, "format": "e4m3"},
        # the pending token and five drafts of one sequence, and of a full batch
        {"name": "verify_1x6", "op": "verify", "seqs": 1, "rows": 6, "tree": False, "probs": False, "vocab": VOCAB, "dtype": "bf16", "temperature": 0.7},
        {"name": "verify_128x6", "op": "verify", "seqs": 128, "rows": 6, "tree": False, "probs": False, "vocab": VOCAB, "dtype": "bf16", "temperature": 1.0},
        # a drafter that samples, with its probabilities
        {"name": "verify_16x5_probs", "op": "verify", "seqs": 16, "rows": 5, "tree": False, "probs": True, "vocab": VOCAB, "dtype": "fp32", "temperature": 1.0},
        # draft trees
        {"name": "verify_16x25_tree", "op": "verify", "seqs": 16, "rows": 25, "tree": True, "probs": False, "vocab": VOCAB, "dtype": "bf16", "temperature": 0.8},
        # what one sequence keeps of its tree, in a stack cut to 4 layers, and what a batch keeps in all 64
        {"name": "keep_1", "op": "keep", "seqs": 1, "nodes": 16, "layers": 4, "kv_heads": 8, "format": "bf16"},
        {"name": "keep_64", "op": "keep", "seqs": 64, "nodes": 25, "layers": 64, "kv_heads": 8, "format": "e4m3"},
    ]


def _spread(rng, lo, hi):
    """An integer in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("cache", "attend", "attend", "tree", "tree", "verify", "verify", "keep"))
    heads, kv_heads = rng.choice(SHAPES)
    kind = rng.choice(("bf16", "e4m3"))
    if op == "cache":
        return {"op": op, "seqs": _spread(rng, 1, 16), "tokens": _spread(rng, 1, 2048), "kv_heads": kv_heads}
    if op == "attend":
        context = _spread(rng, 1, 16384)
        return {"op": op, "seqs": _spread(rng, 1, min(128, 262144 // context)), "rows": rng.randint(1, 8), "context": context, "heads": heads, "kv_heads": kv_heads}
    if op == "tree":
        context = _spread(rng, 1, 8192)
        return {"op": op, "seqs": _spread(rng, 1, min(64, 131072 // context)), "nodes": _spread(rng, 2, 64), "context": context,
                "heads": heads, "kv_heads": kv_heads, "format": kind}
    if op == "verify":
        rows, tree = _spread(rng, 1, 26), rng.random() < 0.4
        return {"op": op, "seqs": _spread(rng, 1, min(128, 768 // rows)), "rows": rows, "tree": tree, "probs": not tree and rng.random() < 0.4,
                "vocab": _spread(rng, 1001, VOCAB) if rng.random() < 0.5 else VOCAB, "dtype": rng.choice(("bf16", "bf16", "fp32")),
                "temperature": round(rng.uniform(0.5, 1.2), 2)}
    return {"op": op, "seqs": _spread(rng, 1, 64), "nodes": _spread(rng, 2, 64), "layers": _spread(rng, 1, 64), "kv_heads": kv_heads, "format": kind}


def _share(i, most, least=0.5):
    """The i-th of a ragged series of lengths between least * most and most."""
    return max(1, int(most * (1 - (1 - least) * ((i * 0.6180339887) % 1.0))))


def _lengths(case):
    """Cached positions of every sequence before the call."""
    return [_share(i, case["context"]) for i in range(case["seqs"])]


def _row_counts(case):
    """Rows of every sequence of a verification, its pending token among them."""
    return [_share(i, case["rows"], 0.6) for i in range(case["seqs"])]


def _kept(case, i):
    """Nodes of sequence i's accepted path, the root among them."""
    return min(case["nodes"], 2 + (3 * i) % 5)


def _kind(case):
    return case.get("format", "e4m3")


def _entry_bytes(case):
    return DIM + 1 if _kind(case) == "e4m3" else 2 * DIM


def work(case):
    op = case["op"]
    if op == "cache":
        n = case["seqs"] * case["tokens"] * case["kv_heads"] * 2
        return {"bytes": n * 2 * (2 * DIM + DIM + 1), "flops": 0}
    if op in ("attend", "tree"):
        rows, heads, kv = case["rows"] if op == "attend" else case["nodes"], case["heads"], case["kv_heads"]
        entries = 2 * kv * sum(n + rows for n in _lengths(case))
        rows_all = rows * case["seqs"]
        return {"bytes": entries * _entry_bytes(case) + rows_all * 2 * DIM * (2 * heads + 2 * kv),
                "flops": 4 * DIM * heads * rows * sum(_lengths(case))}
    if op == "verify":
        rows, size = sum(_row_counts(case)), 2 if case["dtype"] == "bf16" else 4
        return {"bytes": rows * case["vocab"] * size + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0), "flops": 2 * rows * case["vocab"]}
    moved = sum(_kept(case, i) - 1 for i in range(case["seqs"]))
    return {"bytes": 2 * moved * case["layers"] * 2 * case["kv_heads"] * _entry_bytes(case), "flops": 0}


# ---- the plain forms ----------------------------------------------------------------------------------------------------


def _power(e):
    """2^e for whole e in [-126, 127], exactly."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x):
    """FP32 vectors [..., 128] -> e4m3 codes and exponent bytes."""
    m, k = torch.frexp(x.abs().amax(-1))                       # max |x| = m 2^k with m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, k - 8, k - 9).where(m > 0, torch.full_like(k, -40)).clamp(-40, 7)
    code = (x * _power(-e)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return code, (e + 127).to(torch.uint8)


def _values(code, exponent):
    return code.float() * _power(exponent.int() - 127)[..., None]


def _stored(state, which):
    """All sequences' keys or values as FP32 [seqs, positions, kv heads, 128], through the page table."""
    pages, table = state[which], state["page_table"].long()
    x = pages[table] if state[which + "_exp"] is None else _values(pages.view(torch.uint8)[table].view(torch.float8_e4m3fn), state[which + "_exp"][table])
    return x.float().transpose(2, 3).flatten(1, 2)


def _store(state, which, x):
    """Puts FP32 rows [rows, kv heads, 128] where the rows' sequences and positions say."""
    page = state["page_table"].long()[state["row_seq"].long(), state["row_pos"].long() // PAGE]
    at = state["row_pos"].long() % PAGE
    if state[which + "_exp"] is None:
        state[which][page, :, at] = x.to(torch.bfloat16)
    else:
        code, exponent = _quantise(x)
        state[which].view(torch.uint8)[page, :, at] = code.view(torch.uint8)
        state[which + "_exp"][page, :, at] = exponent


def _rotate(x, cos, sin):
    """Rotate-half: FP32 [rows, heads, 128] by tables [rows, 128]."""
    half = DIM // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], dim=-1)
    return x * cos[:, None].float() + turned * sin[:, None].float()


def _cache_plain(s):
    _store(s, "k", s["k_in"].float())
    _store(s, "v", s["v_in"].float())
    seq, pos = s["row_seq"].long(), s["row_pos"].long()
    page, at = s["page_table"].long()[seq, pos // PAGE], pos % PAGE
    read = lambda w: _values(s[w].view(torch.uint8)[page, :, at].view(torch.float8_e4m3fn), s[w + "_exp"][page, :, at]).to(torch.bfloat16)
    return read("k"), read("v")


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
    own_pos = s["row_pos"].long().view(n, per, 1)
    if s["mask"] is None:
        seen = position <= own_pos
    else:
        base = s["base"].long().view(n, per, 1)
        node = position - base
        bit = (s["mask"].view(n, per, 1) >> node.clamp(0, 63)) & 1
        seen = (node < 0) | ((node < 64) & (bit == 1))
    score = torch.einsum("nrgid,npgd->ngirp", q.view(n, per, nkv, nq // nkv, DIM), k) / math.sqrt(DIM)
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    weight = torch.exp(score - score.amax(-1, keepdim=True))
    out = torch.einsum("ngirp,npgd->nrgid", weight / weight.sum(-1, keepdim=True), v)
    return out.reshape(n * per, nq * DIM).to(torch.bfloat16)


def _verify_plain(s):
    """The walk over every sequence's drafts, all sequences and nodes at once; 64 bits, for draws next to a border."""
    index, here = s["index"], s["here"]                        # [seqs, rows]: a row's place among all rows; whether there is one
    seqs, width = index.shape
    lanes = torch.arange(width, device=index.device)
    token, keep = s["tokens"].long()[index], s["u_keep"].double()[index]
    logits = s["logits"].double() / s["temperature"]
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    # the parent of node i as a one-hot row (chains: the node before it)
    parent = (lanes - 1).expand(seqs, width) if s["parent"] is None else s["parent"].long()[index]
    child = here & (lanes > 0)
    up = ((parent[..., None] == lanes) & child[..., None]).double()
    of_token = p[index.gather(1, parent.clamp(min=0)), token]   # the parent's probability of the node's token
    earlier = (parent[..., None] == parent[:, None]) & child[..., None] & child[:, None] & (lanes[:, None] > lanes)   # [.., i, j]: j before i
    again = (earlier & (token[..., None] == token[:, None])).any(-1)
    fresh = torch.where(again | ~child, 0.0, of_token)
    struck = (earlier.double() * fresh[:, None]).sum(-1)
    if s["q"] is None:
        passes = child & (keep * (1 - struck) < fresh)
    else:
        passes = child & (keep * s["q"].double()[index, token] < of_token)
    chosen = passes & ~(earlier & passes[:, None]).any(-1)
    # a node is on the path when it and all its ancestors are chosen: ancestors by repeated squaring of "parent of"
    reach = (up + torch.eye(width, dtype=torch.double, device=up.device)).clamp(max=1)
    for _ in range(max(1, (width - 1).bit_length())):
        reach = (reach @ reach).clamp(max=1)
    refused = (~chosen & (lanes > 0)).double()
    on_path = here & ((reach * refused[:, None]).sum(-1) == 0)
    count = on_path.sum(-1)
    last = torch.where(on_path, lanes, -1).amax(-1)
    final = p[index.gather(1, last[:, None])[:, 0]]
    tried = child & (parent == last[:, None])
    if s["q"] is None:
        strike = torch.zeros_like(final).scatter_add_(1, token, tried.double()) > 0
        rest = final.masked_fill(strike, 0.0)
    else:
        after = (last + 1).clamp(max=width - 1)
        refusal = tried.any(-1)
        rest = torch.where(refusal[:, None], (final - s["q"].double()[index.gather(1, after[:, None])[:, 0]]).clamp(min=0), final)
    running = rest.cumsum(-1)
    drawn = (running <= s["u_draw"].double()[:, None] * running[:, -1:]).sum(-1)
    # nodes of the path in order, and the tokens they and the draw emit
    rank = torch.where(on_path, on_path.long().cumsum(-1) - 1, width)
    rows = torch.full((seqs, width + 1), -1, device=index.device).scatter_(1, rank, lanes.expand(seqs, width))[:, :width]
    rows = torch.where(lanes < count[:, None], rows, -1)
    following = token.gather(1, rows.roll(-1, 1).clamp(min=0))
    out = torch.where(lanes < count[:, None] - 1, following, torch.where(lanes == count[:, None] - 1, drawn[:, None], -1))
    return out.int(), rows.int(), count.int()


def _keep_plain(s):
    """Entries base + path[i] go to base + i for the path's nodes behind the root, in every layer."""
    path, count, base, table = s["path"].long(), s["count"].long(), s["base"].long(), s["page_table"].long()
    step = torch.arange(path.shape[1], device=path.device).expand_as(path)
    seq, node = ((step > 0) & (step < count[:, None])).nonzero(as_tuple=True)
    source, target = base[seq] + path[seq, node], base[seq] + step[seq, node]
    for x in (s["k"], s["v"], s["k_exp"], s["v_exp"]):
        if x is not None:
            x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            x[:, table[seq, target // PAGE], :, target % PAGE] = x[:, table[seq, source // PAGE], :, source % PAGE]
    return tuple(x for x in (s["k"], s["v"], s["k_exp"], s["v_exp"]) if x is not None)



# ---- inputs -------------------------------------------------------------------------------------------------------------


def _tables(positions):
    inv = 1e6 ** (-torch.arange(0, DIM, 2, dtype=torch.float64, device=DEVICE) / DIM)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
    angle = torch.cat([angle, angle], dim=1)
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _vectors(g, *shape):
    """Keys or values as a cache meets them: normal, some channels larger, positions of different size."""
    x = torch.randn(*shape, generator=g, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEVICE))
    return x * torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=g, device=DEVICE))


def _cache(g, state, pages, kv_heads, kind, layers=None, filled=True):
    """Keys and values of `pages` pages (of every layer), with what is in a cache or empty."""
    shape = (pages, kv_heads, PAGE, DIM)
    for w in ("k", "v"):
        parts, exps = [], []
        for _ in range(layers or 1):
            x = _vectors(g, *shape) if filled else torch.zeros(shape, device=DEVICE)
            code, exponent = _quantise(x) if kind == "e4m3" else (x.to(torch.bfloat16), None)
            parts.append(code.view(torch.uint8) if kind == "e4m3" else code)
            exps.append(exponent)
        x = torch.stack(parts) if layers else parts[0]
        state[w] = x.view(torch.float8_e4m3fn) if kind == "e4m3" else x
        state[w + "_exp"] = None if kind == "bf16" else torch.stack(exps) if layers else exps[0]


def _page_table(g, lengths):
    """Pages for the given lengths, scattered over the pool; the places behind a sequence's pages hold page 0."""
    need = [-(-n // PAGE) for n in lengths]
    order = torch.randperm(sum(need), generator=g, device=DEVICE)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].int()
        at += n
    return table, sum(need)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _parents(nodes, pick):
    """A draft tree: node 0 is the pending token; every other node hangs below an earlier one, the first few levels wide."""
    parents = [-1]
    for i in range(1, nodes):
        low = (i - 1) // 3
        parents.append(low + int(pick[i] * (i - low)))
    return parents


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(1000003 * int(seed) + 17)
    return {"cache": _prepare_cache, "attend": _prepare_attention, "tree": _prepare_attention, "verify": _prepare_verify, "keep": _prepare_keep}[case["op"]](case, g)


def _prepare_cache(case, g):
    n, nkv = case["tokens"], case["kv_heads"]
    s = {"op": "cache"}
    s["page_table"], pages = _page_table(g, [n] * case["seqs"])
    _cache(g, s, pages, nkv, "e4m3", filled=False)
    rows = case["seqs"] * n
    s["row_seq"] = torch.arange(case["seqs"], device=DEVICE).repeat_interleave(n).int()
    s["row_pos"] = torch.arange(n, device=DEVICE).repeat(case["seqs"]).int()
    s["k_in"], s["v_in"] = (_vectors(g, rows, nkv, DIM).to(torch.bfloat16) for _ in range(2))
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["k_out"], s["v_out"] = torch.empty_like(s["k_in"]), torch.empty_like(s["v_in"])
    return s


def _prepare_attention(case, g):
    nq, nkv, n = case["heads"], case["kv_heads"], case["seqs"]
    tree = case["op"] == "tree"
    per = case["nodes"] if tree else case["rows"]
    lengths = _lengths(case)
    s = {"op": case["op"], "heads": nq, "kv_heads": nkv, "seqs": n, "per_seq": per, "mask": None}
    s["page_table"], pages = _page_table(g, [length + per for length in lengths])
    _cache(g, s, pages, nkv, _kind(case))
    s["cos"], s["sin"] = _tables(max(lengths) + per)
    s["row_seq"] = torch.arange(n, device=DEVICE).repeat_interleave(per).int()
    s["row_pos"] = _ints([length + j for length in lengths for j in range(per)])
    s["qkv"] = torch.cat([1.5 * torch.randn(n * per, nq * DIM, generator=g, device=DEVICE), _vectors(g, n * per, 2 * nkv, DIM).flatten(1)], dim=1).to(torch.bfloat16)
    if tree:
        pick = torch.rand(n, per, generator=g, device=DEVICE).tolist()
        rope, mask = [], []
        for length, p in zip(lengths, pick):
            parents, depth, seen = _parents(per, p), [], []
            for i, up in enumerate(parents):
                depth.append(0 if up < 0 else depth[up] + 1)
                seen.append((1 << i) | (0 if up < 0 else seen[up]))
            rope += [length + d for d in depth]
            mask += [m - (1 << 64) if m >> 63 else m for m in seen]
        s["rope"], s["base"] = _ints(rope), _ints([length for length in lengths for _ in range(per)])
        s["mask"] = torch.tensor(mask, dtype=torch.int64, device=DEVICE)[:, None]
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"], s["k_exp"], s["v_exp"])
        s["attention"] = ops.TreeAttention(nq, nkv, n * per, s["page_table"].shape[1], DEVICE, kv_format=_kind(case))
        s["tree"] = ops.TreeRows(s["base"], s["rope"], s["mask"]) if tree else None
        s["out"] = torch.empty(n * per, nq * DIM, device=DEVICE, dtype=torch.bfloat16)
    return s


def _prepare_verify(case, g):
    counts, vocab, n = _row_counts(case), case["vocab"], case["seqs"]
    rows, width = sum(counts), max(counts)
    # a few tokens of each row stand out, as they do in a trained model's logits
    logits = 2.0 * torch.randn(rows, vocab, generator=g, device=DEVICE)
    likely = torch.randint(vocab, (rows, 8), generator=g, device=DEVICE)
    logits.scatter_add_(1, likely, 9.0 + 3.0 * torch.randn(rows, 8, generator=g, device=DEVICE))
    s = {"op": "verify", "temperature": case["temperature"], "logits": logits.to(torch.bfloat16) if case["dtype"] == "bf16" else logits, "q": None, "parent": None}
    starts = [sum(counts[:i]) for i in range(n + 1)]
    s["starts"] = _ints(starts)
    pick = torch.rand(n, width, generator=g, device=DEVICE).tolist()
    parents = [_parents(c, p) if case["tree"] else list(range(-1, c - 1)) for c, p in zip(counts, pick)]
    if case["tree"]:
        s["parent"] = _ints([p for ps in parents for p in ps])
    above = torch.tensor([starts[i] + max(p, 0) for i, ps in enumerate(parents) for p in ps], device=DEVICE)
    if case["probs"]:      # a drafter near the target, whose tokens are draws from its own distribution
        q = torch.softmax((logits[above] + 0.7 * torch.randn(rows, vocab, generator=g, device=DEVICE)) / case["temperature"], dim=-1)
        s["q"], tokens = q, torch.multinomial(q, 1, generator=g)[:, 0]
    else:                  # a drafter that names one of the likely tokens, mostly the best
        rank = (torch.rand(rows, generator=g, device=DEVICE) ** 3 * 4).long()
        tokens = logits[above].topk(4, dim=-1).indices.gather(1, rank[:, None])[:, 0]
    s["tokens"] = tokens.int()
    s["u_keep"], s["u_draw"] = torch.rand(rows, generator=g, device=DEVICE), torch.rand(n, generator=g, device=DEVICE)
    lanes = torch.arange(width, device=DEVICE)
    s["here"] = lanes < _ints(counts)[:, None]
    s["index"] = (s["starts"][:-1, None].long() + lanes).clamp(max=rows - 1)
    if own:
        from georefine_b200 import sampling

        s["verifier"] = sampling.DraftVerifier(rows, n, width, DEVICE)
    return s


def _prepare_keep(case, g):
    n, nodes = case["seqs"], case["nodes"]
    lengths = [_share(i, 700) for i in range(n)]
    s = {"op": "keep"}
    s["page_table"], pages = _page_table(g, [length + nodes for length in lengths])
    _cache(g, s, pages, case["kv_heads"], _kind(case), layers=case["layers"])
    s["base"] = _ints(lengths)
    s["count"] = _ints([_kept(case, i) for i in range(n)])
    order = torch.rand(n, nodes - 1, generator=g, device=DEVICE).argsort(dim=1).tolist()
    most = max(_kept(case, i) for i in range(n))
    path = [[0] + sorted(v + 1 for v in row[:_kept(case, i) - 1]) for i, row in enumerate(order)]
    s["path"] = _ints([p + [-1] * (most - len(p)) for p in path])
    s["seqs"] = torch.arange(n, device=DEVICE).int()
    if own:
        from georefine_b200 import ops

        s["pages"] = ops.KVPages(s["k"], s["v"], s["k_exp"], s["v_exp"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------


def _buffers(s):
    return {w: s[w] for w in ("k", "v", "k_exp", "v_exp") if s[w] is not None}


def run(state):
    s, op = state, state["op"]
    if op == "cache":
        if own:
            from georefine_b200 import ops

            ops.kv_write(s["k_in"], s["v_in"], s["row_seq"], s["row_pos"], s["page_table"], s["pages"])
            ops.kv_read(s["row_seq"], s["row_pos"], s["page_table"], s["pages"], s["k_out"], s["v_out"])
            k, v = s["k_out"], s["v_out"]
        else:
            k, v = _cache_plain(s)
        return {"k_read": k, "v_read": v, **_buffers(s)}
    if op in ("attend", "tree"):
        if own:
            s["attention"](s["qkv"], s["cos"], s["sin"], s["row_seq"], s["row_pos"], s["page_table"], s["pages"], s["out"], tree=s["tree"])
            out = s["out"]
        else:
            out = _attention_plain(s)
        return {"out": out, **_buffers(s)}
    if op == "verify":
        if own:
            out, rows, count = s["verifier"](s["logits"], s["tokens"], s["starts"], s["u_keep"], s["u_draw"], temperature=s["temperature"], parent=s["parent"],
                                             draft_probs=s["q"])
        else:
            out, rows, count = _verify_plain(s)
        return {"tokens": out, "rows": rows, "count": count}
    if own:
        from georefine_b200 import ops

        ops.kv_keep(s["seqs"], s["base"], s["path"], s["count"], s["page_table"], s["pages"])
        return _buffers(s)
    _keep_plain(s)
    return _buffers(s)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------


def _held(x):
    """What an 8-bit entry holds of vectors x in 64 bits, by the definition: (values, exponents)."""
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, -40.0)
    for power in range(-40, 8):                               # the smallest power that keeps the largest component below 448
        e = torch.where(a > 448.0 * 2.0 ** (power - 1), torch.full_like(e, power), e)
    powers = torch.tensor([2.0 ** p for p in range(-60, 10)], dtype=torch.float64, device=x.device)
    unit = powers[e.long() + 60]
    y = (x / unit).clamp(-448, 448)
    exponent = torch.frexp(y.abs().clamp(min=2.0 ** -6))[1] - 1      # of the leading bit; codes below 2^-6 share its step
    step = powers[exponent.long() - 3 + 60]
    return torch.round(y / step) * step * unit, e[..., 0]


def exact(case, seed):
    if case["op"] in ("verify", "keep"):                       # whole numbers, and entries moved as they are
        return None
    s = prepare(case, seed)
    if case["op"] == "cache":
        (k, ke), (v, ve) = _held(s["k_in"].double()), _held(s["v_in"].double())
        return {"k_read": k, "v_read": v, "k": None, "v": None, "k_exp": None, "v_exp": None}
    nq, nkv, n, per = s["heads"], s["kv_heads"], s["seqs"], s["per_seq"]
    half, out = DIM // 2, torch.empty(n * per, nq, DIM, dtype=torch.float64, device=DEVICE)
    pos, rope = s["row_pos"].long(), (s["row_pos"] if s["mask"] is None else s["rope"]).long()
    qkv = s["qkv"].double().view(n * per, -1, DIM)
    cos, sin = s["cos"].double()[rope][:, None], s["sin"].double()[rope][:, None]
    first, second = qkv[:, :nq + nkv, :half], qkv[:, :nq + nkv, half:]
    turned = torch.cat([first * cos[..., :half] - second * sin[..., :half], second * cos[..., half:] + first * sin[..., half:]], dim=-1)
    new = {"k": turned[:, nq:], "v": qkv[:, nq + nkv:]}
    if s["k_exp"] is not None:
        new = {w: _held(x)[0] for w, x in new.items()}
    else:
        new = {w: x.to(torch.bfloat16).double() for w, x in new.items()}
    lengths, at = _lengths(case), 0
    for i in range(n):
        rows, total = slice(at, at + per), lengths[i] + per
        places = torch.arange(total, device=DEVICE)
        page, place = s["page_table"][i].long()[places // PAGE], places % PAGE
        held = {}
        for w in ("k", "v"):
            code = s[w].view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn) if s[w + "_exp"] is not None else s[w][page, :, place]
            x = code.double()
            if s[w + "_exp"] is not None:
                x = x * torch.exp2(s[w + "_exp"][page, :, place].double()[..., None] - 127)
            x[pos[rows]] = new[w][rows]
            held[w] = x
        if s["mask"] is None:
            seen = places <= pos[rows][:, None]
        else:
            masks = [m & ((1 << 64) - 1) for m in s["mask"][rows, 0].tolist()]
            bits = torch.tensor([[m >> j & 1 for j in range(per)] for m in masks], device=DEVICE).bool()
            seen = torch.cat([torch.ones(per, lengths[i], device=DEVICE, dtype=torch.bool), bits], dim=1)
        for h in range(nkv):
            group = slice(h * (nq // nkv), (h + 1) * (nq // nkv))
            score = torch.matmul(turned[rows, group].transpose(0, 1), held["k"][:, h].T) / math.sqrt(DIM)
            out[rows, group] = torch.matmul(torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1), held["v"][:, h]).transpose(0, 1)
        at += per
    return {"out": out.view(n * per, nq * DIM), "k": None, "v": None, "k_exp": None, "v_exp": None}
