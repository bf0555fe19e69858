"""The operators of speculative serving by their definitions, in 64 bits and one row at a time, for the tests beside this file."""
import math

import torch

DIM, PAGE = 128, 256


def entry(x):
    """What an 8-bit entry holds of vectors x [..., 128] (any float type): (codes as FP64, exponent bytes, values)."""
    x = x.double()
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    a = x.abs().amax(-1)
    e = torch.full_like(a, -40.0)
    for power in range(-40, 8):                    # the smallest power under which the largest component is at most 448
        e = torch.where(a > 448.0 * 2.0 ** (power - 1), torch.full_like(e, power), e)
    y = (x * torch.exp2(-e)[..., None]).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    code = torch.round(y / step) * step            # (ties to even)
    byte = torch.where(fine, e + 127, torch.full_like(e, 255.0)).to(torch.uint8)
    return torch.where(fine[..., None], code, 0.0), byte, torch.where(fine[..., None], code * torch.exp2(e)[..., None], torch.nan)


def rotate(x, cos, sin):
    """Rotate-half in 64 bits; x [heads, 128], tables' rows [128]."""
    x, h = x.double(), DIM // 2
    return torch.cat([x[:, :h] * cos[:h].double() - x[:, h:] * sin[:h].double(), x[:, h:] * cos[h:].double() + x[:, :h] * sin[h:].double()], dim=1)


def attend(q, k, v, seen, q_half_step, w_half_step):
    """One row: q [nq, 128] rotated, k and v [positions, nkv, 128], seen [positions] bool.  Returns the output [nq, 128] and a
    bound on what the kernel may be off: its query is rounded by q_half_step (relative), each weight by w_half_step, sums and exponentials
    run in 32 bits (2^-14 covers 2^13 positions of 2^-24 each, scores up to 2^8 and the exponential's 2^-22), the result is rounded to BF16."""
    nq, nkv = q.shape[0], k.shape[1]
    if not bool(seen.any()):
        return torch.zeros_like(q), torch.zeros_like(q)
    kk, vv = (t[seen].repeat_interleave(nq // nkv, dim=1) for t in (k, v))
    score = torch.einsum("hd,phd->hp", q, kk) / math.sqrt(DIM)
    off = q_half_step * torch.einsum("hd,phd->hp", q.abs(), kk.abs()).amax(1) / math.sqrt(DIM)      # of any score
    w = torch.softmax(score, dim=1)
    out, size = torch.einsum("hp,phd->hd", w, vv), torch.einsum("hp,phd->hd", w, vv.abs())
    inner = (torch.expm1(2 * off)[:, None] + 2 * w_half_step + 2.0 ** -14) * size
    return out, inner + 2.0 ** -8 * (out.abs() + inner) + 1e-30


def walk(logits, tokens, parents, u_keep, u_draw, temperature, q=None):
    """One sequence: (emitted tokens, walked nodes, how near the nearest decision was to going the other way)."""
    p = torch.softmax(logits.double() / temperature, dim=1).tolist()
    qs = None if q is None else q.double().tolist()
    node, out, path, near = 0, [], [0], 1.0
    while True:
        children = [c for c in range(1, len(tokens)) if parents[c] == node]
        struck, kept = set(), None
        for c in children:
            t = tokens[c]
            mass = p[node][t] if t not in struck else 0.0
            if qs is not None:
                left, right = u_keep[c] * qs[c][t], mass
            else:
                left, right = u_keep[c] * (1 - sum(p[node][s] for s in struck)), mass
            if t not in struck:
                near = min(near, abs(left - right))
            if left < right:
                kept = c
                break
            struck.add(t)
        if kept is None:
            break
        node = kept
        out.append(tokens[node])
        path.append(node)
    if qs is not None and children:
        rest = [max(a - b, 0.0) for a, b in zip(p[node], qs[children[0]])]
    else:
        rest = [0.0 if t in struck else a for t, a in enumerate(p[node])]
    total, run = math.fsum(rest), 0.0
    if total <= 0:
        return out + [tokens[children[-1]] if children else 0], path, near
    drawn = None
    for t, a in enumerate(rest):
        if a <= 0:
            continue
        if drawn is not None and run > u_draw * total:
            break
        run += a
        drawn = t
        if run > u_draw * total:
            break
    return out + [drawn], path, near
