"""Token sampling for the decode engine: temperature, nucleus (top-p) filtering, and speculative sampling against a
drafter that proposes one definite token per position.

Host-side torch arithmetic over the logits a step leaves on the device - plumbing beside the path, as in the reference's
session (``glc_serve/fastserve.py:308-395``: ``_probs``, ``_sample`` and the sampling branch of ``_spec_cycle``).  Every
function works on any device and takes the ``torch.Generator`` the caller seeded, so a run is reproducible and the ranks
of a tensor-parallel decoder, seeded alike and holding the same logits, draw the same tokens.
"""
from __future__ import annotations


def _check(temperature: float, top_p: float) -> None:
    if not temperature > 0:
        raise ValueError("temperature must be positive; temperature 0 is the arg-max path")
    if not 0 < top_p <= 1:
        raise ValueError("top_p must be in (0, 1]")


def probabilities(logits, temperature: float, top_p: float = 1.0):
    """Rows of logits -> rows of FP32 probabilities at ``temperature`` > 0, restricted to the nucleus when ``top_p`` < 1:
    the tokens in descending order of probability up to and including the one that brings the running mass to ``top_p``
    (a token is dropped when the mass of the tokens ranked above it already exceeds ``top_p``; the first is always kept),
    renormalised.  Equal probabilities rank by token id, lowest first, which is also how the arg-max kernel breaks ties."""
    import torch

    _check(temperature, top_p)
    p = torch.softmax(logits.float() / float(temperature), dim=-1)
    if top_p < 1.0:
        ranked, order = torch.sort(p, dim=-1, descending=True, stable=True)
        above = torch.cumsum(ranked, dim=-1) - ranked            # mass of the tokens ranked before this one
        ranked = torch.where(above > top_p, torch.zeros_like(ranked), ranked)
        p = torch.zeros_like(p).scatter_(-1, order, ranked)
        p = p / p.sum(dim=-1, keepdim=True)
    return p


def draw(p, generator=None):
    """One token id per row of probabilities (int64 tensor on p's device)."""
    import torch

    return torch.multinomial(p, 1, generator=generator).reshape(-1)


def accept_drafts(p, drafts, generator=None):
    """Speculative sampling for one sequence.  ``p``: k + 1 rows of target probabilities - row i is the distribution of
    the token after the first i drafts; ``drafts``: the k tokens a deterministic drafter proposed.  Draft i is kept with
    probability p[i, draft]; the first one refused is replaced by a draw from p[i] with that token struck out, and
    nothing behind it is used; if all k are kept, one more token is drawn from row k.  Each emitted token is then
    distributed exactly as if it had been drawn from the target alone: P(t) = p[d]*[t = d] + (1 - p[d]) * p[t] / (1 - p[d])
    for t != d.  Returns the emitted tokens (1 to k + 1 of them)."""
    import torch

    k = len(drafts)
    if p.shape[0] != k + 1:
        raise ValueError("one row of probabilities per draft, and one more")
    u = torch.rand(k + 1, generator=generator, device=p.device).tolist()
    kept = p[torch.arange(k, device=p.device), torch.as_tensor(list(drafts), device=p.device, dtype=torch.long)].tolist() if k else []
    out = []
    for i, d in enumerate(drafts):
        if u[i] < kept[i]:
            out.append(int(d))
            continue
        rest = p[i].clone()
        rest[int(d)] = 0
        mass = float(rest.sum())
        out.append(int(draw((rest / mass)[None], generator)[0]) if mass > 0 else int(d))
        return out
    out.append(int(draw(p[k][None], generator)[0]))
    return out


class Sampler:
    """Temperature, nucleus and generator of one generation call, as the engine passes them around."""

    def __init__(self, temperature: float, top_p: float = 1.0, *, device="cpu", seed=None):
        self.temperature, self.top_p = float(temperature), float(top_p)
        _check(self.temperature, self.top_p)
        self.generator = make_generator(device, seed)
        self._verifier = None

    def probabilities(self, logits):
        return probabilities(logits, self.temperature, self.top_p)

    def draw(self, logits):
        """One token per row of logits."""
        return draw(self.probabilities(logits), self.generator)

    def accept(self, logits, drafts):
        """``logits``: len(drafts) + 1 rows of one sequence's verify pass."""
        return accept_drafts(self.probabilities(logits), drafts, self.generator)

    def verify(self, logits, tokens, parents, starts):
        """Draft trees of several sequences on the GPU: ``logits`` [rows, vocabulary] of all their nodes, sequence s's from row
        ``starts[s]`` on (lists of Python integers, ``starts`` one longer than there are sequences), the pending token first;
        ``parents`` within the sequence.  Returns ``DraftVerifier``'s (tokens, rows, count); the random numbers are the generator's."""
        import torch

        rows, seqs = logits.shape[0], len(starts) - 1
        width = max(hi - lo for lo, hi in zip(starts, starts[1:]))
        if width > 256:
            raise ValueError(f"a draft tree of {width} nodes: at most 256 are looked at")
        if self._verifier is None or rows > self._verifier.max_rows or seqs > self._verifier.max_seqs or width > self._verifier.width:
            self._verifier = DraftVerifier(max(rows, 128), max(seqs, 128), max(width, 16), logits.device)
        if self.top_p < 1:          # the nucleus renormalised is the soft-max over its tokens alone
            logits = logits.float().masked_fill(self.probabilities(logits) == 0, float("-inf"))
        i32 = lambda v: torch.tensor(list(v), dtype=torch.int32).to(logits.device)
        u = torch.rand(rows + seqs, generator=self.generator, device=logits.device)
        return self._verifier(logits, i32(tokens), i32(starts), u[:rows], u[rows:], temperature=self.temperature, parent=i32(parents))


class DraftVerifier:
    """Verification of drafted tokens on the GPU (``csrc/verify_ops.cuh``), for up to ``max_rows`` rows of ``max_seqs`` sequences a
    call: chains and trees, random numbers given by the caller, nothing brought to the host.  ``width``: columns of the outputs,
    the longest walk (a walk stops after ``width`` - 1 kept drafts).  A call's outputs are the object's own and hold until its next
    call; calls that may run at the same time need an object each."""

    def __init__(self, max_rows: int, max_seqs: int, width: int, device):
        import torch

        if max_rows < 1 or max_seqs < 1 or not 1 <= width <= 256:
            raise ValueError("at least one row and sequence, and a width of 1 to 256")
        self.max_rows, self.max_seqs, self.width = int(max_rows), int(max_seqs), int(width)
        self.stats = torch.empty(self.max_rows, 16, device=device, dtype=torch.float64)
        self.tokens, self.rows = (torch.empty(self.max_seqs, self.width, device=device, dtype=torch.int32) for _ in range(2))
        self.count = torch.empty(self.max_seqs, device=device, dtype=torch.int32)
        self.device = self.stats.device
        self._places = tuple(t.data_ptr() for t in (self.stats, self.tokens, self.rows, self.count))

    def __call__(self, logits, tokens, starts, u_keep, u_draw, *, temperature=1.0, parent=None, draft_probs=None):
        """``logits`` (BF16 or FP32 [rows, vocabulary]): the target's, row i those behind node i.  Rows ``starts[s]`` ..
        ``starts[s + 1] - 1`` are sequence s's draft tree: its pending token, then the drafts, parents before children;
        ``tokens`` are the nodes' tokens, ``parent`` their parents' numbers within the sequence (None: chains).  With p =
        softmax(logits / temperature) at a node, its child c is kept when u_keep[c] (1 - S) < p[t_c], S being the mass of the children's
        tokens tried before; where none is kept, the last token is drawn from p without the tried ones: the lowest whose
        cumulative mass exceeds u_draw[s] times what is left.  ``draft_probs`` (FP32 [rows, vocabulary], chains): row i is the
        distribution that token i was drawn from; it is kept when u q[t] < p[t], else the draw is from max(p - q, 0).  Both leave
        the tokens distributed as draws from the target.  A sequence has at most 256 rows: those behind them are not looked at.

        Returns int32 (tokens [seqs, width]: the kept drafts, then the drawn token; rows [seqs, width]: the walk's nodes, the
        root first; count [seqs]: how many of each), padded with -1."""
        import torch

        from . import _native
        from .ops import _launch, _ld, _on, _vector

        device, n = self.device, starts.shape[0] - 1
        kind = 0 if logits.dtype is torch.bfloat16 else 1 if logits.dtype is torch.float32 else None
        if logits.dim() != 2 or kind is None or logits.device != device or (logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ValueError("logits are BF16 or FP32 [rows, vocabulary] on the verifier's device, their rows contiguous")
        rows, vocab = logits.shape
        if not 0 <= n <= self.max_seqs or rows > self.max_rows:
            raise ValueError("more rows or sequences than the verifier was made for")
        if not 1e-30 <= temperature <= 1e20:
            raise ValueError("temperature must be from 1e-30 to 1e20; temperature 0 is the arg-max path")
        for t, size, what in ((u_keep, rows, "u_keep"), (u_draw, n, "u_draw")):
            _on(t, device, torch.float32, what, (size,))
            if not t.is_contiguous():
                raise ValueError(f"{what} has to be contiguous")
        q = ldq = 0
        if draft_probs is not None:
            if parent is not None:
                raise ValueError("the drafter's probabilities go with chains")
            _on(draft_probs, device, torch.float32, "draft_probs", (rows, vocab))
            if vocab > 1 and draft_probs.stride(1) != 1:
                raise ValueError("rows of draft_probs have to be contiguous")
            q, ldq = draft_probs.data_ptr(), _ld(draft_probs, vocab, "draft_probs")
        above = 0 if parent is None else _vector(parent, device, "parent", rows)
        tokens_at, starts_at = _vector(tokens, device, "tokens", rows), _vector(starts, device, "starts")
        out = (self.tokens, self.rows, self.count) if n == self.max_seqs else (self.tokens[:n], self.rows[:n], self.count[:n])
        if n:
            step = _native.VERIFY_STEP.pack(logits.data_ptr(), _ld(logits, vocab, "logits"), tokens_at, above, starts_at, u_keep.data_ptr(), u_draw.data_ptr(), q, ldq,
                                            *self._places, rows, n, vocab, self.width, kind, float(temperature))
            _launch(device, "grb_verify_drafts", step)
        return out


def make_generator(device, seed=None):
    """A generator on ``device``; seeded when a seed is given, else from the system's entropy."""
    import torch

    g = torch.Generator(device=device)
    if seed is None:
        g.seed()
    else:
        g.manual_seed(int(seed))
    return g
