"""The engine's books of its pages, on the host: whatever slots do - grow, fork, write to what they share, go back, end - the pool, which has
as many pages as all slots can name, has one for them.  No GPU: the copies are left out, and the table is the host's."""
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from georefine_b200 import ops, serve  # noqa: E402


def _decoder(monkeypatch, slots, pages):
    d = serve.BatchDecoder.__new__(serve.BatchDecoder)
    d.dev, d.max_slots, d.pages_per_seq, d.max_context, d.scratch_page = torch.device("cpu"), slots, pages, pages * serve.PAGE, slots * pages
    d._table_host = np.full((slots + 1, pages), -1, dtype=np.int64)
    d._free_pages, d._free_slots = list(range(slots * pages - 1, -1, -1)), list(range(slots - 1, -1, -1))
    d._refs, d.page_sets = np.zeros(slots * pages + 1, dtype=np.int32), set()
    d.page_table = torch.full((slots + 1, pages), d.scratch_page, dtype=torch.int32)
    d._pool = lambda: (None, None)

    def kv_fork(parents, children, lengths, fresh, table, refs, pages, *, empty):
        for p, c, n, f in zip(*(x.tolist() for x in (parents, children, lengths, fresh))):
            table[c] = empty
            table[c, :n // 256] = table[p, :n // 256]
            if n % 256:
                table[c, n // 256] = f

    def kv_copy(src, dst, pages, *, positions=None):
        assert not set(dst.tolist()) & {int(p) for p in d._table_host.flatten()} and len(set(dst.tolist())) == len(dst)

    monkeypatch.setattr(ops, "kv_fork", kv_fork)
    monkeypatch.setattr(ops, "kv_copy", kv_copy)
    return d


def _consistent(d):
    named = [int(p) for p in d._table_host.flatten() if p >= 0]
    for p in range(d.scratch_page):
        assert d._refs[p] == named.count(p) and (p in d._free_pages) == (d._refs[p] == 0)
    assert len(set(d._free_pages)) == len(d._free_pages)
    table = d.page_table.numpy()
    assert ((table == d._table_host) | ((d._table_host < 0) & (table == d.scratch_page))).all()


@pytest.mark.parametrize("seed", range(12))
def test_the_pool_has_a_page_for_whatever_slots_do(monkeypatch, seed):
    rng = random.Random(seed)
    slots, pages = rng.choice([(2, 1), (3, 2), (4, 3), (6, 2), (5, 4)])
    d = _decoder(monkeypatch, slots, pages)
    length = {}                                   # of each open slot: positions written
    least = d.scratch_page
    for _ in range(300):
        act = rng.choice(["open", "grow", "grow", "fill", "fork", "fork", "back", "close"])
        if act == "open" and d._free_slots:
            length[d.open_slot()] = 0
        elif act == "close" and length and rng.random() < 0.5:
            slot = rng.choice(list(length))
            d.close_slot(slot)
            del length[slot]
        elif length:
            slot = rng.choice(list(length))
            n = length[slot]
            if act in ("grow", "fill") and n < d.max_context:
                upto = d.max_context - 1 if act == "fill" else min(n + rng.choice([0, 1, 40, 255, 300]), d.max_context - 1)
                d.own_pages(slot, n, upto)
                d.ensure_pages(slot, upto)
                for p in range(n // 256, upto // 256 + 1):
                    assert d._refs[d._table_host[slot, p]] == 1           # what is written to is the slot's own
                length[slot] = upto + 1
            elif act == "fork" and n and d._free_slots:
                for c in d.fork_slot(slot, n, rng.randint(1, len(d._free_slots))):
                    length[c] = n
            elif act == "back" and n > 1:
                length[slot] = rng.randint(1, n)
        least = min(least, len(d._free_pages))
        _consistent(d)
    for slot in list(length):
        d.close_slot(slot)
    _consistent(d)
    assert len(d._free_pages) == d.scratch_page and len(d._free_slots) == slots and least < d.scratch_page
