"""The plan of a step against a one-page-at-a-time reference: every array equal."""
import random

import numpy as np
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu


def run(sqa, dev, state, ring, table, n_past, n_new, page, T, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    tab, rg = i32(table), i32(ring)
    step = sqa.paged_plan(i32(state), rg, tab, i32(n_past), i32(n_new), page,
                          torch.full((T,), 99, dtype=torch.int64, device=dev), **kw)
    torch.cuda.synchronize()
    got = {"state": step.state, "ring": rg, "table": tab, "n_past": step.n_past, "q_start": step.q_start,
           "kv_len": step.kv_len, "slots": step.slots, "pos": step.pos}
    return {k: v.tolist() for k, v in got.items()}


def make(r, B, W, page, free, n_new=None):
    """A consistent state: requests of random lengths, their pages and `free` more in a random order."""
    past = [r.choice([0, 1, page - 1, page, page + 1, r.randint(0, W * page)]) for _ in range(B)]
    past = [min(p, W * page) for p in past]
    held = sum(-(-p // page) for p in past)
    ids = list(range(held + free))
    r.shuffle(ids)
    table, at = [[-1] * W for _ in range(B)], 0
    for b, p in enumerate(past):
        k = -(-p // page)
        table[b][:k] = ids[at:at + k]
        at += k
    n = max(1, held + free)
    head, ring = r.randrange(n), [-1] * n
    for i, x in enumerate(ids[at:]):
        ring[(head + i) % n] = x
    new = n_new or [r.choice([1, 1, 1, 0, -1, r.randint(2, 3 * page), r.randint(1, W * page)]) for _ in range(B)]
    return [head, free, 0, 0], ring, table, past, new


@pytest.mark.parametrize("B,W,page,free", [(1, 1, 16, 1), (1, 4, 16, 0), (3, 5, 32, 4), (7, 9, 16, 40), (64, 8, 16, 300),
                                           (65, 3, 256, 17), (256, 4, 64, 90), (257, 6, 16, 1000), (1000, 5, 16, 700),
                                           (4096, 2, 16, 1500)])
@pytest.mark.parametrize("seed", [0, 1])
def test_plan_equals_reference(sqa, dev, B, W, page, free, seed):
    r = random.Random(1000 * B + seed)
    args = make(r, B, W, page, free)
    total = sum(max(0, n) for n in args[4])
    for T in {max(1, total), total + 37, max(1, total // 2)}:
        want = paged_ref.plan(*args, page, T)
        got = run(sqa, dev, *args, page, T)
        for k in want:
            assert got[k] == want[k], (k, T)


def test_plan_edges(sqa, dev):
    # nothing new; nothing at all fits; one token row; a request that fills its table exactly and one that passes it
    for past, new, free, T in [([5, 0], [0, 0], 2, 4), ([0, 0], [40, 1], 0, 64), ([15], [1], 0, 1), ([15], [2], 1, 2),
                               ([63], [1], 3, 8), ([64], [1], 3, 8), ([0], [64], 4, 64), ([0], [65], 9, 80),
                               ([48, 0], [-1, 64], 1, 64), ([10, 10], [-1, -5], 0, 3), ([0, 3, 0], [16, 30, 1], 1, 64)]:
        page, W = 16, 4
        held = [min(-(-p // page), W) for p in past]
        ids = list(range(sum(held) + free))
        table, at = [[-1] * W for _ in past], 0
        for b, k in enumerate(held):
            table[b][:k] = ids[at:at + k]
            at += k
        n = max(1, len(ids))
        ring = (ids[at:] + [-1] * n)[:n]
        args = ([0, free, 0, 0], ring, table, past, new)
        want, got = paged_ref.plan(*args, page, T), run(sqa, dev, *args, page, T)
        assert got == want, (past, new, free, T)


def test_plan_extreme_lengths_are_refused_whole(sqa, dev):
    big = 2 ** 31 - 1
    args = ([0, 2, 0, 0], [0, 1], [[-1] * 2 for _ in range(4)], [0, big, 0, 7], [big, 1, 5, -big - 1])
    # the first asks for more rows than there are, so nobody behind it has rows left
    got = run(sqa, dev, *args, 16, 32)
    assert got["slots"] == [-1] * 32 and got["kv_len"] == [0] * 4 and got["n_past"] == [0, big, 0, 0]
    assert got["state"][2] == 3 and got["q_start"] == [0, 32, 32, 32, 32]


def test_plan_paths_agree_and_stream(sqa, dev):
    r = random.Random(3)
    args = make(r, 20, 6, 32, 50)
    T = sum(max(0, n) for n in args[4]) + 3
    want = run(sqa, dev, *args, 32, T)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert run(sqa, dev, *args, 32, T, stream=s) == want
    with torch.cuda.stream(s):
        assert run(sqa, dev, *args, 32, T) == want


def test_plan_many_steps_keep_every_page(sqa, dev):
    """A server's life: every page is always in the ring or in one table row, lengths follow."""
    r, page, B = random.Random(11), 16, 12
    kv = sqa.PagedKvCache(1, 256, 2, 60, page, B, 9, device=dev)
    step = kv.new_step(200)
    past = [0] * B
    for _ in range(60):
        new = [-1 if p and r.random() < 0.15 else r.choice([0, 1, 1, r.randint(2, 50)]) for p in past]
        table0, state0, ring0 = kv.table.tolist(), kv.state.tolist(), kv.ring.tolist()
        want = paged_ref.plan(state0, ring0, table0, past, new, page, 200)
        kv.plan(torch.tensor(new, dtype=torch.int32, device=dev), step)
        assert kv.n_past.tolist() == want["n_past"] and step.slots.tolist() == want["slots"]
        past = kv.n_past.tolist()
        head, count = kv.state.tolist()[:2]
        ring, table = kv.ring.tolist(), kv.table.tolist()
        ids = [ring[(head + i) % 60] for i in range(count)]
        ids += [x for b in range(B) for x in table[b][:-(-past[b] // page)]]
        assert sorted(ids) == list(range(60))
        slots = [x for x in step.slots.tolist() if x >= 0]
        assert len(set(slots)) == len(slots)


def test_plan_in_a_graph(sqa, dev):
    r, page, B, T = random.Random(5), 16, 9, 64
    kv = sqa.PagedKvCache(1, 256, 1, 80, page, B, 12, device=dev)
    step = kv.new_step(T)
    n_new = torch.zeros(B, dtype=torch.int32, device=dev)
    kv.plan(n_new, step)  # eager first call
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        kv.plan(n_new, step)
    torch.cuda.synchronize()
    past = [0] * B
    for _ in range(6):
        new = [-1 if p and r.random() < 0.2 else r.randint(0, 6) for p in past]
        want = paged_ref.plan(kv.state.tolist(), kv.ring.tolist(), kv.table.tolist(), past, new, page, T)
        n_new.copy_(torch.tensor(new, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        assert kv.state.tolist() == want["state"] and kv.ring.tolist() == want["ring"]
        assert kv.table.tolist() == want["table"] and step.slots.tolist() == want["slots"]
        past = kv.n_past.tolist()
        assert past == want["n_past"]
        (torch.ones(1000, device=dev) * 2).sum().item()  # the program's own work between replays
