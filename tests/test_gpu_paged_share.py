"""The plan of shared prefixes: whole numbers, equal to the definition's."""
import random

import pytest
import torch

import shared_ref

pytestmark = pytest.mark.gpu

NAMES = ("members", "m_start", "m_pos", "token_group")


def run(sqa, dev, q_start, kv_len, group, shared_len, T, pos=True, **kw):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    before = [random.Random(T).randrange(10000) for _ in range(4 * T)] if pos else None
    p = i32(before) if pos else None
    members = torch.full((T,), 77, dtype=torch.int32, device=dev)
    got = sqa.paged_share(i32(q_start), i32(kv_len), i32(group), i32(shared_len), members, pos=p, **kw)
    assert isinstance(got, sqa.PagedShare) and got.members is members
    want = shared_ref.share(q_start, kv_len, group, shared_len, T, before)
    for name, x in zip(NAMES, got):
        assert x.tolist() == want[name], name
    if pos:
        assert p.tolist() == want["pos"]
    return got


def batch(r, B, G, most, pad, alone=0.15):
    n = [r.choice([0, 1, 1, 1, r.randint(0, most)]) for _ in range(B)]
    q_start = [0]
    for x in n:
        q_start.append(q_start[-1] + x)
    kv = [x + r.randint(0, 500) if r.random() < 0.9 else 0 for x in n]
    group = [r.randrange(G) if r.random() >= alone else r.choice([-1, G, -(1 << 31), 1 << 30]) for _ in range(B)]
    shared = [r.choice([0, -3, r.randint(1, 100000), r.randint(1, 100000)]) for _ in range(G)]
    return q_start, kv, group, shared, max(1, q_start[-1] + pad)


@pytest.mark.parametrize("B,G,most,pad", [(1, 1, 1, 0), (1, 1, 700, 0), (2, 1, 1, 3), (8, 3, 40, 0), (63, 5, 9, 1), (64, 64, 3, 0),
                                          (65, 2, 2, 0), (257, 40, 30, 100), (1000, 1000, 4, 0), (1024, 40, 60, 37), (4096, 300, 3, 5),
                                          (4096, 4096, 2, 0), (3, 2, 5000, 9000)])
def test_share(sqa, dev, B, G, most, pad):
    r = random.Random(B * 31 + G)
    for pos in (True, False):
        run(sqa, dev, *batch(r, B, G, most, pad), pos=pos)


def test_nobody_and_everybody(sqa, dev):
    run(sqa, dev, [0, 1, 2], [5, 6], [-1, -1], [100], 4)
    run(sqa, dev, [0, 1, 2], [5, 6], [0, 0], [0], 2)
    run(sqa, dev, [0, 0, 0], [5, 6], [0, 0], [10], 3)
    run(sqa, dev, [0, 700, 1400], [700, 9000], [0, 0], [60000], 1400)


def test_rows_before_the_requests_and_past_the_buffer(sqa, dev):
    run(sqa, dev, [5, 6, 9], [5, 6], [1, 0], [100, 200], 12)       # q_start[0] > 0
    run(sqa, dev, [0, 3, 9, 14], [5, 9, 9], [0, 0, 0], [100], 10)  # clipped at T
    run(sqa, dev, [-4, 3, 9], [7, 9], [0, 0], [100], 10)


def test_a_given_stream_a_graph_and_what_it_leaves(sqa, dev):
    r = random.Random(3)
    a = batch(r, 30, 4, 20, 6)
    run(sqa, dev, *a, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    ins = [i32(x) for x in a[:4]]
    T = a[4]
    share = sqa.PagedShare(*(torch.zeros(n, dtype=torch.int32, device=dev) for n in (T, 5, T, T)))
    pos = torch.zeros(4 * T, dtype=torch.int32, device=dev)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        sqa.paged_share(*ins, *share, pos=pos)
    for k in range(4):
        b = batch(r, 30, 4, 20, 0)
        if b[0][-1] > T:
            continue
        for t, x in zip(ins, b):
            t.copy_(i32(x))
        start = [r.randrange(1000) for _ in range(4 * T)]
        pos.copy_(i32(start))
        g.replay()
        torch.cuda.synchronize()
        want = shared_ref.share(*b[:4], T, start)
        assert [x.tolist() for x in share] + [pos.tolist()] == [want[n] for n in NAMES] + [want["pos"]]
        again = [x.clone() for x in (*share, pos)]
        sqa.paged_share(*ins, *share, pos=pos)  # the same call again changes nothing
        assert all(torch.equal(x, y) for x, y in zip(again, (*share, pos)))


def test_positions_stop_at_the_largest(sqa, dev):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    got = sqa.paged_share(i32([0, 2]), i32([(1 << 31) - 1]), i32([0]), i32([(1 << 31) - 1]), i32([0, 0, 0]))
    assert got.members.tolist() == [0, 1, -1] and all(p > 1 << 30 for p in got.m_pos.tolist()[:2])


def test_ranges_that_overlap_stay_inside(sqa, dev):
    """q_start that does not ascend gives unspecified numbers, all of them inside."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    T = 50
    got = sqa.paged_share(i32([0, 40, 3, 50, -9, 90]), i32([9] * 5), i32([0, 1, 0, 1, 0]), i32([7, 8]), torch.zeros(T, dtype=torch.int32, device=dev))
    assert all(-1 <= t < T for t in got.members.tolist()) and all(0 <= t <= T for t in got.m_start.tolist())
