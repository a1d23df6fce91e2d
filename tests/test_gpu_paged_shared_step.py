"""A step of requests that continue prompts cached once: plan, share, producer and value writes, attention of both
parts - against a contiguous cache per request that holds the prompt itself, and captured once and replayed."""
import pytest
import torch

from test_gpu_paged_step import D, EPS, H, HKV, fill, weights

pytestmark = pytest.mark.gpu


def layer(sqa, kv, step, share, max_q, s, wt):
    sqa.rope_norm_set_rows_q4_0(kv.rows(0, "k"), s["k"], wt["kw"], EPS, step.pos, wt["rope"], step.slots)
    sqa.set_rows_q4_0(kv.rows(0, "v"), s["v"], step.slots)
    sqa.rope_norm_f32(s["q2"], s["q"], wt["kw"], EPS, step.pos, wt["rope"])
    kv.attend(0, s["q2"], step, max_q, share=share, gate=s["gate"], out=s["att"], workspace=s["ws"])


def buffers(dev, kv, T, max_q, share):
    z = lambda *n: torch.zeros(n, device=dev)  # noqa: E731
    s = {"k": z(T, HKV, D), "v": z(T, HKV * D), "q": z(T, H, D), "q2": z(T, H, D), "gate": z(T, H, D), "att": z(T, H, D),
         "ids": torch.zeros(T, dtype=torch.int32, device=dev)}
    s["ws"] = torch.empty(kv.workspace_size(s["q"], max_q, share=share), dtype=torch.uint8, device=dev)
    return s


def test_children_equal_sequences_that_hold_the_prompt(sqa, dev):
    """Rounding is the same on both sides but for the order of sums: 2e-5 as for a batch without shared prompts."""
    gen = torch.Generator(device=dev).manual_seed(5)
    wt, B, T = weights(sqa, dev, gen), 8, 330
    parent = [-1, -1, 0, 0, 1, 0, -1, 1]
    kv = sqa.PagedKvCache(1, D, HKV, 80, 16, B, 20, device=dev)
    solo = [sqa.KvCache(1, D, HKV, 512, device=dev) for _ in range(B)]
    for c in solo:
        c.zero_caches()
    step, share = kv.new_step(T), kv.new_share(T)
    s, par = buffers(dev, kv, T, 200, share), torch.tensor(parent, dtype=torch.int32, device=dev)
    before = 0
    for new in ([163, 64, 0, 0, 0, 0, 0, 0], [0, 0, 1, 5, 70, 1, 40, 0], [0, 0, 1, 1, 1, 1, 1, 1], [0, 0, 1, 4, 1, 0, 1, 33]):
        fill(s, gen)
        s["att"].fill_(0)
        kv.plan(torch.tensor(new, dtype=torch.int32, device=dev), step)
        kv.share(par, step, share)
        layer(sqa, kv, step, share, max(new), s, wt)
        t0 = 0
        for b, n in enumerate(new):
            at, t0 = slice(t0, t0 + n), t0 + n
            if n == 0:
                continue
            holders = [b] + [c for c in range(B) if before == 0 and parent[c] == b]  # the prompt goes into its children's too
            for c in (solo[h] for h in holders):
                past = c.n_used
                c.begin_step(n)
                pos = torch.arange(past, past + n, dtype=torch.int32, device=dev).repeat(4)
                idx = torch.arange(past, past + n, device=dev)
                sqa.rope_norm_set_rows_q4_0(c.k[0], s["k"][at], wt["kw"], EPS, pos, wt["rope"], idx)
                sqa.set_rows_q4_0(c.v[0], s["v"][at], idx)
                q = torch.empty((n, H, D), device=dev)
                sqa.rope_norm_f32(q, s["q"][at], wt["kw"], EPS, pos, wt["rope"])
                assert torch.equal(q, s["q2"][at])
                want = sqa.flash_attn_ext_causal(q, c.k[0], c.v[0], past + n, past, gate=s["gate"][at])
                err = float((s["att"][at] - want).norm() / want.norm())
                assert err <= 2e-5, (new, b, err)
        assert not s["att"][t0:].any()
        before += 1


def test_step_in_a_graph(sqa, dev):
    """One capture serves steps whose requests change parents and lengths; replays equal eager steps bit for bit."""
    gen = torch.Generator(device=dev).manual_seed(6)
    wt, B, T, max_q = weights(sqa, dev, gen), 6, 150, 60
    kv = sqa.PagedKvCache(1, D, HKV, 200, 16, B, 30, device=dev)
    step, share = kv.new_step(T), kv.new_share(T)
    s = buffers(dev, kv, T, max_q, share)
    n_new, par = (torch.zeros(B, dtype=torch.int32, device=dev) for _ in range(2))
    keep = (kv._now, kv.table, kv.ring, kv.k[0], kv.v[0], s["att"])

    def run():
        kv.plan(n_new, step)
        kv.share(par, step, share)
        layer(sqa, kv, step, share, max_q, s, wt)

    for t in kv.k + kv.v:
        t.zero_()
    par.fill_(-1)
    run()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        run()
    torch.cuda.synchronize()
    for new, parents in (([60, 50, 0, 0, 0, 0], [-1] * 6), ([0, 0, 1, 1, 30, 1], [-1, -1, 0, 1, 0, -1]), ([0, 0, 1, 1, 1, 1], [-1, -1, 0, 1, 0, 0]),
                         ([0, 0, -1, 60, 2, 1], [-1, -1, 0, 1, 1, 0]), ([0, 0, 8, 1, 1, 1], [-1, -1, 1, 1, 1, 1]), ([1, 1, 1, 1, 1, 1], [-1] * 6)):
        fill(s, gen)
        n_new.copy_(torch.tensor(new, dtype=torch.int32))
        par.copy_(torch.tensor(parents, dtype=torch.int32))
        before = [t.clone() for t in keep]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*keep, *share, step.pos, step.slots)]
        for t, x in zip(keep, before):
            t.copy_(x)
        s["ws"].fill_(0xFF)
        run()
        torch.cuda.synchronize()
        for x, y in zip(got, (*keep, *share, step.pos, step.slots)):
            assert torch.equal(x, y), new
        assert torch.isfinite(s["att"]).all()


def test_two_graphs_share_a_workspace(sqa, dev):
    gen = torch.Generator(device=dev).manual_seed(7)
    kv = sqa.PagedKvCache(1, D, HKV, 80, 16, 4, 30, device=dev)
    for t in kv.k + kv.v:
        t.copy_(torch.randint(0, 60, t.shape, generator=gen, device=dev, dtype=torch.uint8))
    step = kv.new_step(700)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    kv.plan(i32([400, 100, 70, 31]), step)
    lens, calls = kv.n_past.clone(), []
    for starts, max_q in (([0, 0, 1, 2, 3], 1), ([0, 0, 60, 61, 92], 60)):
        share, q = kv.new_share(starts[-1]), torch.randn((starts[-1], H, D), generator=gen, device=dev)
        sqa.paged_share(i32(starts), step.kv_len, i32([-1, 0, 0, -1]), lens, *share)
        calls.append((q, kv.k[0], kv.v[0], kv.table, i32(starts), lens, kv.table, lens, share, max_q))
    size = max(sqa.paged_attn_shared_workspace_size(c[0], c[1], c[3], c[6], c[9]) for c in calls)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    outs = [torch.zeros_like(c[0]) for c in calls]
    want = [sqa.paged_attn_shared(*c, out=o, workspace=ws).clone() for c, o in zip(calls, outs)]
    graphs = []
    for c, o in zip(calls, outs):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sqa.paged_attn_shared(*c, out=o, workspace=ws)
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        sqa.paged_attn_shared(*calls[0], out=torch.zeros_like(outs[0]), workspace=ws)


def test_a_conversation_drops_its_oldest_part(sqa, dev):
    """KvCache.move and read, PagedKvCache.move and read: the kept rows go to the front of each cache, whose contents agree."""
    gen = torch.Generator(device=dev).manual_seed(8)
    n, drop, page = 200, 70, 16
    rope = sqa.rope_params(64, (11, 11, 10, 0), 1e7)
    c, kv = sqa.KvCache(1, D, HKV, 256, device=dev), sqa.PagedKvCache(1, D, HKV, 20, page, 1, 16, device=dev)
    c.zero_caches()
    c.begin_step(n)
    k, v = (torch.randn((n, HKV * D), generator=gen, device=dev) for _ in range(2))
    c.append(0, k, v, torch.arange(n, device=dev))
    step = kv.new_step(n)
    kv.plan(torch.tensor([n], dtype=torch.int32, device=dev), step)
    kv.append(0, k, v, step)
    before = c.read(0, torch.arange(n, device=dev))
    assert torch.equal(before, kv.read(0, step.slots))
    # 130 rows forward by 70: in two runs, since a row that is read must not be written by the same call
    delta = torch.full((4 * drop,), -drop, dtype=torch.int32, device=dev)
    for first in (drop, 2 * drop):
        rows = torch.arange(first, min(n, first + drop), device=dev)
        d = delta.view(4, -1)[:, :len(rows)].reshape(-1)
        c.move(0, rows - drop, rows, d, rope)
        kv.move(0, step.slots[rows - drop], step.slots[rows], d, rope)
    c.rewind_to(n - drop)
    left = torch.arange(n - drop, device=dev)
    for which in ("k", "v"):
        got = c.read(0, left, which)
        assert torch.equal(got, kv.read(0, step.slots[left], which))
        half = c.read(0, left, which, dtype=torch.float16)
        assert half.dtype == torch.float16 and torch.equal(half, got.half())
    # V as it was; K's dims that are not rotated too, the others turned (and rounded to a code: half a step of amax / 8)
    assert torch.equal(c.read(0, left, "v"), kv.read(0, step.slots[left], "v"))
    got, was = (x.view(-1, HKV, D) for x in (c.read(0, left), before[drop:]))
    assert torch.equal(got[..., 64:], was[..., 64:]) and not torch.equal(got[..., :64], was[..., :64])
    norm = lambda x: x[..., :64].norm(dim=-1)  # noqa: E731
    # a block of 32: steps of amax / 8 at most, errors within half of one but for the clipped end (a whole one)
    assert ((norm(got) - norm(was)).abs() <= 8 * was[..., :64].abs().amax(-1) * 2 ** 0.5 / 8).all()
