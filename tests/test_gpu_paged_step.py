"""The operators of a batch together, as a server runs them: plan, producer and
value writes into the pages, attention, projection, adapters - eagerly against
KvCache's contiguous path per request, and captured once and replayed."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, HKV, EPS, N = 256, 16, 2, 1e-6, 256


def weights(sqa, dev, gen):
    w = torch.randint(0, 256, (N, H * D // 256, 144), generator=gen, device=dev, dtype=torch.uint8)
    dm = torch.rand((N, H * D // 256, 2), generator=gen, device=dev) * 4e-4 + 1e-4
    w[:, :, :4] = dm.half().view(torch.uint8).reshape(N, -1, 4)
    return {"w": w.reshape(N, -1), "kw": 1 + 0.1 * torch.randn(D, generator=gen, device=dev),
            "a": (torch.randn((3, 16, H * D), generator=gen, device=dev) / 64).half(),
            "b": torch.randn((3, N, 16), generator=gen, device=dev).half(),
            "rope": sqa.rope_params(64, (11, 11, 10, 0), 1e7)}


def layer(sqa, kv, step, max_q, s, wt):
    """One full-attention layer of a step over static buffers s."""
    sqa.rope_norm_set_rows_q4_0(kv.rows(0, "k"), s["k"], wt["kw"], EPS, step.pos, wt["rope"], step.slots)
    sqa.set_rows_q4_0(kv.rows(0, "v"), s["v"], step.slots)
    sqa.rope_norm_f32(s["q2"], s["q"], wt["kw"], EPS, step.pos, wt["rope"])
    kv.attend(0, s["q2"], step, max_q, gate=s["gate"], out=s["att"], workspace=s["ws"])
    T = s["att"].shape[0]
    sqa.out_proj(wt["w"], s["att"].view(T, -1), out=s["y"], workspace=s["ws2"])
    sqa.lora_add(s["y"], s["att"].view(T, -1), wt["a"], wt["b"], s["ids"], out=s["z"])


def buffers(sqa, dev, kv, T, max_q, wt):
    z = lambda *n: torch.zeros(n, device=dev)  # noqa: E731
    s = {"k": z(T, HKV, D), "v": z(T, HKV * D), "q": z(T, H, D), "q2": z(T, H, D), "gate": z(T, H, D), "att": z(T, H, D),
         "y": z(T, N), "z": z(T, N), "ids": torch.zeros(T, dtype=torch.int32, device=dev)}
    s["ws"] = torch.empty(max(16, kv.workspace_size(s["q"], max_q)), dtype=torch.uint8, device=dev)
    s["ws2"] = torch.empty(max(16, sqa.out_proj_workspace_size(wt["w"], s["att"].view(T, -1))), dtype=torch.uint8, device=dev)
    return s


def fill(s, gen):
    for k in ("k", "v", "q", "gate"):
        s[k].copy_(torch.randn(s[k].shape, generator=gen, device=s[k].device))
    s["ids"].copy_(torch.randint(-1, 3, s["ids"].shape, generator=gen, device=s["ids"].device))


def test_batch_equals_single_sequences(sqa, dev):
    gen = torch.Generator(device=dev).manual_seed(1)
    wt, B, T = weights(sqa, dev, gen), 4, 160
    kv = sqa.PagedKvCache(1, D, HKV, 64, 16, B, 16, device=dev)
    solo = [sqa.KvCache(1, D, HKV, 256, device=dev) for _ in range(B)]
    for c in solo:
        c.zero_caches()
    step, s = kv.new_step(T), buffers(sqa, dev, kv, T, 90, wt)
    for new in ([40, 1, 0, 70], [1, 1, 90, 1], [2, 30, 1, 1], [1, 1, 1, 1]):
        fill(s, gen)
        s["att"].fill_(0)
        kv.plan(torch.tensor(new, dtype=torch.int32, device=dev), step)
        layer(sqa, kv, step, max(new), s, wt)
        t0 = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            at, c = slice(t0, t0 + n), solo[b]
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
            t0 += n
        x = s["att"].view(T, -1)
        delta = torch.zeros_like(s["y"], dtype=torch.float64)
        for i in range(3):
            m = s["ids"] == i
            delta[m] = (x[m].double() @ wt["a"][i].double().t()) @ wt["b"][i].double().t()
        assert float((s["z"].double() - s["y"].double() - delta).norm() / delta.norm()) <= 1e-5


def test_step_in_a_graph(sqa, dev):
    """One capture serves decode steps of any lengths; every replay equals the eager step bit for bit."""
    gen = torch.Generator(device=dev).manual_seed(2)
    wt, B, T, max_q = weights(sqa, dev, gen), 5, 64, 40
    kv = sqa.PagedKvCache(1, D, HKV, 200, 16, B, 30, device=dev)
    step, s = kv.new_step(T), buffers(sqa, dev, kv, T, max_q, wt)
    n_new = torch.zeros(B, dtype=torch.int32, device=dev)
    keep = (kv._now, kv.table, kv.ring, kv.k[0], kv.v[0], s["att"])

    def run():
        kv.plan(n_new, step)
        layer(sqa, kv, step, max_q, s, wt)

    for t in kv.k + kv.v:
        t.zero_()
    run()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        run()
    torch.cuda.synchronize()
    for new in ([20, 0, 7, 1, 30], [1, 1, 1, 1, 1], [40, 1, -1, 3, 1], [1, 2, 9, 1, -1], [1, 1, 1, 1, 1]):
        fill(s, gen)
        n_new.copy_(torch.tensor(new, dtype=torch.int32))
        before = [t.clone() for t in keep]
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*keep, s["z"], step.slots)]
        for t, x in zip(keep, before):
            t.copy_(x)
        run()
        torch.cuda.synchronize()
        for x, y in zip(got, (*keep, s["z"], step.slots)):
            assert torch.equal(x, y), new
        assert torch.isfinite(s["z"]).all()


def test_two_graphs_share_a_workspace(sqa, dev):
    gen = torch.Generator(device=dev).manual_seed(3)
    kv = sqa.PagedKvCache(1, D, HKV, 80, 16, 3, 20, device=dev)
    for t in kv.k + kv.v:
        t.copy_(torch.randint(0, 60, t.shape, generator=gen, device=dev, dtype=torch.uint8))
    step = kv.new_step(400)
    kv.plan(torch.tensor([100, 250, 31], dtype=torch.int32, device=dev), step)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    calls = []
    for starts, max_q in (([0, 1, 2, 3], 1), ([0, 60, 61, 92], 60)):
        q = torch.randn((starts[-1], H, D), generator=gen, device=dev)
        calls.append((q, kv.k[0], kv.v[0], kv.table, i32(starts), step.kv_len, max_q))
    ws = torch.empty(max(sqa.paged_attn_workspace_size(c[0], c[1], c[3], c[6]) for c in calls) + 16, dtype=torch.uint8, device=dev)
    outs = [torch.zeros_like(c[0]) for c in calls]
    want = [sqa.paged_attn(*c, out=o, workspace=ws).clone() for c, o in zip(calls, outs)]
    graphs = []
    for c, o in zip(calls, outs):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            sqa.paged_attn(*c, out=o, workspace=ws)
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
