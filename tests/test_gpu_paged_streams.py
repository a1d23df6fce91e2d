"""Calls on a stream other than the current one: what a call makes for itself belongs to its stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, HKV, ROW = 256, 16, 2, 144


def busy(stream):
    with torch.cuda.stream(stream):
        torch.cuda._sleep(24_000_000)  # cycles: 10 ms and more


def batch(sqa, dev, lens, new):
    gen = torch.Generator(device=dev).manual_seed(4)
    pages = [-(-n // 64) for n in lens]
    pools = [torch.empty((sum(pages), 64, HKV, ROW), dtype=torch.uint8, device=dev) for _ in range(2)]
    for p in pools:
        sqa.set_rows_q4_0(p.view(-1, HKV, ROW), torch.randn((p.shape[0] * 64, HKV * D), generator=gen, device=dev),
                          torch.arange(p.shape[0] * 64, device=dev))
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device=dev)
    at, starts = 0, [0]
    for b, n in enumerate(pages):
        table[b, :n] = torch.arange(at, at + n, device=dev)
        at += n
        starts.append(starts[-1] + new[b])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    q = torch.randn((starts[-1] + 3, H, D), generator=gen, device=dev)
    return q, *pools, table, i32(starts), i32(lens), max(new)


def handles(s):
    return [s, s.cuda_stream]


@pytest.mark.parametrize("new", [[1, 2, 1], [1, 90, 30]])
def test_result_made_by_the_call(sqa, dev, new):
    """The zeros of out come before the kernels, however late the current stream is."""
    args = batch(sqa, dev, [3000, 700, 90], new)
    want = sqa.paged_attn(*args)
    s = torch.cuda.Stream()
    for handle in handles(s):
        torch.cuda.synchronize()
        busy(torch.cuda.current_stream())
        got = sqa.paged_attn(*args, stream=handle)
        s.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert torch.equal(sqa.paged_attn(*args, stream=torch.cuda.default_stream().cuda_stream), want)


@pytest.mark.parametrize("new", [[1, 2, 1], [1, 90, 30]])
def test_workspace_made_by_the_call(sqa, dev, new):
    """Freed at the call's return, it is no memory of the current stream's next tensors while the kernels wait."""
    args = batch(sqa, dev, [3000, 700, 90], new)
    want = sqa.paged_attn(*args)
    size = sqa.paged_attn_workspace_size(args[0], args[1], args[3], args[6])
    out = torch.zeros_like(want)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    busy(s)
    sqa.paged_attn(*args, out=out, stream=s)
    others = [torch.full((size,), 0xFF, dtype=torch.uint8, device=dev) for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert all((o == 0xFF).all() for o in others)


def test_a_result_outlives_its_stream_for_the_current_one(sqa, dev):
    """A result of another stream, freed while the current stream has yet to read it, is not written over."""
    args = batch(sqa, dev, [300, 70, 90], [1, 1, 1])
    want = sqa.paged_attn(*args)
    s, cur = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    got = sqa.paged_attn(*args, stream=s)
    cur.wait_stream(s)
    busy(cur)
    copy = got.clone()
    del got
    with torch.cuda.stream(s):
        others = [torch.full_like(want, 9.0) for _ in range(3)]
    torch.cuda.synchronize()
    assert torch.equal(copy, want) and len(others) == 3


def test_plan_and_adapters(sqa, dev):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    def plan(**kw):
        return sqa.paged_plan(i32([0, 9, 0, 0]), i32(list(range(9))), torch.full((3, 4), -1, dtype=torch.int32, device=dev),
                              i32([0, 5, 0]), i32([20, 1, 7]), 16, torch.zeros(32, dtype=torch.int64, device=dev), **kw)

    gen = torch.Generator(device=dev).manual_seed(5)
    x, base = torch.randn((40, 512), generator=gen, device=dev), torch.randn((40, 64), generator=gen, device=dev)
    a, b = (torch.randn(n, generator=gen, device=dev).half() for n in ((2, 8, 512), (2, 64, 8)))
    ids = i32([m % 3 - 1 for m in range(40)])
    want, added = plan(), sqa.lora_add(base, x, a, b, ids)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for handle in handles(s):
        got = plan(stream=handle)
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        got = sqa.lora_add(base, x, a, b, ids, stream=handle)
        torch.cuda.synchronize()
        assert torch.equal(got, added)


def test_a_step_on_another_stream(sqa, dev):
    """plan, append and attend of PagedKvCache all take the stream: in order with each other, whatever
    the current stream does."""
    gen = torch.Generator(device=dev).manual_seed(8)
    kv, vv = torch.randn((2, 40, HKV * D), generator=gen, device=dev)
    q = torch.randn((40, H, D), generator=gen, device=dev)
    n_new = torch.tensor([30, 1, 0, 9], dtype=torch.int32, device=dev)
    s = torch.cuda.Stream()
    got = []
    for handle in (None, *handles(s)):
        cache = sqa.PagedKvCache(1, D, HKV, 12, 16, 4, 4, device=dev)
        for t in cache.k + cache.v:
            t.zero_()
        step = cache.new_step(40)
        torch.cuda.synchronize()
        if handle is not None:
            busy(torch.cuda.current_stream())
        for _ in range(2):
            cache.plan(n_new, step, stream=handle)
            cache.append(0, kv, vv, step, stream=handle)
            out = cache.attend(0, q, step, 30, stream=handle)
        (torch.cuda.current_stream() if handle is None else s).synchronize()
        torch.cuda.synchronize()
        got.append([out, cache.n_past.clone(), cache.state.clone(), cache.table, cache.ring, step.slots, *cache.k, *cache.v])
    for other in got[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got[0], other))
    assert got[0][1].tolist() == [60, 2, 0, 18]
