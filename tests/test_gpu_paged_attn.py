"""Attention over a paged pool against the float64 definition.

Tolerances: a logit is a sum of 8 block terms rounded at 2^-24 each, below 2^5 in
base-2 units here, so it is off by at most 8 * 32 * 2^-24 = 1.5e-5 and a weight by
ln 2 of that, 1.1e-5, relatively; P and P d_v travel with 22 bits (2.4e-7). The
errors of the keys' weights are independent, so the output is off by that share of
itself in the 2-norm (REL, with the cap's tanh within 2^-21 of the logit), and a
single value by some ten times its share of the RMS at most (MAX). With distance
biases the logits that count are those near the row's position."""
import numpy as np
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

D, ROW = 256, 144
REL, MAX = 2e-5, 2e-4


class Batch:
    """Inputs of a call: lengths are per request, pages are dealt out of a pool with spare and garbage pages."""

    def __init__(self, orc, seed, new, past, H=16, Hkv=2, page=16, prefix=None, pad=0, spare=3, gate=False, scale_v=1.0,
                 scale_q=1.0):
        r = self.r = np.random.default_rng(seed)
        self.H, self.Hkv, self.page = H, Hkv, page
        self.kv_len = [n + p for n, p in zip(new, past)]
        used = [max(0, -(-k // page)) for k in self.kv_len]
        n_pages, W = sum(used) + spare, max(1, max(used)) + 1
        order = r.permutation(n_pages)
        self.k, self.v = (np.full((n_pages, page, Hkv, ROW), 0xFF, dtype=np.uint8) for _ in range(2))  # NaN scales
        self.table, at = np.full((len(new), W), -1, dtype=np.int32), 0
        for b, u in enumerate(used):
            ids = self.table[b, :u] = order[at:at + u]
            at += u
            for j in range(0, max(0, self.kv_len[b]), page):
                n = min(page, self.kv_len[b] - j)  # rows behind the request's last token stay garbage
                self.k[ids[j // page], :n] = paged_ref.quantize(orc, r.standard_normal((n, Hkv, D), dtype=np.float32))
                self.v[ids[j // page], :n] = paged_ref.quantize(
                    orc, np.float32(scale_v) * r.standard_normal((n, Hkv, D), dtype=np.float32))
        self.q_start = [0]
        for n in new:
            self.q_start.append(self.q_start[-1] + n)
        T = max(1, self.q_start[-1] + pad)
        self.q = np.float32(scale_q) * r.standard_normal((T, H, D), dtype=np.float32)
        self.gate = r.standard_normal((T, H, D), dtype=np.float32) if gate else None
        self.prefix, self.max_q = prefix, max(1, max(new))

    def ref(self, orc, fill=0.0, **kw):
        return paged_ref.attention(orc, self.q, self.k, self.v, self.table, self.q_start, self.kv_len, self.prefix,
                                   gate=self.gate, fill=fill, **kw)

    def args(self, dev):
        t = lambda x, d=torch.int32: torch.tensor(np.asarray(x), dtype=d, device=dev)  # noqa: E731
        a = [t(self.q, torch.float32), t(self.k, torch.uint8), t(self.v, torch.uint8), t(self.table), t(self.q_start),
             t(self.kv_len), self.max_q]
        kw = {"prefix": None if self.prefix is None else t(self.prefix),
              "gate": None if self.gate is None else t(self.gate, torch.float32)}
        return a, kw


def call(sqa, dev, batch, fill=None, ws=None, **kw):
    a, opt = batch.args(dev)
    out = torch.full(batch.q.shape, 0.0 if fill is None else fill, device=dev)
    if ws is None:
        ws = max(16, sqa.paged_attn_workspace_size(a[0], a[1], a[3], a[6]))
    work = torch.full((ws,), 0xFF, dtype=torch.uint8, device=dev)  # NaN wherever the workspace is not written
    got = sqa.paged_attn(*a, **opt, out=out, workspace=work, **kw)
    assert got is out
    return out.cpu().numpy().astype(np.float64)


def close(got, want, rows=None):
    assert np.isfinite(got).all()
    d = got - want
    norm = np.linalg.norm(want)
    if norm == 0:
        assert not d.any()
        return
    rel = np.linalg.norm(d) / norm
    top = np.abs(d).max() / np.sqrt(np.mean(want ** 2))
    print(f"rel {rel:.2e} max {top:.2e}")
    assert rel <= REL and top <= MAX, (rel, top)


SHAPES = [(16, 2), (16, 1), (8, 1), (4, 4), (6, 2), (28, 4), (5, 1), (1, 1), (24, 2)]


@pytest.mark.parametrize("H,Hkv", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 512])
def test_decode(sqa, orc, dev, H, Hkv, page):
    past = [0, 1, 14, 15, 16, 30, 31, 62, 63, 64, 65, 127, 128, 300, 777]
    b = Batch(orc, H * 100 + page, [1] * len(past), past, H, Hkv, page)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("n", [2, 3, 4])
@pytest.mark.parametrize("H,Hkv", [(16, 2), (4, 4), (6, 2), (16, 4)])
def test_verify(sqa, orc, dev, n, H, Hkv):
    past = [0, 1, 13, 61, 62, 63, 64, 190, 555]
    new = [1 + (i + n) % n for i in range(len(past))]
    new[3] = n
    b = Batch(orc, 7 * n + H, new, past, H, Hkv, 32, pad=5)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("n,past", [(3, 0), (5, 70), (17, 0), (31, 33), (64, 0), (65, 1), (100, 29), (129, 640), (300, 0), (257, 500)])
@pytest.mark.parametrize("H,Hkv,page", [(16, 2, 16), (16, 4, 64), (4, 4, 32)])
def test_chunk(sqa, orc, dev, n, past, H, Hkv, page):
    b = Batch(orc, n + past, [n], [past], H, Hkv, page)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("H,Hkv", SHAPES)
def test_ragged_chunks(sqa, orc, dev, H, Hkv):
    new, past = [1, 40, 0, 7, 150, 2, 33, 1], [90, 0, 50, 300, 17, 0, 31, 0]
    b = Batch(orc, 31 + H, new, past, H, Hkv, 16, pad=11, gate=True)
    close(call(sqa, dev, b, fill=7.0), b.ref(orc, fill=7.0))


@pytest.mark.parametrize("cap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("bias", [0.0, 8.0])
@pytest.mark.parametrize("form", ["decode", "verify", "chunk", "mixed"])
def test_scores(sqa, orc, dev, cap, bias, form):
    new, past = {"decode": ([1] * 4, [0, 40, 129, 900]), "verify": ([2, 1, 2], [3, 200, 800]),
                 "chunk": ([45, 130], [0, 333]), "mixed": ([1, 70, 1, 3, 1], [500, 64, 0, 100, 63])}[form]
    for H, Hkv in [(16, 2), (12, 2)]:
        b = Batch(orc, 5, new, past, H, Hkv, 32, scale_q=3.0)
        close(call(sqa, dev, b, softcap=cap, max_bias=bias), b.ref(orc, cap=cap, bias=bias))


@pytest.mark.parametrize("cap,bias", [(0.0, 0.0), (20.0, 4.0)])
@pytest.mark.parametrize("form", ["decode", "chunk"])
def test_prefix(sqa, orc, dev, cap, bias, form):
    new, past = ([1, 2, 1, 2], [100, 0, 63, 5]) if form == "decode" else ([80, 50, 130, 20, 33], [0, 100, 0, 3, 64])
    prefix = [500, 1, 0, 6] if form == "decode" else [40, 120, 1000, 0, -3]
    b = Batch(orc, 8, new, past, prefix=prefix, gate=True)
    close(call(sqa, dev, b, softcap=cap, max_bias=bias), b.ref(orc, cap=cap, bias=bias))


@pytest.mark.parametrize("new", [[1, 1, 2, 1], [20, 40, 9, 1]])
def test_rows_that_see_nothing(sqa, orc, dev, new):
    """Lengths of zero, more tokens than keys, negative lengths, tables of holes: zeros."""
    b = Batch(orc, 3, new, [50] * 4, spare=2)
    b.kv_len[0] = 0
    b.kv_len[2] = max(1, new[2] // 2)  # the first tokens sit before the first key
    b.table[3, :] = np.resize([-1, b.k.shape[0], 2 ** 31 - 1, -2 ** 31, -7], b.table.shape[1])
    want = b.ref(orc)
    assert not want[0].any() and not want[-1].any()
    close(call(sqa, dev, b), want)
    b.kv_len[1] = -5
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1], [40, 70]])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_holes_in_the_table(sqa, orc, dev, new, page):
    b = Batch(orc, page, new, [400, 300], page=page)
    b.table[0, 0], b.table[0, 2], b.table[1, 1] = -1, b.k.shape[0] + 5, 2 ** 30
    close(call(sqa, dev, b), b.ref(orc))


def test_requests_share_pages(sqa, orc, dev):
    for new in ([1, 1, 1], [30, 1, 60]):
        b = Batch(orc, 12, new, [200, 200, 200], page=16)
        b.table[1, :8] = b.table[0, :8]
        b.table[2, :12] = b.table[0, :12]
        close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 2, 1], [60, 1, 33]])
def test_values_of_any_size(sqa, orc, dev, new):
    for sv in (1e-6, 1e-3, 300.0, 20000.0):
        b = Batch(orc, 4, new, [70, 300, 5], scale_v=sv)
        close(call(sqa, dev, b), b.ref(orc))
    b = Batch(orc, 4, new, [70, 300, 5])
    b.q[:] = 0  # equal weights
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1], [90, 20]])
def test_a_value_far_above_the_others_arrives_late(sqa, orc, dev, new):
    """V scales grow by 2^12 along the keys: the kernels' own scaling of them has to follow."""
    b = Batch(orc, 6, new, [500, 700])
    for r in range(2):
        for j in range(b.kv_len[r]):
            row = b.v[b.table[r, j // 16], j % 16].reshape(-1, 18)
            d = np.ascontiguousarray(row[:, :2]).view(np.float16).astype(np.float64) * 2.0 ** (-6 + 12 * j / b.kv_len[r])
            row[:, :2] = d.astype(np.float16).view(np.uint8)
            b.v[b.table[r, j // 16], j % 16] = row.reshape(b.Hkv, ROW)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1, 1], [130, 1, 70]])
def test_strides_and_alignment(sqa, orc, dev, new):
    b = Batch(orc, 9, new, [90, 400, 33], gate=True)
    want = b.ref(orc)
    (q, k, v, table, qs, kl, max_q), kw = b.args(dev)
    ws = torch.empty(max(16, sqa.paged_attn_workspace_size(q, k, table, max_q)), dtype=torch.uint8, device=dev)
    T, H = q.shape[:2]
    wide = torch.zeros((T, H, 300), device=dev)
    wide[:, :, 7:263] = q
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    gate = torch.zeros((T, H, 260), device=dev)
    gate[:, :, 3:259] = kw["gate"]
    n, page = k.shape[:2]
    pools = []
    for x in (k, v):  # layers of a pool side by side: pages with a stride
        big = torch.full((n, 3, *x.shape[1:]), 0xEE, dtype=torch.uint8, device=dev)
        big[:, 1] = x
        pools.append(big[:, 1])
    tab = torch.full((table.shape[0], table.shape[1] + 5), -9, dtype=torch.int32, device=dev)
    tab[:, 2:2 + table.shape[1]] = table
    for qq, gg, kk, vv, tt in [(wide[:, :, 7:263], gate[:, :, 3:259], k, v, table), (turned, kw["gate"], *pools, table),
                               (q, kw["gate"], pools[0], v, tab[:, 2:2 + table.shape[1]])]:
        out = torch.zeros(q.shape, device=dev)
        sqa.paged_attn(qq, kk, vv, tt, qs, kl, max_q, gate=gg, out=out, workspace=ws)
        close(out.cpu().numpy().astype(np.float64), want)


def test_pool_beyond_4_gib(sqa, orc, dev):
    b = Batch(orc, 2, [1, 40], [300, 200], page=64, spare=0)
    (q, k, v, table, qs, kl, max_q), kw = b.args(dev)
    n, per = b.k.shape[0], 64 * 2 * ROW
    far = (5 << 30) // per
    pools = []
    for x in (k, v):
        big = torch.zeros((far + n, 64, 2, ROW), dtype=torch.uint8, device=dev)
        big[far:] = x
        pools.append(big)
    table = torch.where(table >= 0, table + far, table)
    out = sqa.paged_attn(q, *pools, table, qs, kl, max_q)
    close(out.cpu().numpy().astype(np.float64), b.ref(orc))


@pytest.mark.parametrize("new", [[1] * 5, [2, 1, 2, 1, 1], [1, 90, 1, 200, 5]])
def test_workspaces_paths_and_repeats(sqa, orc, dev, new):
    """A smaller workspace, the other host path, another stream and a second call: the same result, the last three bit for bit."""
    b = Batch(orc, 17, new, [3000, 100, 1500, 700, 0], page=64)
    a, kw = b.args(dev)
    want = b.ref(orc)
    full = sqa.paged_attn_workspace_size(a[0], a[1], a[3], a[6])
    first = call(sqa, dev, b)
    close(first, want)
    assert np.array_equal(call(sqa, dev, b), first)
    assert np.array_equal(call(sqa, dev, b, stream=torch.cuda.current_stream()), first)  # the wrapper's general path
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(sqa, dev, b)
    torch.cuda.synchronize()
    assert np.array_equal(got, first)
    for part in (2, 7):
        try:
            got = call(sqa, dev, b, ws=max(16, full // part))
        except sqa.SqaError as e:
            assert e.status == 3
        else:
            close(got, want)
    out = sqa.paged_attn(*a, **kw)  # everything made by the wrapper
    assert np.array_equal(out.cpu().numpy().astype(np.float64), first)


def test_paged_equals_contiguous(sqa, orc, dev):
    """One request over an identity table: flash_attn_ext_causal over the same rows."""
    for n, past in [(1, 2000), (2, 77), (90, 600)]:
        b = Batch(orc, n, [n], [past], page=64, spare=0)
        a, _ = b.args(dev)
        order = torch.tensor(b.table[0, :b.k.shape[0]], device=dev).long()
        k, v = (x[order].reshape(-1, 2, ROW).contiguous() for x in a[1:3])
        want = sqa.flash_attn_ext_causal(a[0], k, v, n + past, past)
        got = sqa.paged_attn(*a)
        close(got.cpu().numpy().astype(np.float64), want.cpu().numpy().astype(np.float64))


def test_many_requests(sqa, orc, dev):
    r = np.random.default_rng(4)
    for B in (63, 300, 1100):
        new = [int(x) for x in r.choice([0, 1, 1, 1, 2], B)]
        past = [int(x) for x in r.integers(0, 90, B)]
        b = Batch(orc, B, new, past, 4, 2, 16)
        close(call(sqa, dev, b), b.ref(orc))
    new[5], new[700] = 60, 33
    b = Batch(orc, 5, new, past, 4, 2, 16)
    close(call(sqa, dev, b), b.ref(orc))


def test_more_chunks_than_the_plan_lists(sqa, orc, dev):
    """1100 requests of 20 tokens and 4 KV heads are 4400 parts of the many-row kernel."""
    r = np.random.default_rng(6)
    new, past = [20] * 1100, [int(x) for x in r.integers(0, 40, 1100)]
    new[3], new[500], past[500] = 0, 150, 300
    b = Batch(orc, 6, new, past, 4, 4, 16)
    close(call(sqa, dev, b), b.ref(orc))


def test_chunks_among_thousands_of_requests(sqa, orc, dev):
    r = np.random.default_rng(7)
    new = [int(x) for x in r.choice([0, 1, 1, 1, 2, 30], 2700)]
    past = [int(x) for x in r.integers(0, 40, 2700)]
    b = Batch(orc, 7, new, past, 4, 4, 16)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1, 1], [150, 1, 90]])
def test_two_calls_at_once(sqa, orc, dev, new):
    """On two streams, each with its own workspace."""
    pair = [Batch(orc, 40 + i, new, [700 - 300 * i, 2000, 65], gate=i == 1) for i in (0, 1)]
    made = [(b.args(dev), torch.zeros(b.q.shape, device=dev)) for b in pair]
    size = sqa.paged_attn_workspace_size(made[0][0][0][0], made[0][0][0][1], made[0][0][0][3], max(new))
    works = [torch.full((size,), 0xFF, dtype=torch.uint8, device=dev) for _ in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for _ in range(8):
        for ((a, kw), out), work, s in zip(made, works, streams):
            with torch.cuda.stream(s):
                sqa.paged_attn(*a, **kw, out=out, workspace=work)
    torch.cuda.synchronize()
    for b, (_, out) in zip(pair, made):
        close(out.cpu().numpy().astype(np.float64), b.ref(orc))


@pytest.mark.parametrize("n,H,Hkv", [(1, 16, 2), (2, 16, 2), (4, 4, 2), (40, 16, 2)])
def test_bias_over_many_tiles(sqa, orc, dev, n, H, Hkv):
    """Slopes that leave only the last keys, and slopes that leave all, over whole and cut tiles."""
    b = Batch(orc, n + H, [n, n, n], [2000, 65, 0], H, Hkv, 64, gate=n == 2)
    for bias in (1.0, 8.0, 30.0):
        close(call(sqa, dev, b, max_bias=bias), b.ref(orc, bias=bias))


@pytest.mark.parametrize("new", [[1], [2], [40]])
def test_weights_keep_their_bits(sqa, orc, dev, new):
    """Logits within some 3 roundings of 2^-24 of their block terms (about 1 here), P and P d_v at
    22 bits: below 1e-6 of the output together, where thousands of keys share the weight."""
    b = Batch(orc, 3, new, [4096], page=64)
    got, want = call(sqa, dev, b), b.ref(orc)
    assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


def test_more_kv_heads_than_workgroups_run_together(sqa, orc, dev):
    for new in ([1, 1], [30, 1]):
        b = Batch(orc, 8, new, [50, 70], 600, 600, 16)
        close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1], [2, 2, 1], [4, 60, 1]])
@pytest.mark.parametrize("opt", [{}, {"softcap": 20.0, "max_bias": 8.0}])
def test_a_row_that_is_not_finite_stays_alone(sqa, orc, dev, new, opt):
    b = Batch(orc, 12, new, [300, 90, 40][:len(new)], page=32)
    want = b.ref(orc, cap=opt.get("softcap", 0.0), bias=opt.get("max_bias", 0.0))
    bad = [(0, 3, np.nan), (1, 9, np.inf), (b.q_start[-1] - 1, 15, -np.inf)]
    for t, h, x in bad:
        b.q[t, h, 7] = x
    got = call(sqa, dev, b, **opt)
    ok = np.ones(want.shape[:2], dtype=bool)
    for t, h, _ in bad:
        ok[t, h] = False
    close(got[ok], want[ok])


@pytest.mark.parametrize("new", [[1, 2], [40, 1]])
def test_rows_before_and_behind_the_requests_stay(sqa, orc, dev, new):
    b = Batch(orc, 13, new, [100, 30], pad=8)
    b.q_start = [t + 5 for t in b.q_start]
    close(call(sqa, dev, b, fill=7.0), b.ref(orc, fill=7.0))
