"""Attention of requests that share prefixes against the float64 definition; the tolerances are those of
test_gpu_paged_attn.py: the arithmetic of a key is the same, and the merge of the two parts multiplies each by a
weight of 2^-22 or better."""
import math

import numpy as np
import pytest
import torch

import paged_ref
import shared_ref
from test_gpu_paged_attn import SHAPES, close

pytestmark = pytest.mark.gpu

D, ROW = 256, 144


class Batch:
    """Inputs of a call: own and shared pages dealt out of one pool with spare and garbage pages."""

    def __init__(self, orc, seed, new, past, shared, group, H=16, Hkv=2, page=16, prefix=None, pad=0, spare=3, gate=False,
                 scale_v=1.0, scale_q=1.0):
        r = self.r = np.random.default_rng(seed)
        self.H, self.Hkv, self.page, self.shared, self.group = H, Hkv, page, list(shared), list(group)
        self.kv_len = [n + p for n, p in zip(new, past)]
        lens = [max(0, x) for x in self.kv_len + self.shared]
        used = [-(-n // page) for n in lens]
        n_pages, B, W = sum(used) + spare, len(new), max(1, max(used)) + 1
        order = r.permutation(n_pages)
        self.k, self.v = (np.full((n_pages, page, Hkv, ROW), 0xFF, dtype=np.uint8) for _ in range(2))  # NaN scales
        table, at = np.full((len(used), W), -1, dtype=np.int32), 0
        for b, (u, n) in enumerate(zip(used, lens)):
            ids = table[b, :u] = order[at:at + u]
            at += u
            for pool, s in ((self.k, 1.0), (self.v, scale_v)):
                x = paged_ref.quantize(orc, np.float32(s) * r.standard_normal((n, Hkv, D), dtype=np.float32)) if n else None
                for j in range(0, n, page):
                    pool[ids[j // page], :min(page, n - j)] = x[j:j + page]
        self.table, self.shared_table = table[:B].copy(), table[B:].copy()
        self.q_start = [0]
        for n in new:
            self.q_start.append(self.q_start[-1] + n)
        T = max(1, self.q_start[-1] + pad)
        self.q = np.float32(scale_q) * r.standard_normal((T, H, D), dtype=np.float32)
        self.gate = r.standard_normal((T, H, D), dtype=np.float32) if gate else None
        self.prefix, self.max_q = prefix, max(1, max(new))

    def ref(self, orc, fill=0.0, **kw):
        return shared_ref.attention(orc, self.q, self.k, self.v, self.table, self.q_start, self.kv_len, self.shared_table,
                                    self.shared, self.group, self.prefix, gate=self.gate, fill=fill, **kw)

    def args(self, sqa, dev):
        t = lambda x, d=torch.int32: torch.tensor(np.asarray(x), dtype=d, device=dev)  # noqa: E731
        T = self.q.shape[0]
        starts, kv, slen = t(self.q_start), t(self.kv_len), t(self.shared)
        share = sqa.paged_share(starts, kv, t(self.group), slen, torch.zeros(T, dtype=torch.int32, device=dev))
        a = [t(self.q, torch.float32), t(self.k, torch.uint8), t(self.v, torch.uint8), t(self.table), starts, kv,
             t(self.shared_table), slen, share, self.max_q]
        kw = {"prefix": None if self.prefix is None else t(self.prefix),
              "gate": None if self.gate is None else t(self.gate, torch.float32)}
        return a, kw


def call(sqa, dev, batch, fill=None, ws=None, **kw):
    a, opt = batch.args(sqa, dev)
    out = torch.full(batch.q.shape, 0.0 if fill is None else fill, device=dev)
    if ws is None:
        ws = max(16, sqa.paged_attn_shared_workspace_size(a[0], a[1], a[3], a[6], a[9]))
    work = torch.full((ws,), 0xFF, dtype=torch.uint8, device=dev)  # NaN wherever the workspace is not written
    got = sqa.paged_attn_shared(*a, **opt, out=out, workspace=work, **kw)
    assert got is out
    return out.cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("H,Hkv", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 512])
def test_decode(sqa, orc, dev, H, Hkv, page):
    past = [0, 1, 14, 15, 16, 31, 62, 63, 64, 127, 300, 5, 9]
    b = Batch(orc, H * 100 + page, [1] * len(past), past, [331, 64, 1], [0, 0, 1, 0, -1, 2, 0, 0, 1, 0, 0, 0, 1], H, Hkv, page)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("shared", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 257, 1000, 2049])
def test_lengths_of_the_prefix(sqa, orc, dev, shared):
    b = Batch(orc, shared, [1] * 6, [0, 3, 70, 16, 15, 200], [shared], [0] * 6, page=32)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("B", [1, 2, 3, 7, 8, 9, 16, 17, 33, 64, 130])
def test_sizes_of_the_group(sqa, orc, dev, B):
    r = np.random.default_rng(B)
    b = Batch(orc, B, [1] * B, r.integers(0, 60, B).tolist(), [150], [0] * B, page=16)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("n", [2, 3, 4])
@pytest.mark.parametrize("H,Hkv", [(16, 2), (4, 4), (6, 2), (16, 4)])
def test_verify(sqa, orc, dev, n, H, Hkv):
    past = [0, 1, 13, 61, 62, 63, 64, 190, 555]
    new = [1 + (i + n) % n for i in range(len(past))]
    new[3] = n
    b = Batch(orc, 7 * n + H, new, past, [400, 77], [0, 1, 0, 0, 1, -1, 0, 1, 0], H, Hkv, 32, pad=5)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new,past", [([3, 17, 1], [0, 0, 9]), ([64, 65, 31], [0, 1, 33]), ([100, 1, 129], [29, 5, 0]), ([300, 7], [0, 500])])
@pytest.mark.parametrize("H,Hkv,page", [(16, 2, 16), (16, 4, 64), (4, 4, 32), (6, 2, 16), (5, 1, 128)])
def test_chunks(sqa, orc, dev, new, past, H, Hkv, page):
    b = Batch(orc, sum(new) + H, new, past, [333, 50], [0, 0, 1][:len(new)], H, Hkv, page, pad=3)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("opt", [{"softcap": 30.0}, {"max_bias": 8.0}, {"softcap": 5.0, "max_bias": 2.0}, {"scale": 0.02}])
@pytest.mark.parametrize("new", [[1] * 7, [1, 2, 1, 3, 1, 1, 2], [40, 1, 70, 1, 9, 1, 0]])
def test_options_gate_and_own_prefix(sqa, orc, dev, opt, new):
    names = {"softcap": "cap", "max_bias": "bias", "scale": "scale"}
    b = Batch(orc, 11, new, [90, 3, 0, 250, 16, 1, 40], [500, 31], [0, 1, 0, -1, 1, 0, 0], page=32, gate=True, pad=2,
              prefix=[0, 4, 60, 100, 0, 2, 7], scale_q=2.0)
    close(call(sqa, dev, b, **opt), b.ref(orc, **{names[k]: v for k, v in opt.items()}))


def test_equals_a_request_that_holds_the_prefix_itself(sqa, orc, dev):
    """The same keys in one table row, by paged_attn."""
    page, S = 16, 160  # whole pages, so that one row can name both
    b = Batch(orc, 3, [1, 2, 40], [5, 30, 2], [S], [0, 0, 0], page=page)
    got = call(sqa, dev, b)
    a, _ = b.args(sqa, dev)
    table = torch.cat([a[6][:, :S // page].expand(3, -1), a[3]], 1).contiguous()
    want = sqa.paged_attn(a[0], a[1], a[2], table, a[4], a[5] + S, b.max_q)
    close(got, want.cpu().numpy().astype(np.float64))


def test_rows_that_see_nothing_and_rows_of_nobody(sqa, orc, dev):
    """Refused requests (kv_len 0) get zeros, prefix or not; rows of no request stay."""
    b = Batch(orc, 5, [1, 2, 1, 3], [4, 9, 20, 0], [90], [0, 0, 0, 0], pad=4)
    b.kv_len[1] = 0
    got, want = call(sqa, dev, b, fill=7.0), b.ref(orc, fill=7.0)
    assert (got[1:3] == 0).all() and (got[-4:] == 7.0).all()
    close(got[:7], want[:7])
    # rows before the requests
    b.q_start = [2, 3, 5, 6, 7]
    got, want = call(sqa, dev, b, fill=7.0), b.ref(orc, fill=7.0)
    assert (got[:2] == 7.0).all() and (got[7:] == 7.0).all()
    close(got[2:7], want[2:7])


def test_pages_outside_the_pool_and_lengths_past_the_table(sqa, orc, dev):
    b = Batch(orc, 6, [1, 1, 20], [40, 7, 3], [130, 40], [0, 1, 0], page=16)
    b.shared_table[0, 2], b.shared_table[0, 5] = -1, 1 << 30
    b.shared_table[1, :] = -5       # a prefix of which no page is there
    b.table[0, 1] = 10_000
    close(call(sqa, dev, b), b.ref(orc))
    b.table[1, :] = -1               # and nothing of its own: a row that sees nothing
    got = call(sqa, dev, b)
    assert (got[1] == 0).all()
    close(got, b.ref(orc))
    # lengths past the table's last page: those keys are not there
    b = Batch(orc, 7, [1, 1], [4, 4], [64], [0, 0], page=16)
    b.shared_table = b.shared_table[:, :4].copy()
    want = b.ref(orc)
    b.shared = [1 << 30]
    close(call(sqa, dev, b), want)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [1, 30, 1, 2]])
def test_not_finite_rows_stay_alone(sqa, orc, dev, new):
    b = Batch(orc, 8, new, [10, 2, 33, 5], [200], [0, 0, -1, 0])
    want = b.ref(orc)
    clean = call(sqa, dev, b)
    b.q[0, 3, 17], b.q[2, 15, 255], b.q[-1, 0, 0] = np.nan, np.inf, -np.inf
    got = call(sqa, dev, b)
    bad = np.zeros(got.shape[:2], bool)
    bad[0, 3] = bad[2, 15] = bad[-1, 0] = True
    assert np.isnan(got[bad]).all()
    assert np.array_equal(got[~bad], clean[~bad])
    close(clean, want)


@pytest.mark.parametrize("scale_v,scale_q", [(1e-6, 1.0), (3000.0, 1.0), (1.0, 40.0), (1.0, 1e-6)])
def test_sizes_of_values(sqa, orc, dev, scale_v, scale_q):
    """A sharp softmax (a key has nearly all the weight, in either part), a flat one, V of any size."""
    b = Batch(orc, 9, [1, 1, 2, 50], [60, 0, 9, 0], [300], [0, 0, 0, 0], scale_v=scale_v, scale_q=scale_q)
    got, want = call(sqa, dev, b), b.ref(orc)
    # logits grow with q: the error of a logit (and so of a weight) is 1.5e-5 at 2^5, and is relative to the largest one
    top = scale_q * 4 * math.log2(math.e)
    factor = max(1.0, top / 32)
    d = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert d <= 2e-5 * factor, d


def test_garbage_behind_the_prefix_is_never_seen(sqa, orc, dev):
    b = Batch(orc, 10, [1] * 5, [3] * 5, [45], [0] * 5, page=64)
    one = call(sqa, dev, b)
    page = b.shared_table[0, 0]
    b.k[page, 45:], b.v[page, 45:] = 0x7B, 0x00
    assert np.array_equal(call(sqa, dev, b), one)


def test_strides_in_place_and_tables_of_the_batch(sqa, orc, dev):
    """q as the engine permutes it, dst as q, the groups' rows in the batch's own table."""
    b = Batch(orc, 12, [1, 2, 1], [9, 30, 0], [70, 20], [0, 1, 0], pad=1, gate=True)
    want = b.ref(orc)
    a, kw = b.args(sqa, dev)
    T = b.q.shape[0]
    wide = torch.zeros((16, T + 3, D + 5), device=dev)
    wide[:, :T, :D] = a[0].transpose(0, 1)
    view = wide[:, :T, :D].transpose(0, 1)
    ws = torch.empty(sqa.paged_attn_shared_workspace_size(view, a[1], a[3], a[6], a[9]), dtype=torch.uint8, device=dev)
    got = sqa.paged_attn_shared(view, *a[1:], **kw, workspace=ws, out=torch.zeros_like(a[0]))
    close(got.cpu().numpy().astype(np.float64), want)
    both = torch.cat([a[3], a[6]]).contiguous()
    x = a[0].clone()
    sqa.paged_attn_shared(x, a[1], a[2], both[:3], *a[4:6], both[3:], *a[7:], **kw, out=x, workspace=ws)
    assert torch.equal(x[:4], got[:4])
    # a workspace of the least size gives the same up to the order of sums
    for size in (ws.numel() // 64, ws.numel() // 8, ws.numel() // 2):
        try:
            y = sqa.paged_attn_shared(*a, **kw, out=torch.zeros_like(a[0]), workspace=ws[:size])
        except sqa.SqaError as e:
            assert e.status == 3
            continue
        close(y.cpu().numpy().astype(np.float64), want)
    with pytest.raises(sqa.SqaError):
        sqa.paged_attn_shared(*a, **kw, out=torch.zeros_like(a[0]), workspace=ws[:64])


def test_results_repeat_bit_for_bit(sqa, orc, dev):
    b = Batch(orc, 13, [1] * 40 + [30], [int(x) for x in np.random.default_rng(1).integers(0, 300, 41)], [900, 300],
              [i % 3 - 1 for i in range(41)])
    one = call(sqa, dev, b)
    for _ in range(3):
        assert np.array_equal(call(sqa, dev, b), one)


def test_groups_of_another_step_stay_inside(sqa, orc, dev):
    """Members, starts and groups that no plan wrote: unspecified rows, nothing else is touched, later calls are right."""
    b = Batch(orc, 14, [1, 2, 3, 1], [9, 30, 0, 4], [70, 20], [0, 1, 0, -1], pad=2)
    a, _ = b.args(sqa, dev)
    T = b.q.shape[0]
    r = torch.Generator(device=dev).manual_seed(1)
    ws = torch.empty(sqa.paged_attn_shared_workspace_size(a[0], a[1], a[3], a[6], a[9]), dtype=torch.uint8, device=dev)
    guard = torch.full((T + 8, 16, D), 3.0, device=dev)
    for low, high in ((-5, T + 5), (-(1 << 31), (1 << 31) - 1), (0, 2)):
        junk = sqa.PagedShare(*(torch.randint(low, high, x.shape, generator=r, device=dev, dtype=torch.int64).to(torch.int32) for x in a[8]))
        ws.copy_(torch.randint(0, 256, ws.shape, generator=r, device=dev, dtype=torch.uint8))
        sqa.paged_attn_shared(*a[:8], junk, *a[9:], out=guard[4:T + 4], workspace=ws)
        torch.cuda.synchronize()
        assert (guard[:4] == 3.0).all() and (guard[T + 4:] == 3.0).all()
    close(call(sqa, dev, b), b.ref(orc))


def test_a_given_stream_makes_its_own_tensors(sqa, orc, dev):
    b = Batch(orc, 15, [1, 40, 2], [700, 3, 90], [400], [0, 0, -1], page=64)
    a, _ = b.args(sqa, dev)
    want = sqa.paged_attn_shared(*a)
    s = torch.cuda.Stream()
    for handle in (s, s.cuda_stream):
        torch.cuda.synchronize()
        torch.cuda._sleep(24_000_000)
        got = sqa.paged_attn_shared(*a, stream=handle)
        s.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_random_batches(sqa, orc, dev):
    r = np.random.default_rng(77)
    for k in range(30):
        H, Hkv = [(16, 2), (8, 2), (4, 1), (12, 4), (32, 2), (3, 3)][k % 6]
        B, G = int(r.integers(1, 40)), int(r.integers(1, 6))
        new = r.choice([0, 1, 1, 1, 2, 4, int(r.integers(1, 60))], B).tolist()
        past = r.integers(0, 150, B).tolist()
        shared = r.choice([0, 1, 16, 40, 129, int(r.integers(1, 700))], G).tolist()
        group = r.integers(-1, G + 1, B).tolist()
        opt = [{}, {"softcap": 20.0}, {"max_bias": 4.0}][int(r.integers(0, 3))]
        b = Batch(orc, 1000 + k, [int(x) for x in new], past, [int(x) for x in shared], group, H, Hkv, int(r.choice([16, 32, 128])),
                  pad=int(r.integers(0, 5)), gate=bool(r.integers(0, 2)))
        want = b.ref(orc, **{{"softcap": "cap", "max_bias": "bias"}[k]: v for k, v in opt.items()})
        print(k, H, Hkv, B, G, opt)
        close(call(sqa, dev, b, **opt), want)


@pytest.mark.parametrize("B,G", [(70, 1), (70, 90), (300, 300), (1500, 40), (1300, 2500)])
@pytest.mark.parametrize("most", [1, 9, 40])
def test_many_requests_and_groups(sqa, orc, dev, B, G, most):
    """More requests and groups than a wavefront's lanes, and than the few-row kernel keeps."""
    r = np.random.default_rng(B + G)
    new = [int(x) for x in r.choice([0, 1, 1, 1, most], B)]
    group = [int(x) for x in r.integers(-1, G, B)]
    b = Batch(orc, B + G, new, [int(x) for x in r.integers(0, 40, B)], [int(x) for x in r.integers(0, 90, G)], group, 4, 4, 16)
    close(call(sqa, dev, b), b.ref(orc))


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [150, 1, 90, 0]])
def test_two_calls_at_once(sqa, orc, dev, new):
    """On two streams, each with its own workspace."""
    pair = [Batch(orc, 40 + i, new, [700 - 300 * i, 2000, 65, 8], [900, 30 + i], [0, i, 0, 1], gate=i == 1) for i in (0, 1)]
    made = [(b.args(sqa, dev), torch.zeros(b.q.shape, device=dev)) for b in pair]
    a = made[0][0][0]
    size = sqa.paged_attn_shared_workspace_size(a[0], a[1], a[3], a[6], max(new))
    works = [torch.full((size,), 0xFF, dtype=torch.uint8, device=dev) for _ in pair]
    streams = [torch.cuda.Stream() for _ in pair]
    torch.cuda.synchronize()
    for _ in range(8):
        for ((a, kw), out), work, s in zip(made, works, streams):
            with torch.cuda.stream(s):
                sqa.paged_attn_shared(*a, **kw, out=out, workspace=work)
    torch.cuda.synchronize()
    for b, (_, out) in zip(pair, made):
        close(out.cpu().numpy().astype(np.float64), b.ref(orc))


@pytest.mark.parametrize("new", [[40, 1, 17, 130], [9, 9, 8, 1]])
def test_chunks_in_place_and_in_small_workspaces(sqa, orc, dev, new):
    """dst as q and as the gate, chunks and members that split over many keys; every workspace that a call takes."""
    b = Batch(orc, 16, new, [300, 20, 0, 64], [1500, 200], [0, 0, 1, -1], gate=True)
    a, kw = b.args(sqa, dev)
    full = sqa.paged_attn_shared_workspace_size(a[0], a[1], a[3], a[6], a[9])
    ws = torch.full((full,), 0xFF, dtype=torch.uint8, device=dev)
    want = sqa.paged_attn_shared(*a, **kw, out=torch.zeros_like(a[0]), workspace=ws)
    close(want.cpu().numpy().astype(np.float64), b.ref(orc))
    x = a[0].clone()
    sqa.paged_attn_shared(x, *a[1:], **kw, out=x, workspace=ws)
    assert torch.equal(x, want)
    g = kw["gate"].clone()
    sqa.paged_attn_shared(*a, gate=g, out=g, workspace=ws)
    assert torch.equal(g, want)
    taken = 0
    for size in [*range(full // 40 * 40, 0, -full // 40), 256]:
        ws.fill_(0xFF)
        y = torch.zeros_like(a[0])
        try:
            sqa.paged_attn_shared(*a, **kw, out=y, workspace=ws[:size])
        except sqa.SqaError as e:
            assert e.status == 3 and not y.any()
            continue
        taken += 1
        close(y.cpu().numpy().astype(np.float64), b.ref(orc))
        assert (ws[size:] == 0xFF).all()
    assert 0 < taken <= 40  # (some 0.6 MB are needed, and 256 bytes are not enough)


def test_more_tokens_than_max_q(sqa, orc, dev):
    """Rows of requests with more than max_q tokens may be left as they were: the others are right."""
    new = [1, 60, 1, 3]
    b = Batch(orc, 17, new, [30, 20, 100, 64], [700], [0, 0, 0, -1])
    want = b.ref(orc)
    for max_q in (1, 3):
        b.max_q = max_q
        got = call(sqa, dev, b)
        for i, n in enumerate(new):
            if n <= max_q:
                at = slice(b.q_start[i], b.q_start[i + 1])
                close(got[at], want[at])


@pytest.mark.parametrize("n", [1, 2, 40])
def test_bias_over_many_tiles(sqa, orc, dev, n):
    """Slopes that leave only the last keys, and slopes that leave the whole prefix too."""
    b = Batch(orc, 18, [n, n, n], [2000, 65, 0], [900, 64], [0, 1, 1], page=64, gate=n == 2)
    for bias in (1.0, 8.0, 30.0):
        close(call(sqa, dev, b, max_bias=bias), b.ref(orc, bias=bias))


@pytest.mark.parametrize("B,n", [(1, 1), (24, 1), (3, 40)])
def test_weights_keep_their_bits(sqa, orc, dev, B, n):
    """As for requests that share nothing: logits within some 3 roundings of 2^-24, P and P d_v at 22 bits, below 1e-6 of
    the output together; the two parts' weights in the merge add 2^-22."""
    b = Batch(orc, 19, [n] * B, [100] * B, [4096], [0] * B, page=64)
    got, want = call(sqa, dev, b), b.ref(orc)
    assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


@pytest.mark.parametrize("max_q", [1, 4, 40])
def test_ranges_that_overlap_stay_inside(sqa, orc, dev, max_q):
    """q_start that goes up and down, more requests than the workspace has slots for: unspecified rows, nothing else is
    touched whatever the workspace held, later calls are right."""
    b = Batch(orc, 20, [1, 2, 1, 40], [9, 30, 0, 5], [70, 20], [0, 1, 0, 1], pad=2)
    a, _ = b.args(sqa, dev)
    T, n = b.q.shape[0], 600
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    starts, lens = i32([0, 4] * (n // 2) + [0]), i32([40] * n)
    starts[n] = T
    table = a[3][:1].repeat(n, 1)
    ws = torch.empty(sqa.paged_attn_shared_workspace_size(a[0], a[1], table, a[6], max_q), dtype=torch.uint8, device=dev)
    guard = torch.full((T + 8, 16, D), 3.0, device=dev)
    r = torch.Generator(device=dev).manual_seed(2)
    for fill in (0xFF, None):
        if fill is None:
            ws.copy_(torch.randint(0, 256, ws.shape, generator=r, device=dev, dtype=torch.uint8))
        else:
            ws.fill_(fill)
        share = sqa.paged_share(starts, lens, i32([0, 1, -1] * (n // 3)), a[7], torch.zeros(T, dtype=torch.int32, device=dev))
        sqa.paged_attn_shared(a[0], a[1], a[2], table, starts, lens, a[6], a[7], share, max_q, out=guard[4:T + 4], workspace=ws)
        torch.cuda.synchronize()
        assert (guard[:4] == 3.0).all() and (guard[T + 4:] == 3.0).all()
    close(call(sqa, dev, b), b.ref(orc))
