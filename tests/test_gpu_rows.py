"""Cached rows read back and moved, against the definitions in 64 bits.

get_rows: a value is a 4-bit code times an 11-bit scale, exact in float32; float16 is that rounded once.
move_rows: rows without a rope, and blocks without a rotated dim, keep their bytes. A rotated value is two products
and a sum in float32 of float32 cos and sin: off by at most (|x0| + |x1|) * 3 * 2^-24, and requantised it may
land on the code beside the definition's where the definition's own value lies that close to a border between codes
(or, its block's scale being the value of largest size over -8, where two values' sizes lie that close)."""
import numpy as np
import pytest
import torch

import shared_ref as ref

pytestmark = pytest.mark.gpu

ROPE = (64, (11, 11, 10, 0), 1e7)


def cache(orc, r, rows, heads, D=256, scale=1.0):
    x = np.float32(scale) * r.standard_normal((rows, heads * D), dtype=np.float32)
    return orc.quantize_q4_0(x).reshape(rows, heads, D // 32 * 18)


def gpu(x, dev):
    return torch.tensor(np.asarray(x), device=dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,heads,D", [(1, 1, 32), (1, 2, 256), (3, 1, 256), (57, 2, 256), (64, 3, 96), (1000, 2, 256), (4097, 1, 64)])
def test_get_rows(sqa, orc, dev, dtype, n, heads, D):
    r = np.random.default_rng(n + D)
    c = cache(orc, r, 700, heads, D, scale=3.0)
    idx = r.integers(0, 700, n)
    got = sqa.get_rows_q4_0(gpu(c, dev), gpu(idx, dev), dtype=dtype)
    want = ref.values(c[idx].reshape(n, -1))
    assert got.dtype == dtype and got.shape == (n, heads * D)
    want = want.astype(np.float32) if dtype == torch.float32 else want.astype(np.float16)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_get_rows_outside_strides_and_extremes(sqa, orc, dev, dtype):
    r = np.random.default_rng(5)
    c = cache(orc, r, 40, 2)
    c[3].reshape(-1, 18)[:, :2] = np.array([65504.0], np.float16).view(np.uint8)   # largest scale: 8 d is past float16
    c[4].reshape(-1, 18)[:, :2] = np.array([6e-8], np.float16).view(np.uint8)      # smallest subnormal
    c[5].reshape(-1, 18)[:, :2] = np.array([np.inf], np.float16).view(np.uint8)
    idx = np.array([3, 4, -1, 40, 1 << 40, 39, 0, 0, -(1 << 62), 5])
    wide = np.repeat(idx[:, None], 3, 1).copy()
    out = torch.full((12, 640), 7.0, dtype=dtype, device=dev)
    view = out[1:11, 33:33 + 512]  # odd offset, rows apart
    got = sqa.get_rows_q4_0(gpu(c, dev), gpu(wide, dev)[:, 1], out=view)
    assert got.data_ptr() == view.data_ptr()
    ok = (idx >= 0) & (idx < 40)
    with np.errstate(all="ignore"):
        want = np.where(ok[:, None], ref.values(c[np.where(ok, idx, 0)].reshape(10, -1)), 0.0)
        want = want.astype(np.float32).astype(np.float16) if dtype == torch.float16 else want.astype(np.float32)
    assert np.array_equal(view.cpu().numpy(), want, equal_nan=True)
    rest = out.clone()
    rest[1:11, 33:33 + 512] = 7.0
    assert (rest == 7.0).all()
    # a flat cache, two dims
    flat = sqa.get_rows_q4_0(gpu(c, dev).view(40, -1), gpu(np.array([7, 9]), dev))
    assert np.array_equal(flat.cpu().numpy(), ref.values(c[[7, 9]].reshape(2, -1)).astype(np.float32))
    assert sqa.get_rows_q4_0(gpu(c, dev), torch.empty(0, dtype=torch.int64, device=dev)).shape == (0, 512)


def test_get_rows_gives_what_set_rows_wrote(sqa, dev):
    kv = sqa.KvCache(2, 256, 2, 512, device=dev)
    x = torch.randn((300, 512), device=dev)
    idx = torch.randperm(512, device=dev)[:300]
    kv.begin_step(300)
    kv.append(1, x, 2 * x, idx)
    k, v = kv.read(1, idx), kv.read(1, idx, "v", dtype=torch.float16)
    # A code is off by at most half a step d = top / 8, and at the end opposite the largest value, which 7 steps reach,
    # by a whole one. The scale is then rounded to float16, by 2^-11 of it at most, and a code of up to 8 carries 8 times
    # that: 8 * 2^-11 d = 2^-8 d beside the whole step.
    top = x.view(300, 16, 32).abs().amax(-1, keepdim=True)
    assert ((k.view(300, 16, 32) - x.view(300, 16, 32)).abs() <= top / 8 * (1 + 2.0 ** -8)).all()
    again = torch.zeros_like(kv.k[1])
    sqa.set_rows_q4_0(again, k, idx)
    assert torch.equal(again[idx], kv.k[1][idx])  # values on the grid quantize to themselves
    assert torch.equal(v.float(), sqa.get_rows_q4_0(kv.v[1], idx).half().float())


def check_move(orc, before, src, got, to, frm, delta, rope, freq_scale=1.0):
    """got: dst after the call, of `before`; the entries of to and frm that are inside, each row of to once."""
    n_rot, sections, base = rope
    n, (_, heads, rb) = len(to), before.shape
    ok = (frm >= 0) & (frm < src.shape[0]) & (to >= 0) & (to < before.shape[0])
    rows = src[np.where(ok, frm, 0)]
    d = np.asarray(delta).reshape(4, n)
    y = ref.turned(rows, d, n_rot, sections, base, freq_scale)
    turned = (n_rot + 31) // 32
    want = before.copy()
    want[to[ok]] = rows[ok]
    rot = orc.quantize_q4_0(np.ascontiguousarray(y[..., :32 * turned], dtype=np.float32)).reshape(n, heads, turned * 18)
    want[to[ok], :, :turned * 18] = rot[ok]
    same = got == want
    # bytes that differ: the blocks of a value beside a border
    bad = np.argwhere(~same)
    allowed = 0
    half = n_rot // 2
    x = np.abs(ref.values(rows))
    x0 = np.concatenate([x[..., :half] + x[..., half:n_rot]] * 2 + [x[..., n_rot:]], -1)
    back = {int(t): i for i, t in enumerate(to) if ok[i]}
    for r_, h, byte in {(int(a), int(b), int(c) // 18) for a, b, c in bad}:
        assert r_ in back and byte < turned, (r_, h, byte)
        i, at = back[r_], slice(32 * byte, 32 * byte + 32)
        v, slack = y[i, h, at], x0[i, h, at] * 3 * 2.0 ** -24
        top = np.abs(v).max()
        near = np.abs(v) >= top - 2 * slack.max()
        tie = near.sum() > 1
        scale = v[np.argmax(np.abs(v))] / -8
        frac = v / scale + 8.5
        border = np.abs(frac - np.round(frac)) <= 2 * (slack.max() + 2.0 ** -23 * top) / abs(scale) + 2.0 ** -20
        half_ulp = np.spacing(np.float16(abs(scale))) / 2
        edge = abs(abs(abs(scale) - float(np.float16(abs(scale)))) - half_ulp) <= slack.max() / 4
        assert tie or border.any() or edge, (r_, h, byte, got[r_, h, byte * 18:byte * 18 + 18], want[r_, h, byte * 18:byte * 18 + 18])
        allowed += 1
    print(f"{allowed} of {max(1, int(ok.sum()) * heads * turned)} rotated blocks at a border between codes")
    # the chance of a border is some 40 values' slack of 2^-22 steps each
    assert allowed <= 3 + int(ok.sum()) * heads * turned * 32 * 2.0 ** -16


@pytest.mark.parametrize("n,heads", [(1, 1), (2, 2), (31, 2), (500, 2), (1003, 4), (64, 5)])
@pytest.mark.parametrize("D,rope", [(256, ROPE), (128, (128, (16, 24, 24, 0), 1e6)), (64, (40, (8, 6, 6, 0), 1e4)),
                                    (256, (256, (44, 44, 40, 0), 1e7)), (256, (8, (4, 0, 0, 0), 5e5)), (256, (72, (0, 0, 0, 5), 1e7))])
def test_move_rows(sqa, orc, dev, n, heads, D, rope):
    r = np.random.default_rng(n * heads + D)
    src, dst = cache(orc, r, n + 20, heads, D), cache(orc, r, 2 * n + 5, heads, D)
    frm, to = r.permutation(n + 20)[:n], r.permutation(2 * n + 5)[:n]
    delta = r.integers(-200000, 200000, (4, n)).astype(np.int32)
    g = gpu(dst, dev)
    assert sqa.move_rows_q4_0(g, gpu(src, dev), gpu(to, dev), gpu(frm, dev), gpu(delta.reshape(-1), dev), sqa.rope_params(*rope)) is g
    check_move(orc, dst, src, g.cpu().numpy(), to, frm, delta, rope)


def test_move_rows_copies_without_a_rope(sqa, orc, dev):
    r = np.random.default_rng(2)
    for heads, D, n in ((2, 256, 777), (1, 32, 5), (3, 96, 40), (1, 512, 9)):
        src, dst = (r.integers(0, 256, (n + 3, heads, D // 32 * 18)).astype(np.uint8) for _ in range(2))
        frm, to = r.permutation(n + 3)[:n], r.permutation(n + 3)[:n]
        frm[0], to[min(1, n - 1)] = -1, n + 3
        g = gpu(dst, dev)
        sqa.move_rows_q4_0(g, gpu(src, dev), gpu(to, dev), gpu(frm, dev))
        ok = (frm >= 0) & (to < n + 3)
        dst[to[ok]] = src[frm[ok]]
        assert np.array_equal(g.cpu().numpy(), dst)


def test_move_rows_in_place_outside_and_no_turn(sqa, orc, dev):
    r = np.random.default_rng(3)
    c = cache(orc, r, 300, 2)
    rope = sqa.rope_params(*ROPE)
    rows = r.permutation(300)[:100]
    rows[7], rows[50] = -5, 300
    delta = np.repeat(np.array([-1234, 77, 5, 0], np.int32)[:, None], 100, 1)
    g, at = gpu(c, dev), gpu(rows, dev)
    sqa.move_rows_q4_0(g, g, at, at, gpu(delta.reshape(-1), dev), rope)
    check_move(orc, c, c, g.cpu().numpy(), rows, rows, delta, ROPE)
    # disjoint ranges of one cache; a turn of nothing leaves values that a quantizer wrote as they are
    g, lo, hi = gpu(c, dev), torch.arange(0, 120, device=dev), torch.arange(150, 270, device=dev)
    sqa.move_rows_q4_0(g, g, lo, hi, torch.zeros(480, dtype=torch.int32, device=dev), rope)
    want = c.copy()
    want[:120] = c[150:270]
    assert np.array_equal(g.cpu().numpy(), want)
    empty = torch.empty(0, dtype=torch.int64, device=dev)
    sqa.move_rows_q4_0(g, g, empty, empty, torch.empty(0, dtype=torch.int32, device=dev), rope)
    assert np.array_equal(g.cpu().numpy(), want)


def test_moved_keys_are_those_of_the_other_position(sqa, orc, dev):
    """The producer at position p, moved by d, is the producer at p + d but for the two quantizations: each off by at
    most d / 2 (the end opposite the largest value by a whole step), a rotation keeps a pair's 2-norm."""
    r = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn((200, 2, 256), generator=r, device=dev)
    w = torch.ones(256, device=dev)
    rope, idx = sqa.rope_params(*ROPE), torch.arange(200, device=dev)
    pos = torch.arange(500, 700, dtype=torch.int32, device=dev).repeat(4)
    a, b = (torch.zeros((200, 2, 144), dtype=torch.uint8, device=dev) for _ in range(2))
    sqa.rope_norm_set_rows_q4_0(a, x, w, 1e-6, pos, rope, idx)
    sqa.rope_norm_set_rows_q4_0(b, x, w, 1e-6, pos + 321, rope, idx)
    sqa.move_rows_q4_0(a, a, idx, idx, torch.full((800,), 321, dtype=torch.int32, device=dev), rope)
    ka, kb = (sqa.get_rows_q4_0(c, idx).view(-1, 8, 32) for c in (a, b))
    top = kb.abs().amax(-1).view(200, 2, 8)
    # two whole steps of the larger block of a pair after the first quantization and its turn, one of either result
    worst = top[:, :, :2].amax(-1) * 1.5 / 8
    d = (ka - kb).abs().view(200, 2, 8, 32)
    assert (d[:, :, :2].amax((-1, -2)) <= 4 * worst).all()
    assert torch.equal(a.view(200, 2, 8, 18)[:, :, 2:], b.view(200, 2, 8, 18)[:, :, 2:])
    rel = float((ka - kb).norm() / kb.norm())
    assert rel <= 0.15, rel  # a step of 1/8 of the largest of 32 normal values (2.1 sigma), uniform, twice: 0.11


def test_on_another_stream_and_in_a_graph(sqa, orc, dev):
    r = np.random.default_rng(8)
    c = gpu(cache(orc, r, 500, 2), dev)
    idx, to = gpu(r.permutation(500)[:200], dev), gpu(r.permutation(500)[:200], dev)
    delta, rope = torch.full((800,), -99, dtype=torch.int32, device=dev), sqa.rope_params(*ROPE)
    want_dst = torch.zeros_like(c)
    sqa.move_rows_q4_0(want_dst, c, to, idx, delta, rope)
    want = sqa.get_rows_q4_0(want_dst, to)
    s = torch.cuda.Stream()
    for handle in (s, s.cuda_stream):
        dst = torch.zeros_like(c)
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
        sqa.move_rows_q4_0(dst, c, to, idx, delta, rope, stream=handle)
        got = sqa.get_rows_q4_0(dst, to, stream=handle)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(dst, want_dst)
    dst, out = torch.zeros_like(c), torch.empty_like(want)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        sqa.move_rows_q4_0(dst, c, to, idx, delta, rope)
        sqa.get_rows_q4_0(dst, to, out=out)
    for far in (-99, 5000, 0):
        delta.fill_(far)
        dst.zero_(), out.zero_()
        g.replay()
        eager = torch.zeros_like(c)
        sqa.move_rows_q4_0(eager, c, to, idx, delta, rope)
        torch.cuda.synchronize()
        assert torch.equal(dst, eager) and torch.equal(out, sqa.get_rows_q4_0(eager, to))


def test_rows_behind_four_gigabytes(sqa, dev):
    """Offsets of a cache's and a result's bytes pass 32 bits."""
    rows, heads = 16_000_000, 2  # 4.6 GB of cache
    c = torch.zeros((rows, heads, 144), dtype=torch.uint8, device=dev)
    x = torch.randn((3, 512), device=dev)
    at = torch.tensor([rows - 1, 14_913_081, 0], device=dev)
    sqa.set_rows_q4_0(c, x, at)
    want = sqa.get_rows_q4_0(c[:1], torch.zeros(1, dtype=torch.int64, device=dev))
    assert torch.equal(sqa.get_rows_q4_0(c, at)[2:], want)
    small = torch.zeros((3, heads, 144), dtype=torch.uint8, device=dev)
    sqa.set_rows_q4_0(small, x, torch.arange(3, device=dev))
    assert torch.equal(c[at], small)
    n = 2_200_000  # 4.5 GB of float32
    idx = at.repeat(n // 3 + 1)[:n].contiguous()
    got = sqa.get_rows_q4_0(c, idx)
    assert torch.equal(got[-3:], got[:3].roll(-(n % 3), 0)) and torch.equal(got[n // 2 // 3 * 3], got[0])
    sqa.move_rows_q4_0(c, c, at - torch.tensor([5, 5, -5], device=dev), at)
    assert torch.equal(c[rows - 6], c[rows - 1]) and torch.equal(c[5], small[2])
