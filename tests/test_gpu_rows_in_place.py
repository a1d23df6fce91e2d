"""Cached rows rotated in place, each onto itself, as a context shifts its positions: the bytes that the same move
writes into another cache, whichever blocks of a head its rotation pairs span."""
import numpy as np
import pytest
import torch

from test_gpu_rows import ROPE, cache, check_move, gpu

pytestmark = pytest.mark.gpu


def sections(n_rot):
    return (n_rot // 6, n_rot // 6, n_rot // 2 - 2 * (n_rot // 6), 0)


# rotated blocks a head: 3, 5, 6 and 7, of which the threads of a workgroup hold no whole number, and 2, 4 and 8, of
# which they do; rows of many heads, which alone take several passes, and several rows a workgroup
CASES = [(128, 96, 32, 1), (128, 96, 32, 3), (256, 72, 32, 1), (256, 96, 32, 2), (256, 160, 16, 1), (256, 192, 16, 2),
         (256, 224, 16, 1), (256, 136, 128, 1), (256, 72, 2, 12000), (256, 96, 2, 30000), (128, 80, 8, 4000),
         (128, 96, 8, 4000), (256, 160, 8, 4000), (256, 192, 8, 4000), (256, 224, 8, 4000), (256, 64, 2, 30000),
         (128, 128, 8, 4000), (256, 256, 16, 1001), (64, 64, 4, 20000), (64, 40, 64, 7)]


@pytest.mark.parametrize("common", [True, False])
@pytest.mark.parametrize("D,n_rot,heads,n", CASES)
def test_in_place_is_the_move_between_caches(sqa, orc, dev, D, n_rot, heads, n, common):
    r = np.random.default_rng(n_rot * heads + n)
    c = cache(orc, r, n + 3, heads, D)
    rows = r.permutation(n + 3)[:n]
    if n > 4:
        rows[[1, n // 2, n - 1]] = -1, n + 3, 1 << 40  # skipped
    delta = r.integers(-100000, 100000, (4, 1 if common else n)).astype(np.int32)
    delta = np.ascontiguousarray(np.broadcast_to(delta, (4, n)))
    rope = (n_rot, sections(n_rot), 1e6)
    src, at, d = gpu(c, dev), gpu(rows, dev), gpu(delta.reshape(-1), dev)
    want, got = src.clone(), src.clone()
    sqa.move_rows_q4_0(want, src, at, at, d, sqa.rope_params(*rope))
    assert torch.equal(src, gpu(c, dev))
    sqa.move_rows_q4_0(got, got, at, at, d, sqa.rope_params(*rope))
    assert torch.equal(got, want)
    assert not torch.equal(got, src)
    if n <= 7:
        check_move(orc, c, c, got.cpu().numpy(), rows, rows, delta, rope)


def test_in_place_to_other_rows(sqa, orc, dev):
    """Ranges of one cache that do not meet, and a range that turns where it is, in one call."""
    r = np.random.default_rng(1)
    c = cache(orc, r, 9000, 8, 128)
    frm = np.concatenate([np.arange(3000), np.arange(6000, 9000)])
    to = np.concatenate([np.arange(3000, 6000), np.arange(6000, 9000)])
    mix = r.permutation(6000)
    delta = r.integers(-500, 500, 4 * 6000).astype(np.int32)
    rope = sqa.rope_params(96, sections(96), 1e6)
    src = gpu(c, dev)
    want, got = src.clone(), src.clone()
    args = gpu(to[mix], dev), gpu(frm[mix], dev), gpu(delta, dev), rope
    sqa.move_rows_q4_0(want, src, *args)
    sqa.move_rows_q4_0(got, got, *args)
    assert torch.equal(got, want)


@pytest.mark.parametrize("n_rot", [64, 96, 192])
def test_the_caches_own_move(sqa, orc, dev, n_rot):
    """KvCache.move and PagedKvCache.move of a whole context by one distance: K turned, V as it was."""
    rope = sqa.rope_params(n_rot, sections(n_rot), 1e7)
    gen = torch.Generator(device=dev).manual_seed(n_rot)
    at = torch.randperm(4096, generator=gen, device=dev)[:4000]
    delta = torch.full((16000,), -777, dtype=torch.int32, device=dev)
    one, pool = sqa.KvCache(2, 256, 8, 4096, device=dev), sqa.PagedKvCache(2, 256, 8, 256, 16, 4, 64, device=dev)
    for kv, rows in ((one, lambda w: (one.k if w == "k" else one.v)[1]), (pool, lambda w: pool.rows(1, w))):
        x = torch.randn((4096, 2048), generator=gen, device=dev)
        for w in "kv":
            sqa.set_rows_q4_0(rows(w), x if w == "k" else 2 * x, torch.arange(4096, device=dev))
        k, v = rows("k").clone(), rows("v").clone()
        sqa.move_rows_q4_0(k, rows("k").clone(), at, at, delta, rope)
        kv.move(1, at, at, delta, rope)
        assert torch.equal(rows("k"), k) and torch.equal(rows("v"), v)
