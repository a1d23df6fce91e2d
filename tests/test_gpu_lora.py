"""Adapters of a batch against float64.

Tolerance: x, A x and their products keep 22 bits or fp32's 24 and are summed in
fp32 over K <= 4096 and r <= 128 terms in at least 8 separate sums: 2^-22 from the
operands and, of n terms of random sign, sqrt(n) roundings of 2^-24, 3.8e-6 of the
adapter's part; that part is about as large as the base here."""
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu

REL = 1e-5


def inputs(dev, seed, M, K, N, r, n, gate=False, ids=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    d = {"base": randn(M, N), "x": randn(M, K), "a": (randn(n, r, K) * K ** -0.5).half(), "b": (randn(n, N, r) * r ** -0.5).half(),
         "ids": torch.randint(-1, n + 1, (M,), generator=g, device=dev, dtype=torch.int32) if ids is None
         else torch.tensor(ids, dtype=torch.int32, device=dev),
         "scale": torch.rand(n, generator=g, device=dev) + 0.5, "gate": randn(M, K) if gate else None}
    return d


def close(got, want):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    rel = float((got - want).norm() / want.norm())
    print(f"rel {rel:.2e}")
    assert rel <= REL


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 100])
@pytest.mark.parametrize("K,N,r", [(256, 16, 8), (1024, 2048, 16), (4096, 2048, 16), (512, 80, 24), (2048, 1040, 64), (768, 32, 128),
                                   (256, 48, 40)])
def test_lora(sqa, dev, M, K, N, r):
    for seed, n in ((0, 3), (1, 40)):
        d = inputs(dev, M + seed, M, K, N, r, n, gate=seed == 1)
        out = torch.empty_like(d["base"])
        sqa.lora_add(**d, out=out)
        close(out, paged_ref.lora(**d))


@pytest.mark.parametrize("M", [64, 300, 1200])
@pytest.mark.parametrize("K,N,r", [(1024, 256, 16), (512, 512, 64), (256, 144, 8), (512, 64, 128)])
def test_lora_groups(sqa, dev, M, K, N, r):
    """Neighbours share an adapter, some groups have none, groups end inside any tile."""
    ids, i = [], 0
    while len(ids) < M:
        ids += [i % 5 - 1] * (37 + 13 * (i % 4))
        i += 1
    d = inputs(dev, M, M, K, N, r, 4, gate=True, ids=ids[:M])
    out = torch.empty_like(d["base"])
    sqa.lora_add(**d, out=out)
    close(out, paged_ref.lora(**d))
    d["ids"].fill_(-1)
    sqa.lora_add(**d, out=out)
    assert torch.equal(out, d["base"])


@pytest.mark.parametrize("M", [3, 70, 600])
def test_lora_in_place_strides_paths(sqa, dev, M):
    K, N, r = 512, 96, 16
    d = inputs(dev, 2, M, K, N, r, 6, gate=True)
    want = paged_ref.lora(**d)
    first = sqa.lora_add(**d)
    close(first, want)
    assert torch.equal(sqa.lora_add(**d), first)
    assert torch.equal(sqa.lora_add(**d, out=torch.empty_like(first)), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = sqa.lora_add(**d, out=torch.empty_like(first))
    torch.cuda.synchronize()
    assert torch.equal(other, first)
    into = d["base"].clone()
    sqa.lora_add(into, d["x"], d["a"], d["b"], d["ids"], scale=d["scale"], gate=d["gate"], out=into)
    assert torch.equal(into, first)
    wide = {k: torch.zeros((M, K + 11), device=dev) for k in ("x", "gate")}
    for k in wide:
        wide[k][:, 5:5 + K] = d[k]
    rows = {k: torch.full((M, N + 8), 3.0, device=dev) for k in ("base", "out")}
    rows["base"][:, 4:4 + N] = d["base"]
    sqa.lora_add(rows["base"][:, 4:4 + N], wide["x"][:, 5:5 + K], d["a"], d["b"], d["ids"], scale=d["scale"],
                 gate=wide["gate"][:, 5:5 + K], out=rows["out"][:, 4:4 + N])
    close(rows["out"][:, 4:4 + N], want)
    assert (rows["out"][:, :4] == 3).all() and (rows["out"][:, 4 + N:] == 3).all()
    no = dict(d, scale=None)
    close(sqa.lora_add(**no), paged_ref.lora(**no))


def test_lora_of_no_tokens(sqa, dev):
    d = inputs(dev, 2, 0, 256, 32, 8, 2)
    assert sqa.lora_add(**d).shape == (0, 32)


def test_lora_ids_out_of_range(sqa, dev):
    d = inputs(dev, 1, 6, 256, 32, 8, 2, ids=[2, -1, 2 ** 31 - 1, -2 ** 31, 1, 0])
    out = sqa.lora_add(**d)
    assert torch.equal(out[:4], d["base"][:4])
    close(out, paged_ref.lora(**d))


def test_lora_unused_adapters_hold_anything(sqa, dev):
    """NaN in adapters of other tokens, and in x of tokens without one, enters nothing."""
    for M in (5, 90, 700):
        ids = [(m // 9) % 4 - 1 for m in range(M)]
        d = inputs(dev, 3, M, 512, 64, 16, 4, ids=ids)
        want = paged_ref.lora(**d)
        d["a"][3], d["b"][3], d["scale"][3] = float("nan"), float("inf"), float("nan")
        d["x"][d["ids"] < 0] = float("nan")
        close(sqa.lora_add(**d), want)


@pytest.mark.parametrize("M", [1, 5, 40, 130])
@pytest.mark.parametrize("K,N,r", [(1280, 64, 120), (2304, 208, 8), (4352, 64, 32), (5120, 2048, 64), (12288, 80, 56),
                                   (16384, 16, 128), (16640, 64, 16)])
def test_lora_widths(sqa, dev, M, K, N, r):
    """Numbers of runs of K and of ranks that leave wavefronts and lanes without work, and K past
    what the form for few tokens keeps (sums of up to 16640 terms, 2e-8 more than above)."""
    d = inputs(dev, M + K, M, K, N, r, 5, gate=K % 512 == 0)
    out = torch.empty_like(d["base"])
    sqa.lora_add(**d, out=out)
    close(out, paged_ref.lora(**d))


@pytest.mark.parametrize("M", [513, 530, 1037])
@pytest.mark.parametrize("K,N,r", [(256, 16, 8), (512, 80, 24), (4096, 2048, 64), (768, 32, 128), (256, 48, 40), (1280, 144, 120)])
def test_lora_tiles(sqa, dev, M, K, N, r):
    """Tiles whose tokens have one adapter each, or share a few."""
    for seed, n in ((0, 3), (1, 40)):
        d = inputs(dev, M + seed, M, K, N, r, n, gate=seed == 1)
        out = torch.empty_like(d["base"])
        sqa.lora_add(**d, out=out)
        close(out, paged_ref.lora(**d))


@pytest.mark.parametrize("M", [40, 600])
def test_lora_gated_values_keep_their_bits(sqa, dev, M):
    """x sigmoid(gate) and A x at 22 bits or more (2^-22 each, uniform) and sums of some 40
    roundings of 2^-24: below 1e-6 of the adapter's part, here the whole output."""
    d = inputs(dev, 9, M, 4096, 512, 64, 2, gate=True, ids=[m % 2 for m in range(M)])
    d["base"].zero_()
    got, want = sqa.lora_add(**d).double().cpu(), paged_ref.lora(**d)
    assert float((got - want).norm() / want.norm()) <= 1e-6
