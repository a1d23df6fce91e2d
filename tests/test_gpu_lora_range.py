"""Adapters of values past fp16's range, in the form for few tokens and in tiles: every row as close
to float64 as rows of ordinary size are (1e-5 of the row; see test_gpu_lora for that)."""
import pytest
import torch

import paged_ref
from test_gpu_lora import inputs

pytestmark = pytest.mark.gpu


def rows_close(got, want):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    rel = (got - want).norm(dim=1) / want.norm(dim=1)
    print(f"rel {float(rel.max()):.2e}")
    assert float(rel.max()) <= 1e-5


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("M,K,N,r", [(40, 512, 64, 16), (520, 256, 64, 16), (600, 1024, 144, 24), (700, 512, 80, 64), (515, 768, 48, 128),
                                     (30, 16640, 64, 16)])
def test_lora_large_values(sqa, dev, M, K, N, r, gate):
    """Rows of x of 1, 1e5, 1e10 and 1e30 in every tile, single large values, and A x too large where x is not."""
    d = inputs(dev, M + r, M, K, N, r, 3, gate=gate)
    size = torch.tensor([1.0, 1e5, 1.0, 1e10, 1.0, 1e30, 3e4], device=dev)[torch.arange(M, device=dev) % 7]
    d["x"] *= size[:, None]
    d["x"][::5, 3] = 7e4
    d["a"] *= 8
    d["base"] *= size[:, None]
    out = torch.empty_like(d["base"])
    sqa.lora_add(**d, out=out)
    rows_close(out, paged_ref.lora(**d))


def test_lora_large_scales(sqa, dev):
    """scale A x past 65504 by the scale alone."""
    d = inputs(dev, 5, 530, 256, 32, 8, 3)
    d["scale"] = torch.tensor([1e6, 1.0, 1e20], device=dev)
    rows_close(sqa.lora_add(**d), paged_ref.lora(**d))


@pytest.mark.parametrize("M", [20, 600])
def test_lora_values_that_are_not_finite_stay_alone(sqa, dev, M):
    """NaN and Inf in x spoil their own token, among large and ordinary ones, if it has an adapter."""
    d = inputs(dev, 6, M, 512, 64, 16, 3, gate=True, ids=[m % 3 - (m % 4 == 0) for m in range(M)])
    d["x"][3::7] *= 1e6
    x = d["x"].clone()
    d["x"][2::9, 5] = float("nan")
    d["x"][5::9, 400] = float("inf")
    bad = torch.zeros(M, dtype=torch.bool, device=dev)
    bad[2::9] = bad[5::9] = True
    bad &= d["ids"] >= 0
    got, want = sqa.lora_add(**d), paged_ref.lora(**dict(d, x=x))
    assert not torch.isfinite(got[bad]).any()
    rows_close(got[~bad], want[~bad.cpu()])
