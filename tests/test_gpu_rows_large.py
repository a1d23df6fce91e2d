"""Results of more than 96 MB, which get_rows stores past the caches, and results behind 4 GB."""
import numpy as np
import pytest
import torch

import shared_ref as ref
from test_gpu_rows import cache, gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("n,heads,D", [(110001, 2, 256), (70003, 3, 256), (250007, 1, 256)])
def test_large_results(sqa, orc, dev, dtype, n, heads, D):
    r = np.random.default_rng(n)
    rows = 1009
    c = cache(orc, r, rows, heads, D, scale=2.0)
    idx = r.integers(-20, rows + 20, n)
    ok = (idx >= 0) & (idx < rows)
    got = sqa.get_rows_q4_0(gpu(c, dev), gpu(idx, dev), dtype=dtype)
    assert got.nbytes > 96 << 20
    table = torch.tensor(np.concatenate([ref.values(c.reshape(rows, -1)), np.zeros((1, heads * D))]), device=dev)
    at = gpu(np.where(ok, idx, rows), dev)
    assert torch.equal(got, table.to(dtype)[at])  # every value, rounded once


def test_values_behind_four_gigabytes(sqa, dev):
    """4.5 GB of float32: the values there are those of a call for these rows alone."""
    c = torch.randint(0, 256, (5003, 2, 144), dtype=torch.uint8, device=dev)
    c.view(5003, 16, 18)[..., 1] &= 0x3f  # scales below 2
    n = 2_200_000
    idx = torch.randint(0, 5003, (n,), device=dev)
    got = sqa.get_rows_q4_0(c, idx)
    for lo in (0, n // 2, 2_097_000, n - 1000):  # 4 GB end within the third
        assert torch.equal(got[lo:lo + 1000], sqa.get_rows_q4_0(c, idx[lo:lo + 1000].contiguous()))
