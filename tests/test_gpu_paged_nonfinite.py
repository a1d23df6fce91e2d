"""A row of q that holds NaN or Inf and sees a key gives NaN in all of its values, whichever kernel
takes it and however its keys are split; one that sees none gives zeros."""
import numpy as np
import pytest
import torch

from test_gpu_paged_attn import Batch, call, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("opt", [{}, {"softcap": 20.0}, {"max_bias": 8.0}, {"softcap": 20.0, "max_bias": 8.0}])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [0, 90, 5000]), ([2, 1, 2], [3000, 0, 70]), ([1, 60, 3], [40, 0, 900]),
                                      ([70, 1, 40], [9000, 2000, 30]), ([600, 1, 1], [2500, 1, 1])])
def test_rows_that_are_not_finite(sqa, orc, dev, new, past, gate, opt):
    b = Batch(orc, 21, new, past, page=32, gate=gate, scale_q=3.0)
    want = b.ref(orc, cap=opt.get("softcap", 0.0), bias=opt.get("max_bias", 0.0))
    last = b.q_start[-1] - 1
    bad = [(0, 0, 7, np.nan), (0, 5, 255, np.inf), (b.q_start[1], 9, 128, np.nan), (last, 15, 31, -np.inf), (last, 2, 32, np.nan),
           (b.q_start[1] - 1, 11, slice(None), np.nan)]
    ok = np.ones(want.shape[:2], dtype=bool)
    for t, h, d, x in bad:
        b.q[t, h, d] = x
        ok[t, h] = False
    got = call(sqa, dev, b, **opt)
    assert np.isnan(got[~ok]).all()
    close(got[ok], want[ok])


@pytest.mark.parametrize("new", [[1, 1], [2, 1], [50, 3]])
def test_rows_that_see_nothing_are_zero(sqa, orc, dev, new):
    b = Batch(orc, 22, new, [30, 600])
    b.kv_len[0] = 0
    b.q[:new[0], 3] = np.nan
    got = call(sqa, dev, b)
    assert not got[:new[0]].any()
    close(got, b.ref(orc))
