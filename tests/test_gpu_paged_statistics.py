"""The weights of a row's splits where its logits are large.

Keys of two kinds with logits of 75.26 and 75.75 in base 2, made of powers of two and few bits so
that the kernels' own operations on them are exact (the scale is the float32 next to ln 2, times
log2 e exactly 1), equal inside a split: what is left is the merge. Weights from differences of two
values of 75 that are kept as they are lose 2^-24 by exp2 and as much by each sum of the merge, some
2e-7 of an output that is a third of its terms; values rounded on their way, by 2^-19 in nats, lose
4e-6 of a weight. 1e-6 is allowed."""
import numpy as np
import pytest

from test_gpu_paged_attn import Batch, call

pytestmark = pytest.mark.gpu

LN2 = float(np.float32(np.log(2.0)))


def kind(dk, code_k, code_v):
    """One head row of K (first value code_k, others 0) and of V (all code_v, scale 1)."""
    k, v = (np.full((8, 18), 0x88, dtype=np.uint8) for _ in range(2))
    k[:, :2], v[:, :2] = (np.array([x], dtype=np.float16).view(np.uint8) for x in (dk, 1.0))
    k[0, 2] = 0x80 | (code_k + 8)
    v[:, 2:] = (code_v + 8) * 17
    return k.reshape(-1), v.reshape(-1)


@pytest.mark.parametrize("new,past", [([1], [8191]), ([1] * 12, [8191] * 12), ([2, 1, 2], [8190] * 3), ([40], [8152]),
                                      ([90, 1, 1], [6000, 8191, 300]), ([560], [4000])])
def test_splits_keep_their_weights(sqa, orc, dev, new, past):
    b = Batch(orc, 1, new, past, page=64)
    for r, kv in enumerate(b.kv_len):
        for j in range(-(-kv // 64)):
            rows = kind(1387 / 1024, 7, 4) if 64 * j < kv // 2 else kind(1396 / 1024, 7, -4)
            b.k[b.table[r, j]], b.v[b.table[r, j]] = rows
    b.q[:] = 0
    b.q[:, :, 0] = 127 / 16
    got, want = call(sqa, dev, b, scale=LN2), b.ref(orc, scale=LN2)
    err = np.linalg.norm(got - want) / np.linalg.norm(want)
    print(f"{err:.2e}")
    assert err <= 1e-6
