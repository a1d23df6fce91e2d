"""The merge of many rows (more than 8192, four heads a wavefront) with splits to merge: chunks of a
few splits, and decoding requests of more than the 16 that it takes at a time."""
import pytest

from test_gpu_paged_attn import Batch, call, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("H,Hkv,new,past", [
    (16, 2, [1, 560, 2, 1], [9000, 3000, 5000, 20]),
    (18, 2, [1, 480, 1], [7000, 2600, 40]),   # a last wavefront of two heads
    (28, 4, [320, 1], [2000, 6000]),          # 28 heads: rows of 12 heads in the second workgroup
    (17, 17, [500, 1], [1500, 3000]),     # a KV head each, one head left over
    (64, 16, [150, 1, 1], [1100, 4000, 0]),
])
def test_merge_of_many_rows(sqa, orc, dev, H, Hkv, new, past, gate):
    b = Batch(orc, H + gate, new, past, H, Hkv, 64, pad=3, gate=gate, scale_q=4.0)
    assert b.q.shape[0] * H > 8192
    close(call(sqa, dev, b, fill=7.0), b.ref(orc, fill=7.0))
