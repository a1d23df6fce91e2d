"""paged_attn at the ends of its range."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, ROW = 256, 144


def test_long_requests_that_share_a_page_in_the_smallest_workspace(sqa, dev):
    """1024 requests of 2^26 keys, all on one page: 2^28 tiles for the one piece beside them. Every key
    of the page has the same share as in a request of the page alone.

    The sum S of a value over the pages has 2048 additions of 32 keys a page. In a binade of S all its
    values are multiples of one ulp u, at most 2^-23 S, so a page's additions are rounded the same way
    each time and their errors, u / sqrt(12) each, add up over its pages: sqrt(2048) u / sqrt(12) a
    page, times the 512 pages of the last binade and a quarter as much for each one before. That is
    683 * 45 * 2^-23.5 / 3.46 = 7.5e-4 of S (u is 2^-23.5 S between its ends). Four times that is allowed."""
    B, page, W = 1024, 65536, 1024
    gen = torch.Generator(device=dev).manual_seed(1)
    src = torch.randn((2, page, D), generator=gen, device=dev)
    pools = [torch.empty((1, page, 1, ROW), dtype=torch.uint8, device=dev) for _ in range(2)]
    for p, x in zip(pools, src):
        sqa.set_rows_q4_0(p.view(page, 1, ROW), x, torch.arange(page, device=dev))
    q = torch.randn((B, 1, D), generator=gen, device=dev)
    table = torch.zeros((B, W), dtype=torch.int32, device=dev)
    start = torch.arange(B + 1, dtype=torch.int32, device=dev)
    least = 16 * B + (1 + B) * 8 * (D + 2) * 4 + 512  # a slot of 8 rows for every request and one more
    ws = torch.empty(least, dtype=torch.uint8, device=dev)
    out = [torch.full((B, 1, D), 7.0, device=dev) for _ in range(2)]
    for kv, o in zip((page, W * page), out):
        sqa.paged_attn(q, *pools, table, start, torch.full((B,), kv, dtype=torch.int32, device=dev), 1, out=o, workspace=ws)
    torch.cuda.synchronize()
    assert float((out[1] - out[0]).norm() / out[0].norm()) <= 3e-3


@pytest.mark.parametrize("new,past", [([1, 2], [0, 300]), ([60, 1], [90, 700])])
@pytest.mark.parametrize("cap", [1e-45, 1e-40, 1e-30, 1e30, 2.3e38, 2.5e38, 3.4e38])
def test_caps_of_any_size(sqa, orc, dev, new, past, cap):
    """A cap far below the logits leaves equal weights, one far above them leaves them as they are."""
    from test_gpu_paged_attn import Batch, call, close

    b = Batch(orc, 5, new, past, page=32, scale_q=3.0)
    b.q[-1, :3] = 0  # logits of 0 exactly
    close(call(sqa, dev, b, softcap=cap), b.ref(orc, cap=float(torch.tensor(cap, dtype=torch.float32))))
