"""Results that lie among a call's inputs without meeting them are right."""
import pytest
import torch

import paged_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 5, 100, 700])
def test_lora_columns_of_one_buffer(sqa, dev, M):
    """x, base, out and gate side by side in one row; ids between two rows of out; base as out."""
    K, N, r, n = 512, 64, 16, 3
    gen = torch.Generator(device=dev).manual_seed(M)
    wide = torch.randn((M, 2 * K + 3 * N), generator=gen, device=dev)
    x, gate = wide[:, :K], wide[:, K + 2 * N:2 * K + 2 * N]
    base, out = wide[:, K:K + N], wide[:, K + N:K + 2 * N]
    a = (torch.randn((n, r, K), generator=gen, device=dev) / 16).half()
    b = torch.randn((n, N, r), generator=gen, device=dev).half()
    ids = torch.randint(-1, n, (M,), generator=gen, device=dev, dtype=torch.int32)
    last = wide[0, 2 * K + 2 * N:].view(torch.int32)[:min(M, N)]  # behind the first row's out
    if M <= N:
        last.copy_(ids)
        ids = last
    before = wide.clone()
    want = paged_ref.lora(base=base, x=x, gate=gate, a=a, b=b, ids=ids, scale=None)
    sqa.lora_add(base, x, a, b, ids, gate=gate, out=out)
    assert float((out.double().cpu() - want).norm() / want.norm()) <= 1e-5
    before[:, K + N:K + 2 * N] = out
    assert torch.equal(wide, before)
    sqa.lora_add(base, x, a, b, ids, gate=gate, out=base)
    assert torch.equal(base, out)
