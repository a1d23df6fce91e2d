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


@pytest.mark.parametrize("new", [[1, 2, 1], [1, 150, 30], [700, 1, 1]])
@pytest.mark.parametrize("place", ["q", "gate", "both"])
def test_attention_in_place(sqa, dev, new, place):
    D, H, Hkv, page = 256, 16, 2, 64
    gen = torch.Generator(device=dev).manual_seed(2)
    lens = [n + p for n, p in zip(new, (2000, 90, 300))]
    used = [-(-n // page) for n in lens]
    pools = [torch.empty((sum(used), page, Hkv, 144), dtype=torch.uint8, device=dev) for _ in range(2)]
    for p in pools:
        sqa.set_rows_q4_0(p.view(-1, Hkv, 144), torch.randn((sum(used) * page, Hkv * D), generator=gen, device=dev),
                          torch.arange(sum(used) * page, device=dev))
    table = torch.full((3, max(used)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(at, at + n, device=dev)
        at += n
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    rest = (*pools, table, i32([0, new[0], new[0] + new[1], sum(new)]), i32(lens), max(new))
    q = torch.randn((sum(new), H, D), generator=gen, device=dev)
    gate = q if place == "both" else torch.randn(q.shape, generator=gen, device=dev)
    want = sqa.paged_attn(q, *rest, gate=gate)
    out = gate if place == "gate" else q
    assert sqa.paged_attn(q, *rest, gate=gate, out=out) is out
    assert torch.equal(out, want)
