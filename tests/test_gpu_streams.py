"""The single-sequence calls on a stream other than the current one: a workspace made by the call, freed
at its return, is no memory of the current stream's next tensors while the kernels wait."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, H, HKV, ROW, N_KV = 256, 16, 2, 144, 1024


def busy(stream):
    with torch.cuda.stream(stream):
        torch.cuda._sleep(24_000_000)  # cycles: 10 ms and more


def later(call, size, dev):
    """call(stream) behind a busy stream while the current one fills tensors of the workspace's size."""
    want = call(None).clone()
    s = torch.cuda.Stream()
    for handle in (s, s.cuda_stream):
        torch.cuda.synchronize()
        busy(s)
        got = call(handle)
        others = [torch.full((max(16, size),), 0xFF, dtype=torch.uint8, device=dev) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        assert all((o == 0xFF).all() for o in others)


@pytest.fixture
def cache(sqa, dev):
    gen = torch.Generator(device=dev).manual_seed(6)
    kv = sqa.KvCache(1, D, HKV, N_KV, device=dev)
    kv.zero_caches()
    kv.begin_step(N_KV)
    idx = torch.arange(N_KV, device=dev)
    kv.append(0, *torch.randn((2, N_KV, HKV * D), generator=gen, device=dev), idx)
    return kv, torch.randn((90, H, D), generator=gen, device=dev)


@pytest.mark.parametrize("n", [1, 90])
def test_attention(sqa, dev, cache, n):
    kv, q = cache[0], cache[1][:n]
    size = sqa.flash_attn_workspace_size(q, kv.k[0], N_KV)
    later(lambda s: sqa.flash_attn_ext(q, kv.k[0], kv.v[0], N_KV, stream=s), size, dev)
    later(lambda s: sqa.flash_attn_ext_causal(q, kv.k[0], kv.v[0], N_KV, N_KV - n, stream=s), size, dev)
    later(lambda s: kv.attend(0, q, stream=s), kv.workspace_size(0, q), dev)
    if n == 1:
        later(lambda s: sqa.flash_attn_ext_static(q, kv.k[0], kv.v[0], N_KV, stream=s), size, dev)


@pytest.mark.parametrize("m", [1, 90])
def test_projection_and_gate(sqa, dev, cache, m):
    gen = torch.Generator(device=dev).manual_seed(7)
    K, N = H * D, 256
    w = torch.randint(0, 256, (N, K // 256, 144), generator=gen, device=dev, dtype=torch.uint8)
    w[:, :, :4] = torch.full((N, K // 256, 2), 3e-4, device=dev).half().view(torch.uint8)
    w, x = w.reshape(N, -1), cache[1][:m].reshape(m, K)
    later(lambda s: sqa.out_proj(w, x, stream=s), sqa.out_proj_workspace_size(w, x), dev)
    later(lambda s: sqa.sigmoid_mul(x, x, stream=s), 4 * m * K, dev)
