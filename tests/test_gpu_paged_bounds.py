"""Arrays that no plan wrote leave everything outside a call's own buffers as it was."""
import pytest
import torch

pytestmark = pytest.mark.gpu

D, ROW, GUARD = 256, 144, 1 << 20


def call(sqa, dev, n_tok, H, Hkv, q_start, kv_len, max_q, part=1, page=16, held=None):
    """One call between guard bytes behind the workspace and behind out; the guards stay. held: four
    numbers that the workspace is full of."""
    B = len(q_start) - 1
    gen = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn((n_tok, H, D), generator=gen, device=dev)
    pool = torch.randint(0, 60, (2, page, Hkv, ROW), generator=gen, device=dev, dtype=torch.uint8)
    W = max(1, -(-max(max(kv_len), 0) // page))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    table = torch.zeros((B, W), dtype=torch.int32, device=dev)
    size = max(16, sqa.paged_attn_workspace_size(q, pool, table, max_q) // part)
    ws = torch.full((size + GUARD,), 0xA5, dtype=torch.uint8, device=dev)
    if held is not None:
        ws[:size // 16 * 16] = i32(held).repeat(size // 16).view(torch.uint8)
    flat = torch.full((n_tok * H * D + GUARD // 4,), 7.0, device=dev)
    out = flat[:n_tok * H * D].view(n_tok, H, D)
    try:
        sqa.paged_attn(q, pool, pool, table, i32(q_start), i32(kv_len), max_q, out=out, workspace=ws[:size])
    except sqa.SqaError as e:
        assert part > 1 and e.status == 3
    torch.cuda.synchronize()
    assert (ws[size:] == 0xA5).all()
    assert (flat[n_tok * H * D:] == 7).all()
    return out


@pytest.mark.parametrize("part", [1, 3])
@pytest.mark.parametrize("n_tok,H,Hkv,B", [(1, 16, 2, 600), (2, 16, 2, 4096), (1, 600, 600, 12), (1, 16, 1, 40), (3, 4, 4, 300)])
def test_more_requests_with_rows_than_tokens(sqa, dev, n_tok, H, Hkv, B, part):
    """q_start goes to and fro, so that half of the requests have the same rows: more pieces than the workspace holds."""
    call(sqa, dev, n_tok, H, Hkv, [n_tok * (b & 1) for b in range(B + 1)], [5 + b % 90 for b in range(B)], n_tok, part)


@pytest.mark.parametrize("H,Hkv", [(16, 2), (64, 8)])
@pytest.mark.parametrize("held", [[0, 8, 0, 4 << 28 | 2], [0, 256, 0, 4 << 28 | 2], [2 ** 31 - 1, 1, 0, 1], [0, 1, 2 ** 31 - 1, 5]])
def test_tokens_that_no_piece_writes(sqa, dev, H, Hkv, held):
    """The last request's tokens have no piece, so the merge finds what the workspace held: 8 splits of
    2^28 slots between them are no row of it, though 8 * 2^28 is negative in 32 bits."""
    q_start = [b & 1 for b in range(600)] + [3]
    out = call(sqa, dev, 3, H, Hkv, q_start, [9] * 600, 2, held=held)
    assert (out[2] == 7).all()


@pytest.mark.parametrize("n_tok,H,Hkv,B", [(40, 4, 4, 600), (129, 16, 2, 3000), (1 << 24, 1, 1, 4096)])
def test_chunks_whose_ranges_overlap(sqa, dev, n_tok, H, Hkv, B):
    """Half of the requests have all the rows: at 2^24 tokens their query tiles and splits pass 32 bits."""
    call(sqa, dev, n_tok, H, Hkv, [n_tok * (b & 1) for b in range(B + 1)], [3000] * B, n_tok, page=1024)


def test_chunks_whose_ranges_cross(sqa, dev):
    """q_start that does not ascend, of ranges that together have no more tokens than there are."""
    out = call(sqa, dev, 200, 16, 2, [0, 90, 60, 100, 100, 99, 110], [500, 7, 40, 0, 9, 60], 90)
    assert (out[110:] == 7).all() and not (out[:60] == 7).any()
