"""What a call writes must not be what it reads: refused before any launch (no GPU needed)."""
import ctypes

import pytest


def T(sqa, typ, ne, nb, ptr):
    return sqa.Tensor.make(typ, ne, nb, ptr)


def ref(x):
    return None if x is None else ctypes.byref(x)


M, K, N, R, A = 6, 512, 64, 16, 3
FAR = 1 << 20


def lora(sqa, **moved):
    """A call whose arrays lie 1 MiB apart, but for those given as (address, row step or None)."""
    order = ["base", "x", "gate", "a", "b", "ids", "scale", "dst"]
    width = {"base": N, "x": K, "gate": K, "dst": N}
    t = {}
    for i, k in enumerate(order):
        if k in width:
            at, step = moved.get(k, (FAR * (i + 1), None))
            t[k] = T(sqa, 0, [width[k], M], [4, step or 4 * width[k]], at)
    t["a"] = T(sqa, 1, [K, R, A], [2, 2 * K, 2 * K * R], moved.get("a", (4 * FAR,))[0])
    t["b"] = T(sqa, 1, [R, N, A], [2, 2 * R, 2 * R * N], moved.get("b", (5 * FAR,))[0])
    t["ids"] = T(sqa, 26, [M], [4], moved.get("ids", (6 * FAR,))[0])
    t["scale"] = T(sqa, 0, [A], [4], moved.get("scale", (7 * FAR,))[0])
    return sqa.lib().sqa_lora_add(*[ref(t[k]) for k in order], None)


DST = 8 * FAR  # dst: rows of 256 bytes


@pytest.mark.parametrize("moved", [
    {"x": (DST, None)}, {"x": (DST - 4 * K * M + 16, None)}, {"x": (DST + 4 * N * M - 16, None)}, {"gate": (DST + 64, None)},
    {"base": (DST + 16, None)}, {"base": (DST - 16, None)}, {"base": (DST, 4 * N + 16)}, {"base": (DST + 4 * N * (M - 1), None)},
    {"a": (DST + 4 * N * M - 16,)}, {"a": (DST - 2 * K * R * A + 16,)}, {"b": (DST + 16,)}, {"ids": (DST + 4,)}, {"ids": (DST - 20,)},
    {"scale": (DST + 4 * N * M - 4,)},
    # columns of one buffer of rows of 4096 bytes, 16 bytes too near on either side
    {"dst": (DST, 4096), "x": (DST + 4 * N - 16, 4096)}, {"dst": (DST + 2048 - 16, 4096), "x": (DST, 4096)},
    {"dst": (DST, 4096), "x": (DST + 3 * 4096 + 4 * N - 16, 4096)}, {"dst": (DST, 4096), "base": (DST + 4096 - 16, 4096)},
    {"dst": (DST, 4096), "ids": (DST + 4096 + 4 * N - 4,)},
])
def test_lora_refuses_what_overlaps_dst(sqa, moved):
    assert lora(sqa, **moved) == 1, sqa.last_error()
    assert "overlap" in sqa.last_error()


D, H, HKV, TOK, B, W, PAGE, PAGES = 256, 16, 2, 8, 4, 10, 32, 5
OUT = 64 << 20  # dst: 128 KiB


def attn(sqa, ws=None, ws_bytes=0, token=4 * H * D, head=4 * D, **moved):
    """A call whose arrays lie 1 MiB apart, but for those given; without a workspace one that is all right ends at its size."""
    order = ["q", "k", "v", "table", "q_start", "kv_len", "prefix", "gate", "dst"]
    at = {k: moved.get(k, FAR * (i + 1)) for i, k in enumerate(order)} | {"dst": OUT}
    rows = lambda k, a, b: T(sqa, 0, [D, a[0], b[0]], [4, a[1], b[1]], at[k])  # noqa: E731
    pool = lambda k: T(sqa, 2, [D, HKV, PAGE, PAGES], [18, 144, HKV * 144, 2 * PAGE * HKV * 144], at[k])  # noqa: E731
    ints = lambda k, n: T(sqa, 26, [n], [4], at[k])  # noqa: E731
    t = {"q": rows("q", (TOK, token), (H, head)), "k": pool("k"), "v": pool("v"), "table": T(sqa, 26, [W, B], [4, 64], at["table"]),
         "q_start": ints("q_start", B + 1), "kv_len": ints("kv_len", B), "prefix": ints("prefix", B),
         "gate": rows("gate", (H, head), (TOK, token)), "dst": T(sqa, 0, [D, H, TOK], [4, 4 * D, 4 * H * D], OUT)}
    r = [ref(t[k]) for k in order]
    return sqa.lib().sqa_paged_attn(*r[:7], 1, 0.0625, 0.0, 0.0, r[7], r[8], ws, ws_bytes, None)


SIZE = 4 * H * D * TOK
PAGE_BYTES = PAGE * HKV * 144


@pytest.mark.parametrize("moved", [
    {"q": OUT + 16}, {"q": OUT - SIZE + 4}, {"q": OUT + SIZE - 4}, {"gate": OUT + 4 * D}, {"q": OUT, "token": 4 * H * D + 16},
    {"q": OUT, "token": 4 * D, "head": 4 * D * TOK}, {"k": OUT}, {"v": OUT + SIZE - 16},
    {"k": OUT - 8 * PAGE_BYTES - 2 ** 10 * 4}, {"v": OUT - PAGE_BYTES + 16}, {"table": OUT + 8}, {"table": OUT - 3 * 64 - 36}, {"q_start": OUT - 16},
    {"kv_len": OUT + SIZE - 4}, {"prefix": OUT}, {"ws": OUT + SIZE - 256, "ws_bytes": 1 << 30}, {"ws": OUT - 4096, "ws_bytes": 8192},
    {"ws": FAR + SIZE - 16, "ws_bytes": 4096}, {"ws": 2 * FAR + 8 * PAGE_BYTES, "ws_bytes": 4096}, {"ws": 4 * FAR + 4, "ws_bytes": 64},
    {"ws": 8 * FAR - 32, "ws_bytes": 64},
])
def test_attention_refuses_what_overlaps_what_it_writes(sqa, moved):
    assert attn(sqa, **moved) == 1, sqa.last_error()
    assert "overlap" in sqa.last_error()


@pytest.mark.parametrize("moved", [
    {}, {"q": OUT}, {"gate": OUT}, {"q": OUT, "gate": OUT}, {"q": OUT - SIZE}, {"gate": OUT + SIZE}, {"k": OUT - 9 * PAGE_BYTES},
    {"v": OUT + SIZE}, {"table": OUT - 3 * 64 - 40}, {"q_start": OUT - 20}, {"kv_len": OUT + SIZE},
    {"ws": OUT + SIZE, "ws_bytes": 64}, {"ws": OUT - 64, "ws_bytes": 64},
])
def test_attention_takes_what_lies_beside_it(sqa, moved):
    assert attn(sqa, **moved) == 3, sqa.last_error()  # and refuses the workspace for its size
