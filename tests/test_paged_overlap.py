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
