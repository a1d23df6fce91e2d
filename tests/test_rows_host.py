"""Refusals of cached rows that are read back or moved, before any launch (no GPU needed)."""
import ctypes

import pytest

D = 256


def T(sqa, typ, ne, nb, ptr=1 << 20):
    return sqa.Tensor.make(typ, ne, nb, ptr)


def ref(x):
    return None if x is None else ctypes.byref(x)


def test_get_rows_refusals(sqa):
    good = {"dst": T(sqa, 0, [512, 9], [4, 2048], 1 << 22), "src": T(sqa, 2, [512, 40], [18, 288], 1 << 20),
            "idx": T(sqa, 27, [9], [8], 1 << 24)}

    def call(**kw):
        a = {**good, **kw}
        t = [ref(a[k]) for k in ("dst", "src", "idx")]
        return sqa.lib().sqa_get_rows_q4_0(*t, None), sqa.lib().sqa_supports_get_rows(*t)

    src = lambda ne0=512, typ=2, nb0=18, nb1=288, ptr=1 << 20: T(sqa, typ, [ne0, 40], [nb0, nb1], ptr)  # noqa: E731
    dst = lambda ne0=512, n=9, typ=0, nb0=4, nb1=2048, ptr=1 << 22: T(sqa, typ, [ne0, n], [nb0, nb1], ptr)  # noqa: E731
    for status, kw in [
        (1, {"dst": None}), (1, {"src": None}), (1, {"idx": None}), (2, {"src": src(typ=1)}), (2, {"dst": dst(typ=2)}),
        (2, {"dst": dst(typ=26)}), (1, {"src": src(ne0=256)}), (1, {"src": src(ne0=500), "dst": dst(ne0=500)}),
        (1, {"dst": dst(n=8)}), (1, {"idx": T(sqa, 26, [9], [4])}), (1, {"idx": T(sqa, 27, [8], [8])}),
        (2, {"idx": T(sqa, 27, [9], [4])}), (2, {"idx": T(sqa, 27, [9], [8], (1 << 24) + 4)}), (1, {"idx": T(sqa, 27, [9], [8], 0)}),
        (1, {"dst": dst(ptr=0)}), (1, {"src": src(ptr=0)}), (2, {"src": src(nb0=20)}), (2, {"src": src(nb1=289)}),
        (2, {"src": src(ptr=(1 << 20) + 1)}), (2, {"dst": dst(nb0=8)}), (2, {"dst": dst(nb1=2050)}),
        (2, {"dst": dst(ptr=(1 << 22) + 2)}), (1, {"dst": dst(nb1=2044)}), (2, {"dst": dst(typ=1, nb0=4)}),
        (1, {"dst": T(sqa, 0, [512, 9, 2], [4, 2048, 1 << 16], 1 << 22)}),
    ]:
        rc, ok = call(**kw)
        assert rc == status and ok == 0 and sqa.last_error(), (kw.keys(), rc, sqa.last_error())
    # overlaps are refused, though the shapes are supported
    for kw in ({"dst": dst(ptr=(1 << 20) + 40 * 288 - 4)}, {"idx": T(sqa, 27, [9], [8], (1 << 22) + 9 * 2048 - 8)},
               {"dst": dst(ptr=(1 << 20) - 9 * 2048 + 4)}):
        assert call(**kw) == (1, 1) and "overlap" in sqa.last_error()


def test_move_rows_refusals(sqa):
    rope = sqa.rope_params(64, (11, 11, 10, 0), 1e7)
    c = lambda ptr, typ=2, d=D, h=2, n=40, nb0=18, nb1=144, nb2=288: T(sqa, typ, [d, h, n], [nb0, nb1, nb2], ptr)  # noqa: E731
    vec = lambda typ, n, ptr, nb=None: T(sqa, typ, [n], [nb or (8 if typ == 27 else 4)], ptr)  # noqa: E731
    good = {"dst": c(1 << 20), "src": c(1 << 21), "to": vec(27, 9, 1 << 22), "from": vec(27, 9, 1 << 23),
            "delta": vec(26, 36, 1 << 24), "rope": rope}

    def call(**kw):
        a = {**good, **kw}
        t = [ref(a[k]) for k in ("dst", "src", "to", "from", "delta", "rope")]
        return sqa.lib().sqa_move_rows_q4_0(*t, None), sqa.lib().sqa_supports_move_rows(*t)

    def turn(*a, **kw):
        return {"rope": sqa.rope_params(*a, **kw)}

    nan, inf = float("nan"), float("inf")
    for status, kw in [
        (1, {"dst": None}), (1, {"src": None}), (1, {"to": None}), (1, {"from": None}), (1, {"delta": None}), (1, {"rope": None}),
        (2, {"dst": c(1 << 20, typ=1)}), (2, {"src": c(1 << 21, typ=0)}), (1, {"src": c(1 << 21, h=3)}), (1, {"src": c(1 << 21, d=128)}),
        (1, {"dst": c(0)}), (1, {"src": c(0)}), (2, {"src": c((1 << 21) + 1)}), (2, {"dst": c(1 << 20, nb2=291)}),
        (2, {"src": c(1 << 21, nb1=160)}), (2, {"src": c(1 << 21, nb0=20)}), (1, {"dst": c(1 << 20, nb2=286)}),
        (1, {"to": vec(26, 9, 1 << 22)}), (1, {"from": vec(27, 8, 1 << 23)}), (2, {"to": vec(27, 9, 1 << 22, 4)}),
        (1, {"to": vec(27, 9, 0)}), (1, {"delta": vec(26, 9, 1 << 24)}), (1, {"delta": vec(27, 36, 1 << 24)}),
        (1, {"delta": vec(26, 36, 1 << 24, 8)}), (1, {"delta": vec(26, 36, (1 << 24) + 2)}),
        (2, turn(60, (11, 11, 10, 0), 1e7)), (2, turn(0, (11, 11, 10, 0), 1e7)), (2, turn(264, (11, 11, 10, 0), 1e7)),
        (1, turn(64, (11, -1, 10, 0), 1e7)), (1, turn(64, (0, 0, 0, 0), 1e7)), (2, turn(64, (11, 11, 10, 0), 1e7, ext_factor=1.0)),
        (1, turn(64, (11, 11, 10, 0), 0.0)), (1, turn(64, (11, 11, 10, 0), nan)), (1, turn(64, (11, 11, 10, 0), 1e7, freq_scale=inf)),
        (2, {"dst": c(1 << 20, d=96, nb1=54, nb2=108), "src": c(1 << 21, d=96, nb1=54, nb2=108)}),
        (1, {"dst": c(1 << 20, d=100), "src": c(1 << 21, d=100)}),
    ]:
        rc, ok = call(**kw)
        assert rc == status and ok == 0 and sqa.last_error(), (kw, rc, sqa.last_error())
    # what dst meets: src in part, to, from, delta
    for kw in ({"src": c((1 << 20) + 288)}, {"src": c((1 << 20) + 40 * 288 - 18)}, {"src": c(1 << 20, nb2=304)},
               {"to": vec(27, 9, (1 << 20) + 8)}, {"from": vec(27, 9, (1 << 20) + 40 * 288 - 8)}, {"delta": vec(26, 36, (1 << 20) - 4)}):
        assert call(**kw) == (1, 1) and "overlap" in sqa.last_error(), kw


def test_no_rows_are_no_work(sqa):
    z = T(sqa, 27, [0], [8], 0)
    assert sqa.lib().sqa_get_rows_q4_0(ref(T(sqa, 0, [512, 0], [4, 2048], 0)), ref(T(sqa, 2, [512, 40], [18, 288])), ref(z), None) == 0
    c = T(sqa, 2, [D, 2, 40], [18, 144, 288])
    assert sqa.lib().sqa_move_rows_q4_0(ref(c), ref(c), ref(z), ref(z), None, None, None) == 0


def test_python_refuses_tensors_off_the_gpu(sqa):
    import torch

    c, i = torch.zeros((4, 2, 144), dtype=torch.uint8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: sqa.get_rows_q4_0(c, i), lambda: sqa.move_rows_q4_0(c, c, i, i)):
        with pytest.raises(sqa.SqaError):
            call()


def test_move_rows_refuses_pairs_that_turn_too_fast(sqa):
    c = [T(sqa, 2, [D, 2, 40], [18, 144, 288], p) for p in (1 << 20, 1 << 21)]
    to, frm = T(sqa, 27, [9], [8], 1 << 22), T(sqa, 27, [9], [8], 1 << 23)
    delta = T(sqa, 26, [36], [4], 1 << 24)
    # radians a position of the fastest pair: base^-(30/32) * scale where base < 1, else scale
    for base, scale, ok in ((1e7, 1.25, 1), (1e7, 1.3, 0), (1e7, -1.25, 1), (1e7, -1.3, 0), (1.0, 1.0, 1), (0.8, 1.0, 1), (0.7, 1.0, 0), (0.7, 0.8, 1)):
        rope = sqa.rope_params(32, (4, 4, 4, 4), base, freq_scale=scale)
        assert sqa.lib().sqa_supports_move_rows(ref(c[0]), ref(c[1]), ref(to), ref(frm), ref(delta), ref(rope)) == ok, (base, scale)
        if not ok:
            assert sqa.lib().sqa_move_rows_q4_0(ref(c[0]), ref(c[1]), ref(to), ref(frm), ref(delta), ref(rope), None) == 2
            assert "radians" in sqa.last_error()


@pytest.mark.parametrize("shape", [(4, 20), (4, 2, 143), (4, 17), (4, 3, 10)])
def test_get_rows_refuses_rows_of_broken_blocks(sqa, shape):
    import torch

    c, i = torch.zeros(shape, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64)
    ne0 = c[0].numel() // 18 * 32
    for kw in ({}, {"out": torch.zeros((2, ne0))}, {"dtype": torch.float16}):
        with pytest.raises(sqa.SqaError, match="whole 18-byte blocks"):
            sqa.get_rows_q4_0(c, i, **kw)
