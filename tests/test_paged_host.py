"""Refusals of the operators over a paged pool, before any launch (no GPU needed)."""
import ctypes

import pytest

D = 256


def T(sqa, typ, ne, nb, ptr=4096):
    return sqa.Tensor.make(typ, ne, nb, ptr)


def ivec(sqa, n, ptr=4096, typ=26):
    return T(sqa, typ, [n], [8 if typ == 27 else 4], ptr)


def ref(x):
    return None if x is None else ctypes.byref(x)


def attn(sqa, **kw):
    H, Hkv, n_tok, B, W, page, n_pages = 16, 2, 8, 4, 10, 32, 64
    g = kw.get
    H, Hkv, page = g("H", H), g("Hkv", Hkv), g("page", page)
    rb = 144
    a = {"q": T(sqa, 0, [D, n_tok, H], [4, H * D * 4, D * 4]),
         "k": T(sqa, 2, [D, Hkv, page, n_pages], [18, rb, Hkv * rb, page * Hkv * rb]),
         "table": T(sqa, 26, [W, B], [4, W * 4]), "q_start": ivec(sqa, B + 1), "kv_len": ivec(sqa, B), "prefix": None,
         "max_q": 1, "scale": 0.0625, "bias": 0.0, "cap": 0.0, "gate": None,
         "dst": T(sqa, 0, [D, H, n_tok], [4, D * 4, H * D * 4])}
    a["v"] = a["k"]
    a.update({k: v for k, v in kw.items() if k in a})
    rc = sqa.lib().sqa_paged_attn(ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["table"]), ref(a["q_start"]), ref(a["kv_len"]),
                                  ref(a["prefix"]), a["max_q"], a["scale"], a["bias"], a["cap"], ref(a["gate"]), ref(a["dst"]),
                                  None, 0, None)
    ok = sqa.lib().sqa_supports_paged_attn(ref(a["q"]), ref(a["k"]), ref(a["v"]), ref(a["table"]), a["max_q"], a["scale"],
                                           a["bias"], a["cap"], ref(a["dst"]))
    return rc, ok


def test_paged_attn_refusals(sqa):
    inf, nan = float("inf"), float("nan")
    pool = lambda page=32, n=64, typ=2, nb3=None, Hkv=2, ptr=4096, d=D: T(  # noqa: E731
        sqa, typ, [d, Hkv, page, n], [18, 144, Hkv * 144, nb3 or page * Hkv * 144], ptr)
    q = lambda typ=0, nt=8, H=16, nb0=4, nb1=16 * D * 4: T(sqa, typ, [D, nt, H], [nb0, nb1, D * 4])  # noqa: E731
    dst = lambda ptr=4096, nb1=D * 4, typ=0: T(sqa, typ, [D, 16, 8], [4, nb1, 16 * D * 4], ptr)  # noqa: E731
    both = lambda p: {"k": p, "v": p}  # noqa: E731
    for status, kw in [
        (1, {"q": None}), (1, {"k": None}), (1, {"table": None}), (1, {"q_start": None}), (1, {"dst": None}),
        (2, {"q": q(typ=1)}), (2, both(pool(typ=1))), (1, {"v": pool(n=63)}), (1, both(pool(d=128))),
        (2, both(pool(page=8))), (2, both(pool(page=48))), (2, both(pool(nb3=32 * 288 - 16))), (2, both(pool(nb3=32 * 288 + 8))),
        (2, both(pool(ptr=4104))), (1, both(pool(n=0))), (1, both(pool(Hkv=3))),
        (2, {"q": q(H=32), "dst": T(sqa, 0, [D, 32, 8], [4, D * 4, 32 * D * 4]), **both(pool(Hkv=1))}),
        (2, {"q": q(nb0=8)}), (2, {"q": q(nb1=6)}), (1, {"dst": T(sqa, 0, [D, 16, 9], [4, D * 4, 16 * D * 4])}),
        (2, {"dst": dst(ptr=4100)}), (2, {"dst": dst(nb1=D * 4 + 16)}), (2, {"dst": dst(typ=1)}),
        (1, {"table": T(sqa, 27, [10, 4], [8, 80])}), (2, {"table": T(sqa, 26, [10, 5000], [4, 40])}),
        (2, {"table": T(sqa, 26, [10, 4], [8, 80])}), (2, {"table": T(sqa, 26, [1 << 19, 4], [4, 4 << 19])}),
        (1, {"q_start": ivec(sqa, 4)}), (1, {"kv_len": ivec(sqa, 5)}), (1, {"kv_len": ivec(sqa, 4, typ=27)}),
        (1, {"prefix": ivec(sqa, 3)}), (1, {"kv_len": T(sqa, 26, [4], [8])}),
        (6, {"max_q": 0}), (1, {"scale": nan}), (1, {"scale": inf}), (1, {"bias": -1.0}), (1, {"bias": inf}),
        (1, {"cap": -2.0}), (1, {"cap": nan}),
        (1, {"gate": T(sqa, 0, [D, 16, 7], [4, D * 4, 16 * D * 4])}), (1, {"gate": T(sqa, 1, [D, 16, 8], [2, D * 2, 16 * D * 2])}),
    ]:
        rc, ok = attn(sqa, **kw)
        assert rc == status, (kw.keys(), rc, sqa.last_error())
        assert ok == 0 or set(kw) & {"q_start", "kv_len", "prefix", "gate"}
        assert sqa.last_error()


def test_paged_attn_of_no_tokens_is_no_work(sqa):
    rc, ok = attn(sqa, q=T(sqa, 0, [D, 0, 16], [4, 16 * D * 4, D * 4], 0), dst=T(sqa, 0, [D, 16, 0], [4, D * 4, 16 * D * 4], 0))
    assert rc == 0 and ok == 1


def test_paged_plan_refusals(sqa):
    B, W, n, T_ = 4, 10, 64, 20
    names = ["n_past", "n_new", "table", "ring", "state", "state_out", "n_past_out", "q_start", "kv_len", "slots", "pos"]
    good = {k: ivec(sqa, c, 4096 * (i + 1)) for i, (k, c) in enumerate(
        {"n_past": B, "n_new": B, "ring": n, "state": 4, "state_out": 4, "n_past_out": B, "q_start": B + 1, "kv_len": B}.items())}
    good |= {"table": T(sqa, 26, [W, B], [4, W * 4], 1 << 20), "slots": ivec(sqa, T_, 1 << 21, 27), "pos": ivec(sqa, 4 * T_, 1 << 22)}

    def call(page=16, **kw):
        a = {**good, **kw}
        t = [ref(a[k]) for k in names]
        return sqa.lib().sqa_paged_plan(*t[:5], page, *t[5:], None)

    for status, kw in [(1, {k: None}) for k in names] + [
        (2, {"page": 8}), (2, {"page": 0}), (2, {"page": 24}), (2, {"page": 1 << 17}), (2, {"page": -16}),
        (1, {"n_past": ivec(sqa, 3)}), (1, {"n_new": ivec(sqa, 5)}), (1, {"state": ivec(sqa, 3)}), (1, {"pos": ivec(sqa, T_)}),
        (1, {"slots": ivec(sqa, T_)}), (1, {"ring": ivec(sqa, 0)}), (1, {"q_start": ivec(sqa, B)}),
        (1, {"n_past": T(sqa, 26, [B], [8])}), (1, {"n_past": ivec(sqa, B, 0)}), (1, {"kv_len": ivec(sqa, B, 4098)}),
        (1, {"state_out": ivec(sqa, 4, good["state"].data + 8)}), (1, {"n_past_out": ivec(sqa, B, good["n_past"].data)}),
        (2, {"table": T(sqa, 26, [1 << 18, B], [4, 4 << 18]), "page": 1 << 14}),
        (1, {"table": T(sqa, 26, [W, B], [4, 0], 1 << 20)}), (1, {"table": T(sqa, 26, [W, B], [4, W * 4 - 4], 1 << 20)}),
    ]:
        assert call(**kw) == status, (kw, sqa.last_error())


@pytest.mark.parametrize("a,b", [("kv_len", "n_past"), ("n_past_out", "n_new"), ("q_start", "kv_len"), ("slots", "table"),
                                 ("ring", "table"), ("pos", "slots"), ("state_out", "ring"), ("table", "n_new")])
def test_paged_plan_refuses_arrays_that_overlap_what_it_writes(sqa, a, b):
    size = {"n_past": 4, "n_new": 4, "state": 4, "state_out": 4, "n_past_out": 4, "q_start": 5, "kv_len": 4, "ring": 64,
            "pos": 80, "slots": 20}
    names = ["n_past", "n_new", "table", "ring", "state", "state_out", "n_past_out", "q_start", "kv_len", "slots", "pos"]
    t = {k: T(sqa, 26, [10, 4], [4, 48], 4096 * (i + 1)) if k == "table" else ivec(sqa, size[k], 4096 * (i + 1), 27 if k == "slots" else 26)
         for i, k in enumerate(names)}
    end = t[b].data + (3 * 48 + 40 if b == "table" else size[b] * (8 if b == "slots" else 4))
    t[a].data = end - 8
    args = [ref(t[k]) for k in names]
    assert sqa.lib().sqa_paged_plan(*args[:5], 16, *args[5:], None) == 1, sqa.last_error()
    assert "overlap" in sqa.last_error()


def test_lora_refusals(sqa):
    M, K, N, r, n = 6, 512, 64, 16, 3
    f = lambda ne0, ne1, typ=0, nb0=4, pad=0, ptr=4096: T(sqa, typ, [ne0, ne1], [nb0, 4 * (ne0 + pad)], ptr)  # noqa: E731
    h = lambda a, b, c, ptr=4096, typ=1: T(sqa, typ, [a, b, c], [2, 2 * a, 2 * a * b], ptr)  # noqa: E731
    good = {"base": f(N, M), "x": f(K, M), "gate": f(K, M), "a": h(K, r, n), "b": h(r, N, n), "ids": ivec(sqa, M),
            "scale": T(sqa, 0, [n], [4]), "dst": f(N, M)}

    def call(**kw):
        return sqa.lib().sqa_lora_add(*[ref(v) for v in {**good, **kw}.values()], None)

    for status, kw in [(1, {k: None}) for k in ("base", "x", "a", "b", "ids", "dst")] + [
        (1, {"x": f(K, M, typ=1)}), (2, {"a": h(K, r, n, typ=0)}), (1, {"a": h(256, r, n)}), (1, {"b": h(8, N, n)}),
        (1, {"b": h(r, N, 2)}), (2, {"a": h(K, r, n, ptr=4104)}), (2, {"b": h(r, N, n, ptr=4098)}),
        (2, {"x": f(K, M, nb0=8)}), (1, {"gate": f(K, M + 1)}), (1, {"base": f(N, M + 1)}), (2, {"dst": f(N, M, pad=1)}),
        (2, {"dst": f(N, M, ptr=4100)}), (1, {"ids": ivec(sqa, M - 1)}), (1, {"ids": ivec(sqa, M, typ=27)}),
        (1, {"scale": T(sqa, 0, [n - 1], [4])}), (1, {"x": f(K, M, ptr=0)}),
        (2, {"x": f(300, M), "gate": None, "a": h(300, r, n)}), (2, {"a": h(K, 12, n), "b": h(12, N, n)}),
        (2, {"a": h(K, 136, n), "b": h(136, N, n)}), (2, {"b": h(r, 40, n), "base": f(40, M), "dst": f(40, M)}),
        (1, {"dst": T(sqa, 0, [N, M], [4, 4 * N - 16])}),
    ]:
        assert call(**kw) == status, (kw.keys(), sqa.last_error())
    assert call(x=f(K, 0), gate=None, ids=ivec(sqa, 0), base=f(N, 0), dst=f(N, 0)) == 0


def test_wrappers_refuse_tensors_off_the_gpu(sqa):
    import torch

    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(sqa.SqaError):
        sqa.paged_plan(i, i, i.view(4, 1), i, i, 16, torch.zeros(3, dtype=torch.int64))
    x = torch.zeros((2, 512))
    with pytest.raises(sqa.SqaError):
        sqa.lora_add(x[:, :64], x, torch.zeros((1, 8, 512)).half(), torch.zeros((1, 64, 8)).half(), i[:2])
    with pytest.raises(sqa.SqaError):
        sqa.paged_attn(torch.zeros((1, 16, 256)), torch.zeros((1, 16, 2, 144), dtype=torch.uint8),
                       torch.zeros((1, 16, 2, 144), dtype=torch.uint8), i.view(1, 4), i[:2], i[:1], 1)
