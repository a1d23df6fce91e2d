"""Refusals of the operators of shared prefixes, before any launch (no GPU needed)."""
import ctypes

import pytest

from test_paged_host import D, T, ivec, ref

SHARE = ["q_start", "kv_len", "group", "shared_len", "members", "m_start", "m_pos", "token_group", "pos"]
SIZE = {"q_start": 5, "kv_len": 4, "group": 4, "shared_len": 3, "members": 20, "m_start": 4, "m_pos": 20, "token_group": 20, "pos": 80}


def share(sqa, **kw):
    a = {k: ivec(sqa, SIZE[k], 4096 * (i + 1)) for i, k in enumerate(SHARE)} | kw
    return sqa.lib().sqa_paged_share(*[ref(a[k]) for k in SHARE], None)


def test_paged_share_refusals(sqa):
    for status, kw in [(1, {k: None}) for k in SHARE[:-1]] + [(1, {k: ivec(sqa, SIZE[k] - 1, 1 << 20)}) for k in SHARE] + [
        (1, {k: ivec(sqa, SIZE[k], 1 << 20, 27)}) for k in SHARE] + [(1, {k: T(sqa, 26, [SIZE[k]], [8], 1 << 20)}) for k in SHARE] + [
        (1, {k: ivec(sqa, SIZE[k], 0)}) for k in SHARE] + [(1, {k: ivec(sqa, SIZE[k], (1 << 20) + 2)}) for k in SHARE] + [
        (2, {"kv_len": ivec(sqa, 4097, 1 << 20), "group": ivec(sqa, 4097, 1 << 21), "q_start": ivec(sqa, 4098, 1 << 22)}),
        (2, {"shared_len": ivec(sqa, 4097, 1 << 20), "m_start": ivec(sqa, 4098, 1 << 21)}),
        (1, {"kv_len": ivec(sqa, 0, 1 << 20)}), (1, {"shared_len": ivec(sqa, 0, 1 << 20)}),
        (2, {"members": ivec(sqa, (1 << 24) + 1, 1 << 32)}),
    ]:
        if status == 1 and kw.get("members") is not None and kw["members"].ne[0] == 19:
            continue  # T itself: the others then differ from it, which their own entries show
        assert share(sqa, **kw) == status, (kw, sqa.last_error())
    assert share(sqa, members=ivec(sqa, 19, 1 << 20)) == 1


@pytest.mark.parametrize("a", SHARE[4:])
@pytest.mark.parametrize("b", SHARE)
def test_paged_share_refuses_overlaps(sqa, a, b):
    if a == b:
        return
    at = 4096 * (SHARE.index(b) + 1) + 4 * SIZE[b]
    assert share(sqa, **{a: ivec(sqa, SIZE[a], at - 4)}) == 1 and "overlap" in sqa.last_error()


def attn(sqa, **kw):
    H, Hkv, n_tok, B, W, G, page, n_pages = 16, 2, 8, 4, 10, 3, 32, 64
    pool = lambda ptr: T(sqa, 2, [D, Hkv, page, n_pages], [18, 144, Hkv * 144, page * Hkv * 144], ptr)  # noqa: E731
    a = {"q": T(sqa, 0, [D, n_tok, H], [4, H * D * 4, D * 4], 1 << 20), "k": pool(1 << 21), "v": pool(1 << 22),
         "table": T(sqa, 26, [W, B], [4, W * 4], 1 << 23), "q_start": ivec(sqa, B + 1, 4096), "kv_len": ivec(sqa, B, 8192), "prefix": None,
         "shared_table": T(sqa, 26, [W, G], [4, W * 4], 1 << 24), "shared_len": ivec(sqa, G, 12288), "members": ivec(sqa, n_tok, 16384),
         "m_start": ivec(sqa, G + 1, 20480), "m_pos": ivec(sqa, n_tok, 24576), "token_group": ivec(sqa, n_tok, 28672), "max_q": 1,
         "scale": 0.0625, "bias": 0.0, "cap": 0.0, "gate": None, "dst": T(sqa, 0, [D, H, n_tok], [4, D * 4, H * D * 4], 1 << 25),
         "ws": None, "ws_bytes": 0}
    a.update(kw)
    names = ["q", "k", "v", "table", "q_start", "kv_len", "prefix", "shared_table", "shared_len", "members", "m_start", "m_pos", "token_group"]
    rc = sqa.lib().sqa_paged_attn_shared(*[ref(a[k]) for k in names], a["max_q"], a["scale"], a["bias"], a["cap"], ref(a["gate"]),
                                         ref(a["dst"]), a["ws"], a["ws_bytes"], None)
    ok = sqa.lib().sqa_supports_paged_attn_shared(*[ref(a[k]) for k in names[:4]], ref(a["shared_table"]), a["max_q"], a["scale"],
                                                  a["bias"], a["cap"], ref(a["dst"]))
    return rc, ok


def test_paged_attn_shared_refusals(sqa):
    nan = float("nan")
    arrays = {"q_start": 5, "kv_len": 4, "shared_len": 3, "members": 8, "m_start": 4, "m_pos": 8, "token_group": 8}
    cases = [(1, {k: None}, True) for k in ("shared_len", "members", "m_start", "m_pos", "token_group", "q_start", "kv_len")]
    cases += [(1, {k: ivec(sqa, n + 1, 1 << 26)}, True) for k, n in arrays.items()]
    cases += [(1, {k: ivec(sqa, n, 1 << 26, 27)}, True) for k, n in arrays.items()]
    cases += [(1, {k: None}, False) for k in ("q", "k", "v", "table", "shared_table", "dst")]
    cases += [(1, {"shared_table": T(sqa, 27, [10, 3], [8, 80])}, False), (2, {"shared_table": T(sqa, 26, [10, 5000], [4, 40])}, False),
              (2, {"shared_table": T(sqa, 26, [10, 3], [8, 80])}, False), (2, {"shared_table": T(sqa, 26, [1 << 19, 3], [4, 4 << 19])}, False),
              (1, {"shared_table": T(sqa, 26, [10, 3], [4, 40], 0)}, False), (1, {"shared_table": T(sqa, 26, [0, 3], [4, 40])}, False),
              (6, {"max_q": 0}, False), (1, {"scale": nan}, False), (1, {"bias": -1.0}, False), (1, {"cap": nan}, False),
              (1, {"prefix": ivec(sqa, 3)}, True), (1, {"gate": T(sqa, 0, [D, 16, 7], [4, D * 4, 16 * D * 4])}, True),
              (2, {"q": T(sqa, 1, [D, 8, 16], [4, 16 * D * 4, D * 4])}, False)]
    for status, kw, supported in cases:
        rc, ok = attn(sqa, **kw)
        assert rc == status and ok == int(supported) and sqa.last_error(), (kw, rc, ok, sqa.last_error())
    assert attn(sqa)[0] == 3 and attn(sqa, ws=1 << 40, ws_bytes=64)[0] == 3  # no workspace, too small a one


@pytest.mark.parametrize("name", ["k", "v", "table", "shared_table", "shared_len", "members", "m_start", "m_pos", "token_group", "q_start",
                                  "kv_len"])
def test_paged_attn_shared_refuses_overlaps(sqa, name):
    at = {"k": 1 << 21, "v": 1 << 22, "table": 1 << 23, "shared_table": 1 << 24, "q_start": 4096, "kv_len": 8192, "shared_len": 12288,
          "members": 16384, "m_start": 20480, "m_pos": 24576, "token_group": 28672}[name]
    assert attn(sqa, dst=T(sqa, 0, [D, 16, 8], [4, D * 4, 16 * D * 4], at))[0] == 1 and "overlap" in sqa.last_error()
    assert attn(sqa, ws=at - 64, ws_bytes=1 << 30)[0] == 1 and "overlap" in sqa.last_error()


def test_no_tokens_are_no_work(sqa):
    z = ivec(sqa, 0, 0)
    assert attn(sqa, q=T(sqa, 0, [D, 0, 16], [4, 16 * D * 4, D * 4], 0), dst=T(sqa, 0, [D, 16, 0], [4, D * 4, 16 * D * 4], 0), members=z,
                m_pos=z, token_group=z)[0] == 0


def test_python_refuses_tensors_off_the_gpu(sqa):
    import torch

    i = lambda *n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    with pytest.raises(sqa.SqaError):
        sqa.paged_share(i(3), i(2), i(2), i(1), i(4))
    pool, q = torch.zeros((4, 16, 2, 144), dtype=torch.uint8), torch.zeros((2, 16, D))
    with pytest.raises(sqa.SqaError):
        sqa.paged_attn_shared(q, pool, pool, i(2, 3), i(3), i(2), i(1, 3), i(1), sqa.PagedShare(i(2), i(2), i(2), i(2)), 1)


def test_workspace_size_of_shapes_that_are_refused(sqa):
    q, k = T(sqa, 0, [D, 8, 16], [4, 16 * D * 4, D * 4]), T(sqa, 2, [D, 2, 32, 64], [18, 144, 288, 32 * 288])
    t, size = T(sqa, 26, [10, 4], [4, 40]), sqa.lib().sqa_paged_attn_shared_workspace_size
    assert size(ref(q), ref(k), ref(t), ref(t), 1) > 0
    assert size(ref(q), ref(k), ref(t), None, 1) == size(ref(q), ref(k), None, ref(t), 1) == size(ref(q), ref(k), ref(t), ref(t), 0) == 0
    assert size(ref(T(sqa, 0, [D, 0, 16], [4, 4, 4])), ref(k), ref(t), ref(t), 1) == 0
