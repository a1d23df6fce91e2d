"""References of the operators over a paged pool, from their definitions: whole
numbers in plain Python for the plan, float64 for attention and adapters."""
import math

import numpy as np
import torch

D = 256
ROW = D // 32 * 18


def plan(state, ring, table, n_past, n_new, page, T):
    """Python lists in, a dict of lists out; requests in order, one page at a time."""
    ring, table, n = list(ring), [list(r) for r in table], len(ring)
    head, count = state[0], state[1]
    pages = lambda x: -(-x // page)  # noqa: E731
    W = len(table[0])
    for b, new in enumerate(n_new):
        if new < 0:
            for i in range(min(pages(max(n_past[b], 0)), W)):
                ring[(head + count) % n] = table[b][i]
                count += 1
    start, asked, left, refused = 0, 0, count, 0
    q_start, kv_len, after, slots, pos = [0], [], [], [-1] * T, [0] * T
    for b, new in enumerate(n_new):
        past = max(n_past[b], 0)
        if new < 0:
            q_start.append(min(start, T)), kv_len.append(0), after.append(0)
            continue
        fits = past + new <= W * page and start + new <= T
        need = pages(past + new) - pages(past) if fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= left)
        if ok:
            for i in range(need):
                table[b][pages(past) + i] = ring[(head + asked - need + i) % n]
                count -= 1
            for i in range(new):
                p = past + i
                page_id = table[b][p // page]
                slots[start + i] = page_id * page + p % page if 0 <= page_id < n else -1
                pos[start + i] = p
        refused += not ok
        start += new
        q_start.append(min(start, T))
        kv_len.append(past + new if ok else 0)
        after.append(past + new if ok else past)
    return {"state": [(head + left - count) % n, count, refused, q_start[-1]], "ring": ring, "table": table, "n_past": after,
            "q_start": q_start, "kv_len": kv_len, "slots": slots, "pos": pos * 4}


def quantize(orc, x):
    """float32 (..., 256) -> q4_0 rows uint8 (..., 144)."""
    return orc.quantize_q4_0(np.ascontiguousarray(x)).reshape(*x.shape[:-1], ROW)


def dequant(rows):
    b = rows.reshape(*rows.shape[:-1], 8, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    c = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (c * d).reshape(*rows.shape[:-1], D)


def slopes(H, bias):
    n = 2 ** int(math.floor(math.log2(H)))
    return [2.0 ** (-bias * (h + 1) / n) if h < n else 2.0 ** (-bias / 2 * (2 * (h - n) + 1) / n) for h in range(H)]


def attention(orc, q, k, v, table, q_start, kv_len, prefix=None, scale=None, cap=0.0, bias=0.0, gate=None, fill=0.0):
    """q float32 (n_tok, H, 256), k and v uint8 (n_pages, page, Hkv, 144), numpy; rows of no request get `fill`."""
    from fa_ref import q8_dequant

    n_tok, H, _ = q.shape
    n_pages, page, Hkv, _ = k.shape
    G, scale = H // Hkv, D ** -0.5 if scale is None else scale
    out = np.full(q.shape, fill, dtype=np.float64)
    qd, m = q8_dequant(orc, np.ascontiguousarray(q)), slopes(H, bias)
    for b in range(len(kv_len)):
        t0, n, L = q_start[b], q_start[b + 1] - q_start[b], max(0, kv_len[b])
        if n <= 0:
            continue
        ids = np.array([table[b][j // page] for j in range(L)], dtype=np.int64)
        there = (ids >= 0) & (ids < n_pages)
        at = np.where(there, ids, 0)
        with np.errstate(invalid="ignore"):
            kd, vd = (dequant(x[at, np.arange(L) % page]) if L else np.zeros((0, Hkv, D)) for x in (k, v))
        p = kv_len[b] - n + np.arange(n)[:, None]
        j = np.arange(L)[None, :]
        see = ((j <= p) | (j < (prefix[b] if prefix is not None else 0))) & there[None, :]
        some = see.any(0)
        for h in range(H):
            K, V = np.where(some[:, None], kd[:, h // G], 0), np.where(some[:, None], vd[:, h // G], 0)
            s = scale * (qd[t0:t0 + n, h] @ K.T)
            if cap:
                s = cap * np.tanh(s / cap)
            if bias:
                s = s - m[h] * np.abs(p - j)
            s = np.where(see, s, -np.inf)
            top = s.max(1, keepdims=True) if L else np.full((n, 1), -np.inf)
            w = np.exp(s - np.where(np.isfinite(top), top, 0))
            l = w.sum(1, keepdims=True)
            out[t0:t0 + n, h] = np.where(l > 0, (w @ V) / np.where(l > 0, l, 1), 0)
        if gate is not None:
            out[t0:t0 + n] /= 1 + np.exp(-gate[t0:t0 + n].astype(np.float64))
    return out


def lora(base, x, a, b, ids, scale=None, gate=None):
    """Torch tensors; float64 on the CPU."""
    x = x.double().cpu()
    if gate is not None:
        x = x * torch.sigmoid(gate.double().cpu())
    out = base.double().cpu().clone()
    for m, i in enumerate(ids.tolist()):
        if 0 <= i < a.shape[0]:
            s = 1.0 if scale is None else float(scale[i])
            out[m] += s * (b[i].double().cpu() @ (a[i].double().cpu() @ x[m]))
    return out
