"""References of the operators of shared prefixes and of cached rows, from their definitions: whole numbers in
plain Python for the plan, float64 for attention and rotations, the quantizer's float32 operations in numpy."""
import numpy as np

import paged_ref

D, ROW = 256, 144


def share(q_start, kv_len, group, shared_len, T, pos=None):
    """Python lists in, a dict of lists out."""
    B, G = len(kv_len), len(shared_len)
    start = [min(max(x, 0), T) for x in q_start]
    rows, token_group = [[] for _ in range(G)], [-1] * T
    pos = list(pos) if pos is not None else None
    for b in range(B):
        g, n = group[b], max(0, start[b + 1] - start[b])
        if not 0 <= g < G or kv_len[b] <= 0 or shared_len[g] <= 0:
            continue
        for i in range(n):
            t, p = start[b] + i, shared_len[g] + kv_len[b] - n + i
            rows[g].append((t, p))
            token_group[t] = g
            if pos is not None:
                for c in range(4):
                    pos[c * T + t] = p
    m_start = [0]
    for r in rows:
        m_start.append(m_start[-1] + len(r))
    flat = [x for r in rows for x in r]
    rest = [-1] * (T - len(flat))
    return {"members": [t for t, _ in flat] + rest, "m_start": m_start, "m_pos": [p for _, p in flat] + rest,
            "token_group": token_group, "pos": pos}


def attention(orc, q, k, v, table, q_start, kv_len, shared_table, shared_len, group, prefix=None, scale=None, cap=0.0,
              bias=0.0, gate=None, fill=0.0):
    """q float32 (n_tok, H, 256), k and v uint8 (n_pages, page, Hkv, 144), numpy; rows of no request get `fill`."""
    from fa_ref import q8_dequant

    n_tok, H, _ = q.shape
    n_pages, page, Hkv, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out = np.full(q.shape, fill, dtype=np.float64)
    qd, m = q8_dequant(orc, np.ascontiguousarray(q)), paged_ref.slopes(H, bias)

    def pages(row, n):
        ids = np.array([row[j // page] for j in range(n)], dtype=np.int64)
        there = (ids >= 0) & (ids < n_pages)
        at = np.where(there, ids, 0)
        with np.errstate(invalid="ignore"):
            kd, vd = (paged_ref.dequant(x[at, np.arange(n) % page]) if n else np.zeros((0, Hkv, D)) for x in (k, v))
        return kd, vd, there

    for b in range(len(kv_len)):
        t0, n, L = q_start[b], q_start[b + 1] - q_start[b], max(0, kv_len[b])
        if n <= 0:
            continue
        g = group[b] if 0 <= group[b] < len(shared_len) and kv_len[b] > 0 else -1
        S = max(0, shared_len[g]) if g >= 0 else 0
        ks, vs, ts = pages(shared_table[g] if S else [], S)
        ko, vo, to = pages(table[b], L)
        p = kv_len[b] - n + np.arange(n)[:, None]  # among its own keys
        j = np.arange(L)[None, :]
        own = ((j <= p) | (j < (prefix[b] if prefix is not None else 0))) & to[None, :]
        see = np.concatenate([np.repeat(ts[None, :], n, 0), own], 1)
        far = np.abs(S + p - np.arange(S + L)[None, :])
        kd, vd, some = np.concatenate([ks, ko]), np.concatenate([vs, vo]), see.any(0)
        for h in range(H):
            K, V = (np.where(some[:, None], x[:, h // (H // Hkv)], 0) for x in (kd, vd))
            s = scale * (qd[t0:t0 + n, h] @ K.T)
            if cap:
                s = cap * np.tanh(s / cap)
            if bias:
                s = s - m[h] * far
            s = np.where(see, s, -np.inf)
            top = s.max(1, keepdims=True) if S + L else np.full((n, 1), -np.inf)
            w = np.exp(s - np.where(np.isfinite(top), top, 0))
            l = w.sum(1, keepdims=True)
            out[t0:t0 + n, h] = np.where(l > 0, (w @ V) / np.where(l > 0, l, 1), 0)
        if gate is not None:
            out[t0:t0 + n] /= 1 + np.exp(-gate[t0:t0 + n].astype(np.float64))
    return out


def values(rows):
    """q4_0 bytes (..., 18 * blocks) -> float64 (..., 32 * blocks), (code - 8) * d."""
    b = rows.reshape(*rows.shape[:-1], -1, 18)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    c = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8
    return (c * d).reshape(*rows.shape[:-1], -1)


def which(n_rot, sections):
    """Position component (t, h, w, e) of every rotation pair."""
    total, out = sum(sections), []
    for ic in range(n_rot // 2):
        s = ic % total
        out.append(1 if s % 3 == 1 and s < 3 * sections[1] else 2 if s % 3 == 2 and s < 3 * sections[2] else
                   0 if s % 3 == 0 and s < 3 * sections[0] else 3)
    return out


def turned(rows, delta, n_rot, sections, base, freq_scale=1.0):
    """Values (n, heads, D) of rows (n, heads, bytes) with the heads' first n_rot dims rotated on, float64."""
    n, half = rows.shape[0], n_rot // 2
    x = values(rows)
    comp = which(n_rot, sections)
    d = np.asarray(delta, dtype=np.float64).reshape(4, n)
    angle = np.stack([d[comp[i]] * (float(np.float32(freq_scale)) * float(np.float32(base)) ** (-2.0 * i / n_rot))
                      for i in range(half)], -1)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    y = x.copy()
    y[..., :half] = x[..., :half] * c - x[..., half:n_rot] * s
    y[..., half:n_rot] = x[..., :half] * s + x[..., half:n_rot] * c
    return y
