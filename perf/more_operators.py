"""Performance cases of the operators for requests that share cached keys, and for cached rows that are read back or moved.

Four kinds, each one call of the package:

  share  paged_share: which tokens of a step go with which shared prefix, and their positions behind it, on the GPU.
  attn   paged_attn_shared: attention of every request's new tokens over its own pages and over the pages of the prefix
         that its group shares, whose keys are read and multiplied once for all tokens of the group.
  get    get_rows_q4_0: cached rows read back as float32 or float16.
  move   move_rows_q4_0: cached keys moved to other rows and rotated to other positions, then read back.

The lengths of a case follow from its own numbers (`lens` seeds them), the values from prepare's seed.
"""
import math
import random

import torch

own = False

D = 256  # head dim of the attention kernels
ROW = D // 32 * 18
SCRATCH = 512 << 20   # the workspace that a serving loop keeps for every step
MOST_PAIRS = 1 << 29  # (query row, key) pairs of the plain form, requests and groups padded to the longest
ROPE = (64, (11, 11, 10, 0), 1e7)


def listed():
    def share(name, B, groups, tokens, pad, lens):
        return {"name": name, "kind": "share", "B": B, "groups": groups, "tokens": tokens, "pad": pad, "lens": lens}

    def attn(name, B, groups, shared, n, past, page, lens, alone=0.0, cap=0.0, bias=0.0, gate=False, pad=0, H=16, Hkv=2):
        return {"name": name, "kind": "attn", "B": B, "groups": groups, "shared_lo": shared[0], "shared_hi": shared[1],
                "n_lo": n[0], "n_hi": n[1], "past_lo": past[0], "past_hi": past[1], "page": page, "lens": lens,
                "alone": alone, "cap": cap, "bias": bias, "gate": gate, "pad": pad, "H": H, "Hkv": Hkv}

    def get(name, n, rows, half, lens, Hkv=2):
        return {"name": name, "kind": "get", "n": n, "rows": rows, "half": half, "lens": lens, "Hkv": Hkv}

    def move(name, n, far, lens, Hkv=2):
        return {"name": name, "kind": "move", "n": n, "far": far, "lens": lens, "Hkv": Hkv}

    return [
        # one decode step of eight conversations under one system prompt: a latency, nothing else
        share("share_decode_8", 8, 1, 8, 0, 1),
        # a full server's step: a thousand requests under forty prompts, prompt chunks among them, spare rows behind
        share("share_step_1024", 1024, 40, 8192, 37, 2),
        # two conversations that have just begun
        attn("decode_2_after_500", 2, 1, (500, 500), (1, 1), (3, 40), 64, 3),
        # the ordinary decode step of a server whose requests share its system prompt and tools, gated
        attn("decode_64_after_8k", 64, 1, (8191, 8191), (1, 1), (100, 2000), 64, 4, gate=True),
        # many questions about one long document
        attn("decode_128_after_60k", 128, 1, (60001, 60001), (1, 1), (20, 600), 256, 5),
        # several prompts and some requests without one, small pages, a model with capped logits, spare rows
        attn("decode_80_5_prompts", 80, 5, (300, 12000), (1, 1), (0, 3000), 16, 6, alone=0.2, cap=30.0, pad=13),
        # drafts to verify, a model with distance biases
        attn("verify_24_bias", 24, 2, (3000, 20000), (1, 4), (50, 1500), 32, 7, bias=8.0),
        # prompts that arrive together behind the same long instructions
        attn("prompts_12_after_16k", 12, 1, (16000, 16000), (37, 300), (0, 0), 128, 8, gate=True),
        # a few rows to look at
        get("get_57", 57, 4096, False, 9),
        # a long conversation's keys for an engine that holds its cache in float16
        get("get_131072_half", 131072, 140000, True, 10),
        # a retrieved passage behind another prompt
        move("move_500", 500, 20000, 11),
        # a conversation at its context's end drops its oldest part
        move("move_100001", 100001, 30000, 12),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    lens = rng.randrange(1 << 20)
    kind = rng.choice(["share", "attn", "attn", "attn", "get", "move"])
    if kind == "share":
        B = log(1, 1024)
        return {"kind": kind, "B": B, "groups": log(1, min(B, 64)), "tokens": log(B, 8192), "pad": rng.choice([0, rng.randint(1, 60)]),
                "lens": lens}
    if kind == "get":
        n = log(1, 131072)
        return {"kind": kind, "n": n, "rows": rng.randint(max(64, n // 2), 140000), "half": rng.random() < 0.5, "lens": lens,
                "Hkv": rng.choice([1, 2, 2, 4])}
    if kind == "move":
        Hkv = rng.choice([1, 2, 2, 4])
        return {"kind": kind, "n": log(1, 200000 // Hkv), "far": log(1, 200000), "lens": lens, "Hkv": Hkv}
    H, Hkv = rng.choice([(16, 2), (16, 2), (16, 2), (16, 4), (8, 2), (8, 1), (4, 4)])
    case = {"kind": kind, "B": 1, "groups": 1, "shared_lo": 0, "shared_hi": 0, "n_lo": 1, "n_hi": 1, "past_lo": 0, "past_hi": 0,
            "page": rng.choice([16, 32, 64, 128, 256]), "lens": lens, "alone": rng.choice([0.0, 0.0, 0.3]),
            "cap": rng.choice([0.0, 0.0, 0.0, 30.0]), "bias": rng.choice([0.0, 0.0, 0.0, 8.0]), "gate": rng.random() < 0.4,
            "pad": rng.choice([0, 0, rng.randint(1, 40)]), "H": H, "Hkv": Hkv}
    form = rng.choice(["decode", "decode", "verify", "chunk"])
    if form == "chunk":
        case["B"] = rng.randint(2, 16)
        case["n_hi"] = log(20, 2400 // case["B"])
        case["past_hi"] = rng.choice([0, log(16, 2000)])
    else:
        case["B"], case["n_hi"] = log(2, 128), 1 if form == "decode" else rng.randint(2, 4)
        case["past_hi"] = log(1, 4000)
    case["n_lo"], case["past_lo"] = rng.randint(1, case["n_hi"]), rng.randint(0, case["past_hi"])
    case["groups"] = rng.choice([1, 1, rng.randint(1, max(1, min(8, case["B"] // 2)))])
    tokens = case["B"] * case["n_hi"] * H
    most = min(60001, MOST_PAIRS // (tokens * (1 if case["groups"] == 1 else case["groups"])))
    case["shared_hi"] = log(min(200, most), most)
    case["shared_lo"] = rng.randint(case["shared_hi"] // 8, case["shared_hi"])
    return case


# ------------------------------------------------------------------ lengths --

def _attn_lens(case):
    """(new, past, group, shared): new and cached own tokens and group (-1: none) of every request, keys of every group."""
    r = random.Random(case["lens"])
    B, G = case["B"], case["groups"]
    new = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(B)]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(B)]
    group = [r.randrange(G) if r.random() >= case["alone"] else -1 for _ in range(B)]
    shared = [r.randint(case["shared_lo"], case["shared_hi"]) for _ in range(G)]
    return new, past, group, shared


def _share_lens(case):
    """(new, kv, group, shared) of every request and group: decoding requests, some prompt chunks, some that wait (kv 0)."""
    r = random.Random(case["lens"])
    B, G = case["B"], case["groups"]
    new = [1 if r.random() < 0.95 else 0 for _ in range(B)]
    left = case["tokens"] - sum(new)
    while left > 0:
        n = min(left, r.randint(1, 1 + max(1, case["tokens"] // 6)))
        new[r.randrange(B)] += n
        left -= n
    kv = [n + r.randint(0, 3000) if r.random() < 0.97 else 0 for n in new]
    group = [r.randrange(G) if r.random() < 0.9 else -1 for _ in range(B)]
    shared = [r.randint(1, 60000) if r.random() < 0.95 else 0 for _ in range(G)]
    return new, kv, group, shared


def _pages(n, page):
    return (n + page - 1) // page


# ------------------------------------------------------------------ inputs --

def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def _q4_0(x):
    """Rows of q4_0 blocks (fp16 scale, 16 bytes of codes) of float32 rows."""
    b = x.reshape(-1, 32)
    top = b.gather(1, b.abs().argmax(1, keepdim=True))
    d = top / -8.0
    inv = torch.where(d != 0, torch.ones_like(d) / d, torch.zeros_like(d))
    c = (b * inv + 8.5).to(torch.int32).clamp_(0, 15).to(torch.uint8)
    out = torch.empty((b.shape[0], 18), dtype=torch.uint8, device=x.device)
    out[:, :2] = d.to(torch.float16).view(torch.uint8)
    out[:, 2:] = c[:, :16] | (c[:, 16:] << 4)
    return out.reshape(x.shape[0], -1)


def _cache(gen, rows, Hkv):
    out = torch.empty((rows, Hkv * ROW), dtype=torch.uint8, device="cuda")
    for r in range(0, rows, 65536):
        n = min(65536, rows - r)
        out[r:r + n] = _q4_0(_randn(gen, n, Hkv * D))
    return out.view(rows, Hkv, ROW)


def _table(gen, used, first, total):
    """Page table of rows of `used` pages, out of a permutation of `total` pages from place `first` on."""
    W = max(1, max(used))
    ids = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)[first:first + sum(used)]
    table = torch.full((len(used), W), -1, dtype=torch.int32, device="cuda")
    table[torch.arange(W, device="cuda")[None, :] < torch.tensor(used, device="cuda")[:, None]] = ids
    return table


def _share_buffers(T, G):
    i32 = dict(dtype=torch.int32, device="cuda")
    return {"members": torch.zeros(T, **i32), "m_start": torch.zeros(G + 1, **i32), "m_pos": torch.zeros(T, **i32),
            "token_group": torch.zeros(T, **i32), "pos": torch.zeros(4 * T, **i32)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "share":
        new, kv, group, shared = _share_lens(case)
        T = sum(new) + case["pad"]
        kv, shared = _i32(kv), _i32(shared)
        more = [torch.randint(0, 500, x.shape, generator=gen, device="cuda", dtype=torch.int32) for x in (kv, shared)]
        s |= {"q_start": _i32(_starts(new)), "kv_len": torch.where(kv > 0, kv + more[0], kv), "group": _i32(group),
              "shared_len": torch.where(shared > 0, shared + more[1], shared), **_share_buffers(max(1, T), case["groups"])}
        s["pos"].random_(0, 4000, generator=gen)  # what the step's plan wrote
    elif case["kind"] == "attn":
        new, past, group, shared = _attn_lens(case)
        page, H, Hkv = case["page"], case["H"], case["Hkv"]
        kv = [n + p for n, p in zip(new, past)]
        used, held = [_pages(k, page) for k in kv], [_pages(k, page) for k in shared]
        total, T = sum(used) + sum(held), sum(new) + case["pad"]
        s["k"], s["v"] = (_cache(gen, total * page, Hkv).view(total, page, Hkv, ROW) for _ in range(2))
        both = _table(gen, used + held, 0, total)
        s |= {"table": both[:case["B"], :max(used)].contiguous(), "shared_table": both[case["B"]:, :max(1, max(held))].contiguous(),
              "q_start": _i32(_starts(new)), "kv_len": _i32(kv), "group": _i32(group), "shared_len": _i32(shared),
              "max_q": max(new), "max_kv": max(kv), "max_shared": max(shared), "q": _randn(gen, T, H, D),
              "gate": _randn(gen, T, H, D) if case["gate"] else None,
              "out": torch.zeros((T, H, D), dtype=torch.float32, device="cuda")}
        s |= _share_buffers(T, case["groups"])
        s |= _share_plain(s)  # a step's plan, there before its layers
        s["most"] = int((s["m_start"][1:] - s["m_start"][:-1]).max())
        s["ws"] = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    elif case["kind"] == "get":
        s["cache"] = _cache(gen, case["rows"], case["Hkv"])
        s["idx"] = torch.randint(0, case["rows"], (case["n"],), generator=gen, device="cuda")
        dtype = torch.float16 if case["half"] else torch.float32
        s["out"] = torch.zeros((case["n"], case["Hkv"] * D), dtype=dtype, device="cuda")
    else:
        n, gone = case["n"], 64 + case["n"] // 3
        s["cache"], s["dst"] = _cache(gen, n + gone, case["Hkv"]), _cache(gen, n + gone, case["Hkv"])
        s["from"] = torch.arange(gone, gone + n, device="cuda")
        s["to"] = torch.randperm(n + gone, generator=gen, device="cuda")[:n]
        far = int(torch.randint(1, case["far"] + 1, (1,), generator=gen, device="cuda"))
        s["delta"] = torch.full((4 * n,), -far, dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros((n, case["Hkv"] * D), dtype=torch.float16, device="cuda")
    return s


# ------------------------------------------------------------ plain forms --

def _share_plain(s):
    start, kv, group, shared = (s[k].long() for k in ("q_start", "kv_len", "group", "shared_len"))
    B, G, T, dev = kv.shape[0], shared.shape[0], s["members"].shape[0], kv.device
    start = start.clamp(0, T)
    n = start[1:] - start[:-1]
    ok = (group >= 0) & (group < G) & (kv > 0)
    g_of = torch.where(ok, group, torch.full_like(group, G))
    g_of = torch.where(torch.cat([shared, shared.new_zeros(1)])[g_of] > 0, g_of, torch.full_like(g_of, G))
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True).clamp(max=B - 1)
    live = (t >= start[0]) & (t < start[-1])
    tg = torch.where(live, g_of[b], torch.full_like(t, G))
    order = torch.argsort(tg, stable=True)
    count = torch.zeros(G + 1, dtype=torch.int64, device=dev).index_add_(0, tg, torch.ones_like(tg))
    m_start = torch.cat([count.new_zeros(1), torch.cumsum(count[:G], 0)])
    pos = torch.cat([shared, shared.new_zeros(1)])[tg] + kv[b] - n[b] + t - start[b]
    some = t < m_start[-1]
    member = tg < G
    minus = torch.full_like(t, -1)
    i32 = torch.int32
    return {"members": torch.where(some, order, minus).to(i32), "m_start": m_start.to(i32),
            "m_pos": torch.where(some, pos[order], minus).to(i32), "token_group": torch.where(member, tg, minus).to(i32),
            "pos": torch.where(member.repeat(4), pos.repeat(4), s["pos"].long()).to(i32)}


def _q8_0(q):
    """q rounded to q8_0 blocks of 32 values: fp16 scale amax / 127, codes round(x * 127 / amax)."""
    b = q.reshape(-1, 32)
    amax = b.abs().amax(1, keepdim=True)
    inv = torch.where(amax != 0, torch.full_like(amax, 127.0) / amax, torch.zeros_like(amax))
    return (torch.round(b * inv) * (amax / 127.0).half().float()).reshape(q.shape)


def _dequant(rows):
    """(..., 144) q4_0 rows -> (..., 256) float32."""
    b = rows.reshape(*rows.shape[:-1], D // 32, 18)
    d = b[..., :2].contiguous().view(torch.float16).float()
    c = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8.0
    return (c * d).reshape(*rows.shape[:-1], D)


def _slopes(H, bias, device):
    """Distance slope of every head: 2^(-bias (h + 1) / n) for the first n = 2^floor(log2 H) heads, between them after."""
    n = 1 << (H.bit_length() - 1)
    h = torch.arange(H, device=device, dtype=torch.float64)
    e = torch.where(h < n, -bias * (h + 1) / n, -0.5 * bias * (2 * (h - n) + 1) / n)
    return torch.exp2(e)


def _part(s, q, table, L, pos, see):
    """Maximum, sum and weighted values of rows q (R, n, H, D) at positions pos (R, n) over the first L keys of the
    table's rows, of which each row sees the first `see` (R, n)."""
    case = s["case"]
    H, Hkv, page = case["H"], case["Hkv"], case["page"]
    G, (R, n), dev = H // Hkv, pos.shape, q.device
    j = torch.arange(L, device=dev)
    pid = table.long()[:, torch.div(j, page, rounding_mode="floor")]  # (R, L)
    at = pid.clamp(min=0) * page + j % page
    k = _dequant(s["k"].reshape(-1, Hkv, ROW)[at]).transpose(1, 2).contiguous()  # (R, Hkv, L, D)
    q = q.reshape(R, n, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, n * G, D)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous())
    del k
    x = x.mul_(D ** -0.5).reshape(R, Hkv, n, G, L)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["bias"]:
        far = (pos[:, :, None] - j).abs().float()
        x = x.sub_(_slopes(H, case["bias"], dev).float().reshape(1, Hkv, 1, G, 1) * far[:, None, :, None, :])
    dead = ((j >= see[:, :, None]) | (pid < 0)[:, None, :])[:, None, :, None, :]
    x = x.masked_fill_(dead, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    l = x.sum(-1, keepdim=True)
    v = _dequant(s["v"].reshape(-1, Hkv, ROW)[at]).transpose(1, 2).contiguous()
    o = torch.matmul(x.reshape(R, Hkv, n * G, L), v).reshape(R, Hkv, n, G, D)
    return tuple(y.permute(0, 2, 1, 3, 4).reshape(R, n, H, y.shape[-1]) for y in (m, l, o))


def _attn_plain(s):
    case = s["case"]
    B, T, dev = case["B"], s["q"].shape[0], s["q"].device
    q = _q8_0(s["q"])

    def rows_of(starts, order, longest):
        """(token rows, which of them are there) of every range, padded to the longest."""
        i = torch.arange(longest, device=dev)
        at = (starts[:-1, None] + i).clamp(max=T - 1)
        return (at if order is None else order[at].clamp(min=0)), i < (starts[1:] - starts[:-1])[:, None]

    parts = []
    start, kv = s["q_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    rows, live = rows_of(start, None, s["max_q"])
    own_pos = kv[:, None] - n[:, None] + torch.arange(s["max_q"], device=dev)
    parts.append((rows, live, _part(s, q[rows], s["table"], s["max_kv"], own_pos, torch.minimum(own_pos + 1, kv[:, None]))))
    if s["most"] > 0:
        ms, order = s["m_start"].long(), s["members"].long()
        rows, live = rows_of(ms, order, s["most"])
        at = (ms[:-1, None] + torch.arange(s["most"], device=dev)).clamp(max=T - 1)
        see = s["shared_len"].long()[:, None].expand(-1, s["most"])
        parts.append((rows, live, _part(s, q[rows], s["shared_table"], s["max_shared"], s["m_pos"].long()[at], see)))
    m = torch.full((len(parts), T, case["H"], 1), -math.inf, device=dev)
    l, o = torch.zeros_like(m), torch.zeros((len(parts), *s["q"].shape), device=dev)
    for i, (rows, live, part) in enumerate(parts):
        m[i, rows[live]], l[i, rows[live]], o[i, rows[live]] = (y[live] for y in part)
    top = m.amax(0)
    w = torch.exp(m - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = (w * l).sum(0)
    out = torch.where(total > 0, (w * o).sum(0) / total, torch.zeros_like(s["q"]))
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"])
    return out


def _get_plain(s):
    rows = s["cache"][s["idx"]]
    return _dequant(rows).reshape(s["out"].shape).to(s["out"].dtype)


def _pairs(n_rot, sections):
    """Which of the positions t, h, w, e turns each rotation pair."""
    total = sum(sections)
    out = []
    for i in range(n_rot // 2):
        k = i % total
        c = [c for c in (1, 2, 0) if k % 3 == c and k < 3 * sections[c]]
        out.append(c[0] if c else 3)
    return out


def _move_plain(s):
    n_rot, sections, base = ROPE
    half, n = n_rot // 2, s["from"].shape[0]
    rows = s["cache"][s["from"]]                                       # (n, Hkv, 144)
    x = _dequant(rows)[..., :n_rot]
    turn = s["delta"].view(4, n)[torch.tensor(_pairs(n_rot, sections), device=x.device)].t().double()  # (n, half)
    freq = torch.tensor(base, dtype=torch.float64, device=x.device) ** (
        torch.arange(half, device=x.device, dtype=torch.float64) * (-2.0 / n_rot))
    c, si = (f(turn * freq).float()[:, None, :] for f in (torch.cos, torch.sin))
    a, b = x[..., :half], x[..., half:]
    y = torch.cat([a * c - b * si, a * si + b * c], -1)
    moved = torch.cat([_q4_0(y.reshape(-1, n_rot)).reshape(n, -1, n_rot // 32 * 18), rows[..., n_rot // 32 * 18:]], -1)
    s["dst"][s["to"]] = moved
    return _dequant(s["dst"][s["to"]]).reshape(s["out"].shape).half()


def run(s):
    kind = s["case"]["kind"]
    if own:
        sqa = _package()
        if kind == "share":
            sqa.paged_share(s["q_start"], s["kv_len"], s["group"], s["shared_len"], s["members"], s["m_start"], s["m_pos"],
                            s["token_group"], pos=s["pos"])
            return {k: s[k] for k in ("members", "m_start", "m_pos", "token_group", "pos")}
        if kind == "attn":
            share = sqa.PagedShare(s["members"], s["m_start"], s["m_pos"], s["token_group"])
            return sqa.paged_attn_shared(s["q"], s["k"], s["v"], s["table"], s["q_start"], s["kv_len"], s["shared_table"],
                                         s["shared_len"], share, s["max_q"], softcap=s["case"]["cap"],
                                         max_bias=s["case"]["bias"], gate=s["gate"], out=s["out"], workspace=s["ws"])
        if kind == "get":
            return sqa.get_rows_q4_0(s["cache"], s["idx"], out=s["out"])
        sqa.move_rows_q4_0(s["dst"], s["cache"], s["to"], s["from"], s["delta"], sqa.rope_params(*ROPE))
        return sqa.get_rows_q4_0(s["dst"], s["to"], out=s["out"])
    return {"share": _share_plain, "attn": _attn_plain, "get": _get_plain, "move": _move_plain}[kind](s)


def _package():
    import __graft_entry__ as graft

    return graft.load_package()


# ------------------------------------------------------------------- floors --

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    if case["kind"] == "share":
        new, kv, group, shared = _share_lens(case)
        n = sum(x for x, k, g in zip(new, kv, group) if k and g >= 0 and shared[g])
        return {"bytes": 12 * len(new) + 8 * len(shared) + 12 * (sum(new) + case["pad"]) + 16 * n, "flops": 0}
    if case["kind"] == "get":
        values = case["n"] * case["Hkv"] * D
        return {"bytes": case["n"] * (case["Hkv"] * ROW + 8) + values * (2 if case["half"] else 4), "flops": 2 * values}
    if case["kind"] == "move":
        n, Hkv = case["n"], case["Hkv"]
        return {"bytes": n * (3 * Hkv * ROW + 32) + n * Hkv * D * 2, "flops": n * Hkv * (6 * ROPE[0] + 2 * D)}
    new, past, group, shared = _attn_lens(case)
    pairs = sum(n * p + n * (n + 1) // 2 + (n * shared[g] if g >= 0 else 0) for n, p, g in zip(new, past, group))
    keys = sum(n + p for n, p in zip(new, past)) + sum(shared[g] for g in set(group) if g >= 0)
    rows = sum(new) * case["H"]
    return {"bytes": keys * case["Hkv"] * 2 * ROW + rows * D * 4 * (3 if case["gate"] else 2) + 12 * case["B"] +
            4 * keys // case["page"] + 12 * sum(new), "flops": 4 * D * pairs * case["H"]}


# ------------------------------------------------- definitions in 64 bits --

def _values(rows, n_values):
    """q4_0 bytes (n, 18 * blocks) as float64."""
    raw = rows.reshape(rows.shape[0], -1, 18)
    d = raw[:, :, :2].contiguous().view(torch.float16).double()
    return torch.cat([(raw[:, :, 2:] & 15).double() - 8, (raw[:, :, 2:] >> 4).double() - 8], 2).mul_(d).reshape(-1, n_values)


def _exact_attn(case, s):
    new, past, group, shared = _attn_lens(case)
    H, Hkv, page = case["H"], case["Hkv"], case["page"]
    G, out, t0 = H // Hkv, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    blocks = s["q"].reshape(-1, 32)  # q8_0 is defined by its float32 operations
    top = blocks.abs().max(1).values
    code = torch.where(top[:, None] > 0, (blocks * (torch.full_like(top, 127.0) / top)[:, None]).round(), 0 * blocks)
    q8 = (code.double() * (top / 127.0).to(torch.float16).double()[:, None]).reshape(s["q"].shape)

    def keys(pool, pages, n, h):
        return _values(pool[pages[:_pages(n, page)].long()][:, :, h].reshape(-1, ROW)[:n], D)

    prefix = [[(keys(s["k"], s["shared_table"][g], shared[g], h), keys(s["v"], s["shared_table"][g], shared[g], h))
               for h in range(Hkv)] for g in range(case["groups"])]
    nl2 = 2 ** int(math.floor(math.log2(H)))
    for b in range(case["B"]):
        n, L, before = new[b], new[b] + past[b], shared[group[b]] if group[b] >= 0 else 0
        j = torch.arange(before + L, device="cuda", dtype=torch.float64)
        p = torch.arange(before + past[b], before + L, device="cuda", dtype=torch.float64)[:, None]
        for h in range(Hkv):
            K, V = keys(s["k"], s["table"][b], L, h), keys(s["v"], s["table"][b], L, h)
            if before:
                K, V = torch.cat([prefix[group[b]][h][0], K]), torch.cat([prefix[group[b]][h][1], V])
            x = (q8[t0:t0 + n, h * G:(h + 1) * G].reshape(n * G, D) @ K.t()).reshape(n, G, -1) / 16.0
            if case["cap"]:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["bias"]:
                hq = [h * G + g for g in range(G)]
                m = [2.0 ** (-case["bias"] * (i + 1) / nl2) if i < nl2 else
                     2.0 ** (-case["bias"] / 2 * (2 * (i - nl2) + 1) / nl2) for i in hq]
                x = x - torch.tensor(m, device="cuda", dtype=torch.float64)[None, :, None] * (p - j).abs()[:, None, :]
            x = torch.where((j <= p)[:, None, :], x, torch.full_like(x, -math.inf))
            out[t0:t0 + n, h * G:(h + 1) * G] = (torch.softmax(x, 2).reshape(n * G, -1) @ V).reshape(n, G, D)
        t0 += n
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))


def _exact_move(s):
    n_rot, sections, base = ROPE
    n, Hkv = s["from"].shape[0], s["cache"].shape[1]
    x = _values(s["cache"][s["from"]].reshape(n * Hkv, ROW), D)
    half, total = n_rot // 2, sum(sections)
    z = torch.complex(x[:, :half].clone(), x[:, half:n_rot].clone()).reshape(n, Hkv, half)
    for i in range(half):
        k = i % total
        which = 1 if k % 3 == 1 and k < 3 * sections[1] else 2 if k % 3 == 2 and k < 3 * sections[2] else \
            0 if k % 3 == 0 and k < 3 * sections[0] else 3
        angle = s["delta"][which * n:(which + 1) * n].double() * base ** (-2.0 * i / n_rot)
        z[:, :, i] *= torch.polar(torch.ones_like(angle), angle)[:, None]
    turned = torch.cat([z.real, z.imag], -1).reshape(n * Hkv, n_rot)
    # q4_0 is defined by its float32 operations
    blocks = turned.float().reshape(-1, 32)
    largest = blocks.abs().max(1, keepdim=True).values
    d = blocks.gather(1, (blocks.abs() == largest).int().argmax(1, keepdim=True)) / -8.0
    code = torch.where(d != 0, (blocks * (1.0 / d) + 8.5).trunc().clamp(0, 15), torch.full_like(blocks, 8.0))
    x[:, :n_rot] = ((code.double() - 8) * d.half().double()).reshape(n * Hkv, n_rot)
    return x.reshape(n, Hkv * D)


def exact(case, seed):
    if case["kind"] == "share":
        return None  # whole numbers, compared as they are
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    if case["kind"] == "get":
        return _values(s["cache"][s["idx"]].reshape(-1, ROW), D).reshape(s["out"].shape)
    return _exact_move(s)
