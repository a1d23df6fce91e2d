"""Performance cases of the operators that serve a batch of requests from one paged q4_0 pool.

Three kinds, each one call of the package:

  plan  paged_plan: the page table, slot map, rotary positions and request bounds of a step, on the GPU.
  attn  paged_attn: attention of every request's new tokens over its pages, causal, with the options a model may
        bring: a tanh cap of the logits, a distance bias (max_bias), a prefix that every token sees, an output gate.
  lora  lora_add: the low-rank adapters of the step's requests added to a shared projection's output.

The lengths of a case follow from its own numbers (`lens` seeds them), the values from prepare's seed.
"""
import math
import random

import torch

own = False

D = 256        # head dim of the attention kernels
N_EMBD = 2048  # width of the W_o output
ROW = D // 32 * 18
MOST_PAIRS = 2048 * 32049 * 16  # (query row, key) pairs of the largest attention case
SCRATCH = 256 << 20  # the workspace that a serving loop keeps for every step
MOST_DENSE = 5e9                # the same, every request padded to the longest


def listed():
    def plan(name, B, W, page, tokens, ended, lens):
        return {"name": name, "kind": "plan", "B": B, "W": W, "page": page, "tokens": tokens, "ended": ended, "lens": lens}

    def attn(name, B, page, n, past, lens, H=16, Hkv=2, chunks=0, cap=0.0, bias=0.0, prefix=0, gate=False, pad=0):
        return {"name": name, "kind": "attn", "B": B, "page": page, "n_lo": n[0], "n_hi": n[1], "past_lo": past[0],
                "past_hi": past[1], "lens": lens, "H": H, "Hkv": Hkv, "chunks": chunks, "cap": cap, "bias": bias,
                "prefix": prefix, "gate": gate, "pad": pad}

    def lora(name, M, K, N, r, adapters, group, lens, gate):
        return {"name": name, "kind": "lora", "M": M, "K": K, "N": N, "r": r, "adapters": adapters, "group": group,
                "lens": lens, "gate": gate}

    return [
        # one decode step of eight conversations: a latency, nothing else
        plan("plan_decode_8", 8, 256, 64, 8, 0, 1),
        # a full server's step: a thousand requests, prompt chunks among them, some that end, small pages
        plan("plan_step_1024", 1024, 1024, 16, 8192, 40, 2),
        # a single conversation's decode step
        attn("decode_1x4k", 1, 64, (1, 1), (4095, 4095), 3),
        # the ordinary decode step of a busy server: short and long contexts side by side, small pages
        attn("decode_64_ragged", 64, 16, (1, 1), (150, 8191), 4, gate=True),
        # decode of few users with very long contexts, 1.1 GB of cache
        attn("decode_16x120k", 16, 256, (1, 1), (100000, 131071), 5),
        # speculative verify of two positions in a batch, a model with capped logits
        attn("verify2_12_capped", 12, 32, (2, 2), (3000, 20000), 6, cap=30.0),
        # prompts that arrive together, from their first token, a model with distance biases
        attn("prompts_8_bias", 8, 16, (37, 1200), (0, 0), 7, bias=8.0),
        # a step that mixes decoding requests with two prompt chunks; the token buffer has spare rows
        attn("mixed_24_2", 26, 64, (1, 1), (500, 6000), 8, chunks=512, gate=True, pad=19),
        # images before text: every token sees the prefix; continued and first chunks of odd sizes
        attn("prefix_3_capped_gate", 3, 128, (150, 700), (0, 2500), 9, cap=50.0, prefix=600, gate=True),
        # the largest ubatch behind a long prompt
        attn("chunk2048_after_30001", 1, 64, (2048, 2048), (30001, 30001), 10),
        # W_o adapters of a decode step, every request its own
        lora("lora_decode_48", 48, 4096, N_EMBD, 16, 32, 1, 11, True),
        # W_o adapters of prompt chunks
        lora("lora_chunks_4096", 4096, 4096, N_EMBD, 64, 8, 512, 12, True),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    lens = rng.randrange(1 << 20)
    kind = rng.choice(["plan", "attn", "attn", "attn", "attn", "lora", "lora"])
    if kind == "plan":
        B = log(1, 1024)
        return {"kind": kind, "B": B, "W": log(8, 1024), "page": rng.choice([16, 32, 64, 128, 256]),
                "tokens": log(B, 8192), "ended": rng.randint(0, max(0, B // 8)), "lens": lens}
    if kind == "lora":
        M = log(1, 4096)
        return {"kind": kind, "M": M, "K": rng.choice([1024, 2048, 4096, 4096]),
                "N": rng.choice([1024, N_EMBD, N_EMBD, 16 * rng.randint(30, 160)]), "r": rng.choice([8, 16, 16, 32, 64]),
                "adapters": log(1, 64), "group": rng.choice([1, log(1, 512)]) if M <= 256 else log(64, 1024), "lens": lens,
                "gate": rng.random() < 0.5}
    H, Hkv = rng.choice([(16, 2), (16, 2), (16, 2), (16, 4), (8, 2), (8, 1), (4, 4)])
    case = {"kind": kind, "B": 1, "page": rng.choice([16, 32, 64, 128, 256]), "n_lo": 1, "n_hi": 1, "past_lo": 0,
            "past_hi": 0, "lens": lens, "H": H, "Hkv": Hkv, "chunks": 0, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]),
            "bias": rng.choice([0.0, 0.0, 0.0, 8.0]), "prefix": 0, "gate": rng.random() < 0.4,
            "pad": rng.choice([0, 0, rng.randint(1, 40)])}
    form = rng.choice(["decode", "decode", "verify", "chunk", "chunk", "mixed"])
    if form in ("decode", "verify"):
        case["n_hi"] = 1 if form == "decode" else rng.randint(2, 4)
        case["n_lo"] = rng.randint(1, case["n_hi"])
        case["B"] = log(1, 128)
        most = min(131000, 2000000 // case["B"])
    elif form == "mixed":
        case["B"], case["chunks"] = rng.randint(3, 32), log(64, 512)
        most = 8000
    else:
        case["B"] = rng.choice([1, 1, rng.randint(2, 8)])
        case["n_hi"] = log(20, 2048 // case["B"] if case["B"] < 4 else 900)
        case["n_lo"] = log(5, case["n_hi"])
        case["prefix"] = rng.choice([0, 0, log(16, 1000)])
        most = 30000
    case["past_hi"] = log(16, most) if rng.random() < 0.85 else 0
    case["past_lo"] = rng.randint(0, case["past_hi"])
    dense = case["B"] * max(case["n_hi"], case["chunks"]) * H
    case["past_hi"] = max(0, min(case["past_hi"], int(min(MOST_DENSE, MOST_PAIRS) // dense) - max(case["n_hi"], case["chunks"])))
    case["past_lo"] = min(case["past_lo"], case["past_hi"])
    return case


# ------------------------------------------------------------------ lengths --

def _attn_lens(case):
    """(new, past, prefix) of every request."""
    r = random.Random(case["lens"])
    new = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["B"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["B"])]
    if case["chunks"]:  # two prompt chunks among the others
        for b in r.sample(range(case["B"]), min(2, case["B"])):
            new[b] = case["chunks"] - r.randint(0, case["chunks"] // 8)
    prefix = [r.randint(case["prefix"] // 2, case["prefix"]) if r.random() < 0.8 else 0 for _ in range(case["B"])]
    if case["lens"] % 3 == 0 and case["B"] > 4:  # a place of the batch without tokens in this step
        new[r.randrange(case["B"])] = 0
    return new, past, prefix


def _plan_lens(case):
    """(n_new, n_past) of every request: decoding ones, some prompt chunks, some that end, some idle."""
    r = random.Random(case["lens"])
    B, most = case["B"], case["W"] * case["page"]
    new = [1 if r.random() < 0.95 else 0 for _ in range(B)]
    left = case["tokens"] - sum(new)
    while left > 0 and B:
        n = min(left, r.randint(1, 1 + max(1, case["tokens"] // 6)))
        new[r.randrange(B)] += n
        left -= n
    for b in r.sample(range(B), min(case["ended"], B)):
        new[b] = -1
    past = [r.randint(0, most) if r.random() < 0.02 else r.randint(0, max(0, most - max(0, n)) // 2) for n in new]
    return new, past


def _pages(n, page):
    return (n + page - 1) // page


def _ids(case):
    """Adapter of every token: `group` neighbours share one, some have none."""
    r = random.Random(case["lens"])
    ids = []
    while len(ids) < case["M"]:
        n = max(1, case["group"] - r.randint(0, case["group"] // 3))
        ids += [r.randrange(case["adapters"]) if r.random() < 0.9 else -1] * n
    return ids[:case["M"]]


# ------------------------------------------------------------------ inputs --

def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


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


def _pool(gen, pages, page, Hkv):
    rows = torch.empty((pages * page, Hkv * ROW), dtype=torch.uint8, device="cuda")
    for r in range(0, pages * page, 65536):
        n = min(65536, pages * page - r)
        rows[r:r + n] = _q4_0(_randn(gen, n, Hkv * D))
    return rows.view(pages, page, Hkv, ROW)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    if case["kind"] == "plan":
        new, past = _plan_lens(case)
        B, W, page = case["B"], case["W"], case["page"]
        held = sum(min(_pages(p, page), W) for p in past)
        wanted = sum(_pages(p + max(n, 0), page) - _pages(p, page) for n, p in zip(new, past))
        free = wanted * 9 // 10 + 8  # now and then a request has to wait
        ids = torch.randperm(held + free, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
        count = torch.tensor([min(_pages(p, page), W) for p in past], device="cuda")
        at = torch.arange(W, device="cuda")[None, :] < count[:, None]
        table[at] = ids[free:]
        head = int(torch.randint(0, held + free, (1,), generator=gen, device="cuda"))
        ring = torch.full((held + free,), -1, dtype=torch.int32, device="cuda")
        ring[(head + torch.arange(free, device="cuda")) % (held + free)] = ids[:free]
        T = case["tokens"] + 5
        s |= {"state": _i32([head, free, 0, 0]), "ring": ring, "table": table, "n_past": _i32(past), "n_new": _i32(new),
              "state_out": _i32([0] * 4), "n_past_out": _i32([0] * B), "q_start": _i32([0] * (B + 1)),
              "kv_len": _i32([0] * B), "slots": torch.zeros(T, dtype=torch.int64, device="cuda"),
              "pos": torch.zeros(4 * T, dtype=torch.int32, device="cuda")}
    elif case["kind"] == "attn":
        new, past, prefix = _attn_lens(case)
        B, page, H, Hkv = case["B"], case["page"], case["H"], case["Hkv"]
        kv = [n + p for n, p in zip(new, past)]
        used = [_pages(k, page) for k in kv]
        W, total, T = max(1, max(used)), max(1, sum(used)), sum(new) + case["pad"]
        T = max(1, T)
        s["k"], s["v"] = _pool(gen, total, page, Hkv), _pool(gen, total, page, Hkv)
        table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
        at = torch.arange(W, device="cuda")[None, :] < torch.tensor(used, device="cuda")[:, None]
        table[at] = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)[:sum(used)]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s |= {"table": table, "q_start": _i32(starts), "kv_len": _i32(kv), "max_q": max(1, max(new)), "max_kv": max(kv),
              "prefix": _i32(prefix) if case["prefix"] else None, "q": _randn(gen, T, H, D),
              "gate": _randn(gen, T, H, D) if case["gate"] else None,
              "out": torch.zeros((T, H, D), dtype=torch.float32, device="cuda")}
        s["ws"] = torch.empty(SCRATCH, dtype=torch.uint8, device="cuda")
    else:
        M, K, N, r = case["M"], case["K"], case["N"], case["r"]
        s["x"], s["base"] = _randn(gen, M, K), _randn(gen, M, N)
        s["gate"] = _randn(gen, M, K) if case["gate"] else None
        s["a"] = (_randn(gen, case["adapters"], r, K) * K ** -0.5).half()
        s["b"] = (_randn(gen, case["adapters"], N, r) * r ** -0.5).half()
        s["scale"] = torch.rand(case["adapters"], generator=gen, device="cuda") * 1.5 + 0.5
        s["ids"] = _i32(_ids(case))
        s["out"] = torch.zeros((M, N), dtype=torch.float32, device="cuda")
    return s


# ------------------------------------------------------------ plain forms --

def _plan_plain(s):
    case = s["case"]
    page, W, T, n = case["page"], case["W"], s["slots"].shape[0], s["ring"].shape[0]
    table, past = s["table"].long(), s["n_past"].long().clamp(min=0)
    new, ended = s["n_new"].long().clamp(min=0), s["n_new"] < 0
    B, dev = past.shape[0], past.device
    head, count = s["state"][0].long(), s["state"][1].long()
    have = torch.div(past + page - 1, page, rounding_mode="floor")
    # pages of ended requests go behind the free ones
    cols = torch.arange(W, device=dev)
    gone = ended[:, None] & (cols[None, :] < have[:, None])
    rank = torch.cumsum(gone.reshape(-1).long(), 0) - 1
    to = torch.where(gone.reshape(-1), (head + count + rank) % n, torch.full_like(rank, n))
    ring = torch.cat([s["ring"], s["ring"].new_zeros(1)]).scatter(0, to, s["table"].reshape(-1))[:n]
    count = count + gone.sum()
    # pages of new tokens leave in the order of the requests
    end = torch.cumsum(new, 0)
    fits = ~ended & (past + new <= W * page) & (end <= T)
    need = torch.where(fits, torch.div(past + new + page - 1, page, rounding_mode="floor") - have, torch.zeros_like(have))
    upto = torch.cumsum(need, 0)
    ok = fits & ((need == 0) | (upto <= count))
    popped = torch.where(ok & (need > 0), upto, torch.zeros_like(upto)).max()
    k = cols[None, :] - have[:, None]
    fresh = ok[:, None] & (k >= 0) & (k < need[:, None])
    page_id = ring[(head + (upto - need)[:, None] + k.clamp(min=0)) % n].long()
    table = torch.where(fresh, page_id, table)
    # tokens
    start = end - new
    q_start = torch.cat([start.new_zeros(1), end]).clamp(max=T)
    t = torch.arange(T, device=dev)
    b = torch.searchsorted(end, t, right=True).clamp(max=B - 1)
    p = past[b] + t - start[b]
    live = (t < end[-1]) & ok[b]
    p = torch.where(live, p, torch.zeros_like(p))
    slot = table[b, torch.div(p, page, rounding_mode="floor").clamp(max=W - 1)] * page + p % page
    slot = torch.where(live, slot, torch.full_like(slot, -1))
    kv_len = torch.where(ok, past + new, torch.zeros_like(past))
    n_past = torch.where(ok, past + new, torch.where(ended, torch.zeros_like(past), past))
    state = torch.stack([(head + popped) % n, count - popped, (~ok & ~ended).sum(), q_start[-1]])
    i32 = torch.int32
    return {"table": table.to(i32), "ring": ring, "state": state.to(i32), "n_past": n_past.to(i32),
            "q_start": q_start.to(i32), "kv_len": kv_len.to(i32), "slots": slot, "pos": p.to(i32).repeat(4)}


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


def _attn_plain(s):
    case = s["case"]
    H, Hkv, page, L, nq = case["H"], case["Hkv"], case["page"], s["max_kv"], s["max_q"]
    G, T, B, dev = H // Hkv, s["q"].shape[0], case["B"], s["q"].device
    start, kv = s["q_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    i, j = torch.arange(nq, device=dev), torch.arange(max(L, 1), device=dev)
    rows = (start[:-1, None] + i).clamp(max=T - 1)                       # (B, nq)
    q = _q8_0(s["q"])[rows].reshape(B, nq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, nq * G, D)
    pid = s["table"].long()[:, torch.div(j, page, rounding_mode="floor")]  # (B, L)
    at = pid.clamp(min=0) * page + j % page
    k = _dequant(s["k"].reshape(-1, Hkv, ROW)[at]).transpose(1, 2).contiguous()  # (B, Hkv, L, D)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous())
    del k
    x = x.mul_(D ** -0.5).reshape(B, Hkv, nq, G, -1)
    if case["cap"]:
        x = x.div_(case["cap"]).tanh_().mul_(case["cap"])
    pos = kv[:, None] - n[:, None] + i                                   # (B, nq)
    if case["bias"]:
        far = (pos[:, :, None] - j).abs().float()
        slope = _slopes(H, case["bias"], dev).float().reshape(1, Hkv, 1, G, 1)
        x = x.sub_(slope * far[:, None, :, None, :])
    see = torch.maximum(pos + 1, s["prefix"].long()[:, None]) if s["prefix"] is not None else pos + 1
    see = torch.minimum(see, kv[:, None])
    dead = ((j >= see[:, :, None]) | (pid < 0)[:, None, :])[:, None, :, None, :]
    x = x.masked_fill_(dead, -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    l = x.sum(-1, keepdim=True)
    v = _dequant(s["v"].reshape(-1, Hkv, ROW)[at]).transpose(1, 2).contiguous()
    o = torch.matmul(x.reshape(B, Hkv, nq * G, -1), v).reshape(B, Hkv, nq, G, D)
    o = torch.where(l > 0, o / l, torch.zeros_like(o)).permute(0, 2, 1, 3, 4).reshape(B, nq, H, D)
    live = i < n[:, None]
    out = torch.zeros_like(s["q"])
    out[rows[live]] = o[live]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"])
    return out


def _lora_plain(s):
    x = s["x"] if s["gate"] is None else s["x"] * torch.sigmoid(s["gate"])
    A, N, r = s["b"].shape
    K = x.shape[1]
    ids = s["ids"].long()
    # every adapter's products of every token, then the token's own
    t = torch.matmul(x, s["a"].float().reshape(A * r, K).t()).reshape(-1, A, r)
    own_id = torch.arange(A, device=x.device)[None, :] == ids[:, None]
    t = torch.where(own_id[:, :, None], t * s["scale"][None, :, None], torch.zeros_like(t))
    return s["base"] + torch.matmul(t.reshape(-1, A * r), s["b"].float().transpose(1, 2).reshape(A * r, N))


def run(s):
    kind = s["case"]["kind"]
    if own:
        sqa = _package()
        if kind == "plan":
            sqa.paged_plan(s["state"], s["ring"], s["table"], s["n_past"], s["n_new"], s["case"]["page"],
                           state_out=s["state_out"], n_past_out=s["n_past_out"], q_start=s["q_start"],
                           kv_len=s["kv_len"], slots=s["slots"], pos=s["pos"])
            return {"table": s["table"], "ring": s["ring"], "state": s["state_out"], "n_past": s["n_past_out"],
                    "q_start": s["q_start"], "kv_len": s["kv_len"], "slots": s["slots"], "pos": s["pos"]}
        if kind == "attn":
            return sqa.paged_attn(s["q"], s["k"], s["v"], s["table"], s["q_start"], s["kv_len"], s["max_q"],
                                  softcap=s["case"]["cap"], max_bias=s["case"]["bias"], prefix=s["prefix"],
                                  gate=s["gate"], out=s["out"], workspace=s["ws"])
        return sqa.lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], scale=s["scale"], gate=s["gate"], out=s["out"])
    return _plan_plain(s) if kind == "plan" else _attn_plain(s) if kind == "attn" else _lora_plain(s)


def _package():
    import __graft_entry__ as graft

    return graft.load_package()


# ------------------------------------------------------------------- floors --

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    if case["kind"] == "plan":
        new, past = _plan_lens(case)
        moved = sum(_pages(p, case["page"]) if n < 0 else _pages(p + n, case["page"]) - _pages(p, case["page"])
                    for n, p in zip(new, past))
        return {"bytes": 20 * len(new) + 24 * (case["tokens"] + 5) + 8 * moved, "flops": 0}
    if case["kind"] == "lora":
        M, K, N, r = case["M"], case["K"], case["N"], case["r"]
        ids = [i for i in _ids(case) if i >= 0]
        return {"bytes": 4 * M * (K * (2 if case["gate"] else 1) + 2 * N) + 2 * r * (K + N) * len(set(ids)) + 4 * M,
                "flops": 2 * r * (K + N) * len(ids)}
    new, past, prefix = _attn_lens(case)
    pairs = 0
    for n, p, f in zip(new, past, prefix):
        f = min(f, n + p) if case["prefix"] else 0
        low = min(n, max(0, f - p))  # tokens that see the prefix and nothing behind it
        pairs += low * f + sum(range(p + low + 1, p + n + 1))
    keys = sum(n + p for n, p in zip(new, past) if n)
    rows = sum(new) * case["H"]
    return {"bytes": keys * case["Hkv"] * 2 * ROW + rows * D * 4 * (3 if case["gate"] else 2) + 12 * case["B"] +
            4 * keys // case["page"], "flops": 4 * D * pairs * case["H"]}


# ------------------------------------------------- definitions in 64 bits --

def _exact_attn(case, s):
    new, past, prefix = _attn_lens(case)
    H, Hkv, page = case["H"], case["Hkv"], case["page"]
    G, out, t0 = H // Hkv, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    blocks = s["q"].reshape(-1, 32)  # q8_0 is defined by its float32 operations
    top = blocks.abs().max(1).values
    code = torch.where(top[:, None] > 0, (blocks * (torch.full_like(top, 127.0) / top)[:, None]).round(), 0 * blocks)
    q8 = (code.double() * (top / 127.0).to(torch.float16).double()[:, None]).reshape(s["q"].shape)

    def values(pool, pages, n, h):
        raw = pool[pages.long()][:, :, h].reshape(-1, ROW)[:n].reshape(n, 8, 18)
        d = raw[:, :, :2].contiguous().view(torch.float16).double()
        return torch.cat([(raw[:, :, 2:] & 15).double() - 8, (raw[:, :, 2:] >> 4).double() - 8], 2).mul_(d).reshape(n, D)

    nl2 = 2 ** int(math.floor(math.log2(H)))
    for b in range(case["B"]):
        n, L = new[b], new[b] + past[b]
        if n:
            pages = s["table"][b, :_pages(L, page)]
            j = torch.arange(L, device="cuda", dtype=torch.float64)
            for h in range(Hkv):
                K, V = values(s["k"], pages, L, h), values(s["v"], pages, L, h)
                step = max(1, int(3e8 // L))
                for g in range(G):
                    hq = h * G + g
                    m = 2.0 ** (-case["bias"] * (hq + 1) / nl2) if hq < nl2 else \
                        2.0 ** (-case["bias"] / 2 * (2 * (hq - nl2) + 1) / nl2)
                    for i0 in range(0, n, step):
                        i1 = min(n, i0 + step)
                        x = q8[t0 + i0:t0 + i1, hq] @ K.t() / 16.0
                        if case["cap"]:
                            x = case["cap"] * torch.tanh(x / case["cap"])
                        p = torch.arange(past[b] + i0, past[b] + i1, device="cuda", dtype=torch.float64)[:, None]
                        if case["bias"]:
                            x = x - m * (p - j).abs()
                        x = torch.where((j <= p) | (j < (prefix[b] if case["prefix"] else 0)), x, torch.full_like(x, -math.inf))
                        out[t0 + i0:t0 + i1, hq] = torch.softmax(x, 1) @ V
        t0 += n
    return out if s["gate"] is None else out / (1 + torch.exp(-s["gate"].double()))


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers, compared as they are
    s = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, s)
    x = s["x"].double()
    if s["gate"] is not None:
        x = x / (1 + torch.exp(-s["gate"].double()))
    out = s["base"].double()
    for i in sorted({i for i in _ids(case) if i >= 0}):
        at = s["ids"] == i
        out[at] += s["scale"][i].double() * ((x[at] @ s["a"][i].double().t()) @ s["b"][i].double().t())
    return out
