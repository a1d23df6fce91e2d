"""Seeded random batches: head layouts, lengths, holes, prefixes, options and workspaces in combinations
that nobody chose. Tolerances as in test_gpu_paged_attn and test_gpu_lora."""
import random

import pytest
import torch

import paged_ref
from test_gpu_lora import close as lora_close
from test_gpu_lora import inputs
from test_gpu_paged_attn import Batch, call, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(48))
def test_random_batches(sqa, orc, dev, seed):
    r = random.Random(seed)
    Hkv = r.choice([1, 1, 2, 2, 3, 4, 8])
    G = r.choice([1, 2, 3, 4, 5, 7, 8, 8, 9, 12, 16])
    B = r.choice([1, 2, 3, r.randint(4, 40), r.randint(41, 140)])
    long = max(1, int(2e6 / (B * Hkv * G * 40)))
    most = r.choice([1, 1, 2, 4, 40, 130])
    new = [r.choice([0, 1, 1, r.randint(1, most)]) for _ in range(B)]
    if not any(new):
        new[0] = 1
    past = [r.choice([0, r.randint(0, 70), r.randint(0, min(4000, long))]) for _ in range(B)]
    prefix = [r.choice([0, -1, r.randint(0, 100), 5000]) for _ in range(B)] if r.random() < 0.3 else None
    b = Batch(orc, 100 + seed, new, past, Hkv * G, Hkv, r.choice([16, 32, 64, 128]), prefix=prefix, pad=r.choice([0, 0, 5]),
              gate=r.random() < 0.4, scale_q=r.choice([1.0, 3.0]))
    for _ in range(r.choice([0, 0, 3])):  # pages that are not there
        b.table[r.randrange(B), r.randrange(b.table.shape[1])] = r.choice([-1, b.k.shape[0], 2 ** 31 - 1])
    if r.random() < 0.2:
        b.kv_len[r.randrange(B)] = r.choice([0, 1, -3])
    b.max_q = max(new) + r.choice([0, 0, 1, 30])
    opt = {"cap": r.choice([0.0, 0.0, 5.0, 50.0]), "bias": r.choice([0.0, 0.0, 2.0, 8.0])}
    want = b.ref(orc, fill=7.0, **opt)
    opt = {"softcap": opt["cap"], "max_bias": opt["bias"]}
    got = call(sqa, dev, b, fill=7.0, **opt)
    close(got, want)
    (a, kw) = b.args(dev)
    size = sqa.paged_attn_workspace_size(a[0], a[1], a[3], a[6])
    try:
        close(call(sqa, dev, b, fill=7.0, ws=max(16, int(size * r.random())), **opt), want)
    except sqa.SqaError as e:
        assert e.status == 3


@pytest.mark.parametrize("seed", range(32))
def test_random_adapters(sqa, dev, seed):
    r = random.Random(seed)
    M = r.choice([r.randint(1, 40), r.randint(41, 512), r.randint(513, 900)])
    K, N, rank, n = 256 * r.randint(1, 12), 16 * r.randint(1, 40), 8 * r.randint(1, 16), r.randint(1, 50)
    ids, run = [], r.choice([1, 1, 7, 100])
    while len(ids) < M:
        ids += [r.randint(-1, n)] * r.randint(1, run)
    d = inputs(dev, seed, M, K, N, rank, n, gate=r.random() < 0.5, ids=ids[:M])
    if r.random() < 0.3:
        d["scale"] = None
    want = paged_ref.lora(**d)
    out = d["base"] if r.random() < 0.3 else torch.empty_like(d["base"])
    lora_close(sqa.lora_add(**d, out=out), want)
