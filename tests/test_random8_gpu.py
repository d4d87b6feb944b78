"""Seeded random batches of paged_attn_fp8_fwd against attention in 64 bits.

The grids of test_attn_fp8_gpu.py cover the edges one at a time; this draws whole
batches (requests, tokens and keys of each, with more tokens than keys here and there,
head groups, head size, windows, causality, pages, layouts, types, the hints that choose
kernel and split), so that combinations nobody thought of meet the same tolerances. Every
case prints itself before it runs.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

from fp8_cases import assert_close, attend, make_cache, queries, reference, workspace

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def draw(seed):
    rng = random.Random(seed)
    many = rng.random() < 0.2  # requests, more than a wave has lanes
    R = rng.randint(65, 150) if many else rng.randint(1, 9)
    D = rng.choice([64, 128, 256])
    G = rng.choice([1, 2, 3, 4, 5, 8, 12, 17, 64])
    Hkv = rng.choice([1, 1, 2, 3, 4, 8]) if G <= 8 else rng.choice([1, 2])
    longest = rng.choice([1, 1, 4, 20]) if many else rng.choice([1, 2, 8, 40, 300, 900])
    q_lens = [rng.choice([0, 1, 1, rng.randint(1, longest)]) for _ in range(R)]
    if rng.random() < 0.3:
        q_lens = [min(n, 1) for n in q_lens]
    most = rng.choice([20, 200, 700]) if many else rng.choice([20, 300, 2000, 6000])
    lens = [rng.randint(0, most) + (n if rng.random() < 0.8 else 0) for n in q_lens]
    causal = rng.random() < 0.8
    window = rng.choice([0, 0, 1, 17, rng.randint(2, 300), 1500]) if causal else 0
    return dict(q_lens=q_lens, lens=lens, D=D, Hq=G * Hkv, Hkv=Hkv, causal=causal, window=window,
                block=rng.choice([16, 32, 48, 128, 816]), layout=rng.choice(["NHD", "HND"]),
                dtype=rng.choice([BF, BF, HF]), max_q=rng.choice([None, None, 1, 17, 4096]),
                max_len=rng.choice([None, None, 1 << 17]), width=rng.choice([None, 1 << 13]))


@pytest.mark.parametrize("seed", range(120))
def test_random_batch(seed):
    c = draw(seed)
    print(f"random batch {seed}: {c}", flush=True)
    D, q_lens = c["D"], c["q_lens"]
    cache = make_cache(c["lens"], Hkv=c["Hkv"], D=D, block=c["block"], seed=seed, layout=c["layout"],
                       width=c["width"])
    q = queries(sum(q_lens) + 2, c["Hq"], D, c["dtype"], seed)
    scale, ws = 1 / math.sqrt(D), workspace(D)
    kw = dict(window=c["window"], causal=c["causal"])
    longest = max(q_lens) if c["max_q"] is None else c["max_q"]
    out = attend(cache, q, q_lens, scale, max_q=longest, max_len=c["max_len"], ws=ws, **kw)
    # P may be rounded once wherever the kernel of many rows may take a request of bf16.
    single = c["dtype"] == BF and longest * c["Hq"] // c["Hkv"] > 16
    want, tol = reference(q, cache.keys, q_lens, scale, single=single, **kw)
    assert out[-2:].isnan().all()
    assert_close(out[:-2], want[:-2], tol[:-2])
    again = attend(cache, q, q_lens, scale, max_q=longest, max_len=c["max_len"], ws=ws, **kw)
    assert torch.equal(out[:-2], again[:-2])
