"""paged_attn_fp8_fwd: how 128-row units share the work-groups, at its ends."""

from __future__ import annotations

import math

import pytest
import torch

from fp8_cases import (assert_close, attend, make_cache, queries, reference, starts_of, workspace)
from pth_flash_attn import capi, ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
MANY = 17  # max_query_len: the kernel of 128-row units


@pytest.mark.parametrize("window", [0, 500])
@pytest.mark.parametrize(("D", "Hq", "Hkv"), [(64, 2, 2), (128, 6, 2), (256, 4, 1)])
def test_more_tokens_than_keys(D, Hq, Hkv, window):
    """Tokens without a place among the keys, many of them, beside requests of long
    prefixes: these rows are 0, the others as ever, and keys are cut over work-groups."""
    q_lens, lens = [6000, 40, 3000, 2], [100, 9000, 0, 5000]
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, seed=D)
    q = queries(sum(q_lens), Hq, D, BF, D)
    scale, ws = 1 / math.sqrt(D), workspace(D)
    out = attend(c, q, q_lens, scale, window=window, max_q=MANY, ws=ws)
    assert capi.AttnLib().last_kernel() == "f8_wide"
    assert not ws.isnan().all()  # sums of cut units
    assert not out[:5900].any() and not out[6040:9040].any()
    want, tol = reference(q, c.keys, q_lens, scale, window=window, single=True)
    assert_close(out, want, tol)


def sampled(q, keys, q_lens, scale, tokens, *, window=0, causal=True, single):
    """(rows of q, out, tolerance) of some tokens (request, place), each as a request
    of its own whose keys end where its sight does."""
    starts = [sum(q_lens[:r]) for r in range(len(q_lens))]
    rows = torch.tensor([starts[r] + t for r, t in tokens], device=q.device)
    ends = [max(len(keys[r][0]) - (q_lens[r] - 1 - t if causal else 0), 0) for r, t in tokens]
    own = [tuple(x[:e] for x in keys[r]) for (r, _), e in zip(tokens, ends)]
    out, tol = reference(q[rows], own, [1] * len(tokens), scale, window=window, causal=causal,
                         single=single)
    return rows, out, tol


@pytest.mark.parametrize(("causal", "window"), [(True, 0), (True, 9000), (True, 700), (False, 0)])
@pytest.mark.parametrize(("D", "Hq", "Hkv", "dtype"), [(64, 32, 8, BF), (128, 32, 8, BF),
                                                       (128, 32, 8, HF), (256, 16, 4, BF)])
def test_long_units_left_whole(D, Hq, Hkv, dtype, causal, window):
    """Units of up to 10,300 keys that no work-group shares: by length over requests
    alone and behind prefixes, and over more keys than the addresses of 64 tiles, twice.
    Nothing is written to the workspace then."""
    q_lens, lens = [2200, 10300, 150, 0, 1500, 33], [2200, 10300, 5000, 40, 7000, 20]
    c = make_cache(lens, Hkv=Hkv, D=D, block=48, seed=D)
    q = queries(sum(q_lens), Hq, D, dtype, D + 1)
    scale, ws = 1 / math.sqrt(D), workspace(D)
    out = attend(c, q, q_lens, scale, window=window, causal=causal, ws=ws)
    assert capi.AttnLib().last_kernel() == "f8_wide"
    assert ws.isnan().all()
    assert not out.isnan().any()
    gen = torch.Generator().manual_seed(D)
    per = 128 * Hkv // Hq  # tokens of a unit
    tokens = [(1, t) for t in (0, 1, per - 1, per, 4095, 4096, 8191, 8192, 10299)]
    tokens += [(1, int(t)) for t in torch.randint(0, 10300, (14,), generator=gen)]
    tokens += [(1, 10299 - int(t)) for t in torch.randint(0, 1500, (5,), generator=gen)]
    for r in (0, 2, 4, 5):
        tokens += [(r, t) for t in (0, q_lens[r] - 1)]
        tokens += [(r, int(t)) for t in torch.randint(0, q_lens[r], (4,), generator=gen)]
    rows, want, tol = sampled(q, c.keys, q_lens, scale, tokens, window=window, causal=causal,
                              single=dtype == BF)
    assert_close(out[rows], want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("tokens", [1, 20])
def test_lengths_near_2_to_31(D, tokens):
    """One request of as many keys as a position may count, over pages that repeat: its
    table's last entries are the tensor's. All weights are equal and all values of a
    column the same power of two, so that sums and outputs are exact."""
    block, reach = 816, 1 << 31
    width = -(-reach // block)
    codes = torch.full((2, 2, block, 1, D), 0x7F, dtype=torch.uint8, device="cuda")
    column = torch.exp2(torch.arange(D, device="cuda") % 7 - 3.0)
    column = torch.where(torch.arange(D, device="cuda") % 2 == 0, column, -column)
    codes[1] = column.to(torch.float8_e4m3fn).view(torch.uint8)
    scale = torch.full((2, 2, block // 16, 1), 127, dtype=torch.uint8, device="cuda")
    k, v = codes[:, 0].view(torch.float8_e4m3fn), codes[:, 1].view(torch.float8_e4m3fn)
    table = torch.ones(1, width, dtype=torch.int32, device="cuda")
    lens = torch.tensor([reach - 1], dtype=torch.int32, device="cuda")
    q = torch.zeros(tokens, 1, D, dtype=BF, device="cuda")
    out = torch.full_like(q, math.nan)
    ops.paged_attn_fp8_fwd(out, q, k, v, scale[0], scale[1], table, lens, starts_of([tokens]),
                           tokens, reach - 1, 0.125, workspace(D))
    assert capi.AttnLib().last_kernel() == ("f8_rows" if tokens == 1 else "f8_wide")
    assert torch.equal(out, column.to(BF).expand_as(out))
