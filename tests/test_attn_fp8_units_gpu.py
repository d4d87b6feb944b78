"""paged_attn_fp8_fwd: how 128-row units share the work-groups, at its ends."""

from __future__ import annotations

import math

import pytest
import torch

from fp8_cases import assert_close, attend, make_cache, queries, reference, workspace
from pth_flash_attn import capi

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
