"""Values near the ends of a type's range through the 128-row kernel, whose
running maximum may lag behind the scores: what it keeps must not leave 32
bits where the formula's sums with the exact maximum do not."""

from __future__ import annotations

import math

import pytest
import torch

from paged16_cases import DEV, assert_close, cross, make_cache, queries, reference
from pth_flash_attn import capi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens", [[128], [4096 + 64]])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("up", [2.875, 7.875, 8.125])
def test_large_values_behind_a_lagging_maximum(D, lens, up, dtype):
    """The first 64 keys' scores are 0 and the others' `up` powers of two above,
    whole tiles of each. V is one power of two whose sum over all keys, each of
    weight 1, is less than 2^128 (2^113 x 2^13), so the output is it again."""
    big = 2.0**121 if lens == [128] else 2.0**114
    if dtype == torch.float16:
        big = 32768.0
    c = make_cache(lens, Hkv=1, D=D, block=16, dtype=dtype, seed=1)
    L = lens[0]
    k = torch.zeros(L, 1, D, dtype=dtype, device=DEV)
    k[64:, 0, 0] = up
    v = torch.full((L, 1, D), big, dtype=dtype, device=DEV)
    pos = torch.arange(L, device=DEV)
    page = c.table[0].long()[pos // 16]
    c.k[page, pos % 16], c.v[page, pos % 16] = k, v
    q = torch.zeros(40, 1, D, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    got = cross(c, q, [40], math.log(2.0))
    assert capi.AttnLib().last_kernel() == "p16_wide"
    assert_close(got, *reference(q, [(k, v)], [40], math.log(2.0)))
