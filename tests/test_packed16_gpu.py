"""A decode step in which some requests bring no token: build_step_tables packs
the others' rows, and cross_attn_fwd over the decoder's own cache attends from
them."""

from __future__ import annotations

import math

import pytest
import torch

from paged16_cases import DEV, assert_close, reference, workspace
from pth_flash_attn import ops
from pth_flash_attn.cache import paged16_views

pytestmark = pytest.mark.gpu
BF, BLOCK = torch.bfloat16, 16
I32 = dict(dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("new", [[0, 1, 1, 0, 1], [1, 0, 0, 1, 1], [1, 1, 1, 1, 1],
                                 [0, 0, 0, 0, 0]])
def test_packed_decode_step(new, D):
    Hq, Hkv, R, T = 8, 2, 5, 7  # two rows of padding or more
    ctx = [40, 15, 16, 300, 0]
    gen = torch.Generator(device=DEV).manual_seed(D)
    kv = torch.full((40, 2, BLOCK, Hkv, D), math.nan, dtype=BF, device=DEV)
    k_cache, v_cache = paged16_views(kv)
    table, at, keys = torch.zeros(R, 24, **I32), 40, []
    for r, n in enumerate(ctx):
        old = torch.randn(2, n, Hkv, D, generator=gen, device=DEV).to(BF)
        for j in range(-(-n // BLOCK)):
            at -= 1
            table[r, j] = at
            part = old[:, j * BLOCK : (j + 1) * BLOCK]
            kv[at, :, : part.shape[1]] = part
        keys.append((old[0], old[1]))
    free = torch.tensor([i for i in range(1, 40) if i not in set(table.flatten().tolist())], **I32)
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=gen, device=DEV).to(BF)
    q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
    slots = torch.zeros(T, dtype=torch.int64, device=DEV)
    seq, starts, pool = (torch.zeros(n, **I32) for n in (R, R + 1, 2))
    ops.build_step_tables(table, slots, seq, starts, pool, torch.tensor(ctx, **I32),
                          torch.tensor(new, **I32), free, torch.zeros(2, **I32), BLOCK)
    ops.reshape_and_cache_16bit(k, v, k_cache, v_cache, slots)
    out = torch.full((T, Hq, D), 7.0, dtype=BF, device=DEV)
    ops.cross_attn_fwd(out, q, k_cache, v_cache, table, seq, starts, 1, 24 * BLOCK, 0.1,
                       workspace(D))
    assert seq.tolist() == [c + n for c, n in zip(ctx, new)]
    t = 0
    for r, n in enumerate(new):
        if n:
            keys[r] = (torch.cat([keys[r][0], k[t : t + 1]]), torch.cat([keys[r][1], v[t : t + 1]]))
            t += 1
    assert_close(out[:t], *reference(q[:t], keys, new, 0.1, pair=True))
    assert (out[t:] == 7.0).all()
