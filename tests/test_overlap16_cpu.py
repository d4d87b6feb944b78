"""Which outputs of the 16-bit cache's ops may lie in one buffer with an input,
against the sets of addresses: every view that shares no element is taken, every
other one but q itself is refused. (CPU tensors: a call that passes the checks
is refused for its device.)"""

from __future__ import annotations

import itertools
import random

import pytest
import torch

from pth_flash_attn import ops
from pth_flash_attn.cache import paged16_views

pytestmark = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
BF, I32 = torch.bfloat16, torch.int32
ON_GPU = "computes on CUDA tensors only"
SHARED = "out must be q itself or share no memory with it"


def attend(out, q, cross):
    R = q.shape[0]
    k, v = paged16_views(torch.zeros(3, 2, 16, 1, q.shape[2], dtype=BF))
    table, lens, ws = torch.zeros(R, 2, dtype=I32), torch.ones(R, dtype=I32), torch.zeros(64)
    with pytest.raises(RuntimeError) as e:
        if cross:
            ops.cross_attn_fwd(out, q, k, v, table, lens, torch.arange(R + 1, dtype=I32), 1, 20,
                               0.1, ws)
        else:
            ops.paged_decode_fwd(out, q, k, v, table, lens, 20, 0.1, ws)
    return str(e.value)


@pytest.mark.parametrize("cross", [False, True])
def test_out_shifted_against_q_is_refused(cross):
    buf = torch.zeros(5, 4, 64, dtype=BF)
    for out, q in ((buf[1:], buf[:-1]), (buf[:-1], buf[1:]), (buf[:, 1:], buf[:, :-1]),
                   (buf[:4], buf.flatten()[8:][: 4 * 256].view(4, 4, 64)),
                   (buf[:4, :2], buf[:2].view(4, 2, 64))):
        assert SHARED in attend(out, q, cross)


@pytest.mark.parametrize("cross", [False, True])
def test_out_beside_q_is_taken(cross):
    fused = torch.zeros(5, 12, 64, dtype=BF)
    pairs = torch.zeros(5, 4, 2, 64, dtype=BF)
    turned = torch.zeros(4, 5, 64, dtype=BF).transpose(0, 1)
    wide = torch.zeros(5, 12, 64, dtype=BF)
    for out, q in ((fused[:, 4:8], fused[:, :4]), (fused[:, :4], fused[:, 8:]),
                   (pairs[:, :, 1], pairs[:, :, 0]), (fused[:, :4], fused[:, :4]),
                   (turned, turned), (fused[:1, 2:6], fused[2:3, 4:8]),
                   (wide[:, 1:9:2], wide[:, 0:8:2]), (wide[:, 8:], wide[:, 0:8:2])):
        assert ON_GPU in attend(out, q, cross)


def addresses(offset, shape, strides):
    return {offset + sum(i * s for i, s in zip(at, strides))
            for at in itertools.product(*map(range, shape))}


def test_random_views_of_one_buffer():
    """Token and head strides of every order and size; only views that take too
    many steps to tell apart could be refused needlessly, and none here does."""
    rng, seen = random.Random(3), {True: 0, False: 0}
    buf = torch.zeros(6000, dtype=BF)
    while sum(seen.values()) < 400:
        T, H = rng.randint(1, 4), rng.randint(1, 4)
        views = []
        for _ in range(2):
            inner = rng.choice([64, 64, 65, 80, 128, 192, 320])
            outer = rng.choice([inner * (H if rng.random() < 0.5 else T), 64, 256, 400, 650, 1000])
            strides = (outer, inner, 1) if rng.random() < 0.7 else (inner, outer, 1)
            views.append((rng.choice([0, 1, 32, 64, 128, rng.randint(0, 1500)]), strides))
        shape = (T, H, 64)
        (a, sa), (b, sb) = views
        if rng.random() < 0.4:
            sb = sa
        if max(a + sum((n - 1) * s for n, s in zip(shape, sa)),
               b + sum((n - 1) * s for n, s in zip(shape, sb))) >= buf.numel():
            continue
        own = addresses(a, shape, sa)
        out, q = buf.as_strided(shape, sa, a), buf.as_strided(shape, sb, b)
        said = attend(out, q, False)
        if len(own) < T * H * 64:
            assert "out must not overlap itself" in said
            continue
        if "out must not overlap itself" in said:
            continue  # strides that do not nest
        same = a == b and all(x == y or n == 1 for n, x, y in zip(shape, sa, sb))
        shares = not same and bool(own & addresses(b, shape, sb))
        assert (SHARED if shares else ON_GPU) in said, (shape, views)
        seen[shares] += 1
    assert min(seen.values()) > 50


def write(k_cache, v_cache, key, value):
    with pytest.raises(RuntimeError) as e:
        ops.reshape_and_cache_16bit(key, value, k_cache, v_cache,
                                    torch.zeros(key.shape[0], dtype=torch.int64))
    return str(e.value)


def test_caches_that_share_memory_are_refused():
    """A token's key and value would go to one place, in no order."""
    kv = torch.zeros(6, 2, 16, 2, 64, dtype=BF)
    k, v = paged16_views(kv)
    key, value = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF)
    shifted = kv.flatten()[8:].as_strided(k[:5].shape, k.stride())
    for a, b in ((k, k), (k[1:], k[:-1]), (k[:, :8], k[:, 4:12]), (k[:3], k[2:5]),
                 (k[:5], shifted)):
        assert "k_cache and v_cache must share no memory" in write(a, b, key, value)
    # One cache for both is written by one tensor for both.
    assert "must share no memory" in write(k, k, key, value)
    assert ON_GPU in write(k, k, key, key)


def test_caches_of_one_buffer_are_taken():
    key, value = torch.zeros(3, 2, 64, dtype=BF), torch.zeros(3, 2, 64, dtype=BF)
    for layout, inner in (("NHD", (16, 2)), ("HND", (2, 16))):
        kv = torch.zeros(6, 2, *inner, 64, dtype=BF)
        assert ON_GPU in write(*paged16_views(kv, layout=layout), key, value)
    mixed = torch.zeros(6, 4096, dtype=BF)  # keys NHD, values HND
    assert ON_GPU in write(mixed[:, :2048].view(6, 16, 2, 64),
                           mixed[:, 2048:].view(6, 2, 16, 64).transpose(1, 2), key, value)
    beside = torch.zeros(6, 16, 2, 128, dtype=BF)  # a head's key and value side by side
    assert ON_GPU in write(beside[..., :64], beside[..., 64:], key, value)
    apart = torch.zeros(2, 6, 16, 2, 64, dtype=BF)
    assert ON_GPU in write(apart[0], apart[1], key, value)
