"""Attention over a paged 16-bit cache where its integer tensors hold anything:
requests whose own are in order keep their results, and nothing else is
written; and where out and q are columns of one buffer."""

from __future__ import annotations

import math

import pytest
import torch

from paged16_cases import (DEV, assert_close, cross, decode, make_cache, queries, reference,
                           workspace)
from pth_flash_attn import capi, ops, planner

pytestmark = pytest.mark.gpu
LOW = -(2**31)


@pytest.mark.parametrize("low", [LOW, LOW + 1, LOW + 200, -(2**30)])
@pytest.mark.parametrize("heads", [(2, 2), (8, 2)])
@pytest.mark.parametrize("n", [2, 40])
def test_starts_far_below_zero(n, heads, low):
    """A request that ends before it begins has no tokens, however far before
    (the difference of its starts passes 32 bits)."""
    Hq, Hkv = heads
    c = make_cache([300, 700, 64, 200], Hkv=Hkv, D=64, block=16, dtype=torch.bfloat16, seed=n)
    q = queries(200 + 4 * n, Hq, 64, torch.bfloat16, n)
    starts = torch.tensor([0, n, 200, low, low], dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 7.0)
    cross(c, q, [n], 0.125, max_q=n, out=out, starts=starts)
    torch.cuda.synchronize()
    q_lens = [n, 200 - n]
    want, tol = reference(q[:200], c.keys[:2], q_lens, 0.125, pair=n * Hq // Hkv <= 16)
    assert_close(out[:200], want, tol)
    assert (out[200:] == 7.0).all()


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [70, 0, 130]])
def test_out_beside_q_in_one_buffer(q_lens):
    c = make_cache([900, 40, 333], Hkv=2, D=128, block=16, dtype=torch.bfloat16, seed=3)
    T = sum(q_lens)
    fused = queries(T, 20, 128, torch.bfloat16, 3)
    before, q, out = fused.clone(), fused[:, :8], fused[:, 12:]
    if T == 3:
        decode(c, q, 0.1, out=out)
    else:
        cross(c, q, q_lens, 0.1, out=out)
    assert_close(out, *reference(before[:, :8], c.keys, q_lens, 0.1, pair=T == 3))
    assert torch.equal(fused[:, :12], before[:, :12])


def test_caches_of_one_buffer():
    """Keys NHD and values HND in one page, and one cache for both."""
    T, Hkv, D = 40, 2, 64
    key, value = (queries(T, Hkv, D, torch.bfloat16, i) for i in (1, 2))
    slots = torch.arange(16, 16 + T, device=DEV)
    table = torch.tensor([[1, 2, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([T], dtype=torch.int32, device=DEV)
    q, n = queries(1, 4, D, torch.bfloat16, 3), 16 * Hkv * D
    pages = torch.full((5, 2 * n), math.nan, dtype=torch.bfloat16, device=DEV)
    k = pages[:, :n].view(5, 16, Hkv, D)
    v = pages[:, n:].view(5, Hkv, 16, D).transpose(1, 2)
    for caches, values in (((k, v), value), ((k, k), key)):
        pages.fill_(math.nan)
        ops.reshape_and_cache_16bit(key, values, *caches, slots)
        out = torch.empty_like(q)
        ops.paged_decode_fwd(out, q, *caches, table, lens, T, 0.1, workspace(D))
        assert_close(out, *reference(q, [(key, values)], [1], 0.1, pair=True))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_workspace_of_the_planner_s_size_is_enough(D):
    """Both kernels with every work-group's slots in use leave what lies behind
    the workspace as it was; a float less is refused."""
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    floats = planner.paged16_workspace_floats(D=D, num_sms=cus)
    assert capi.AttnLib().lib.pth_attn_paged16_workspace_floats(D) == floats
    buf = torch.full((floats + 4096,), 7.0, device=DEV)
    for Hkv, n, lens in ((16, 1, [2100 + 7 * i for i in range(64)]), (8, 130, [1700] * 12)):
        c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=torch.bfloat16, seed=D)
        q_lens = [n] * len(lens)
        q = queries(sum(q_lens), 4 * Hkv, D, torch.bfloat16, D)
        out = cross(c, q, q_lens, D**-0.5, ws=buf[:floats])
        assert capi.AttnLib().last_kernel() == ("p16_rows" if n == 1 else "p16_wide")
        assert_close(out, *reference(q, c.keys, q_lens, D**-0.5, pair=n == 1))
        assert (buf[floats:] == 7.0).all()
        with pytest.raises(RuntimeError, match="ws must be 16-byte aligned and hold"):
            cross(c, q, q_lens, D**-0.5, ws=buf[: floats - 1])
