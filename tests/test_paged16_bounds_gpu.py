"""Attention over a paged 16-bit cache where its integer tensors hold anything:
requests whose own are in order keep their results, and nothing else is
written; and where out and q are columns of one buffer."""

from __future__ import annotations

import pytest
import torch

from paged16_cases import DEV, assert_close, cross, decode, make_cache, queries, reference

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
