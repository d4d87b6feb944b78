"""The cosines and sines of rotary_embedding, read out with pairs (1, 0) in 32 bits."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from pth_flash_attn import ops, rotary

pytestmark = pytest.mark.gpu

# Off the exact value, of a sine: half a step of 32 bits of a value of at most 1, 2^-25;
# the angle's 32 bits of a turn, 2 pi 2^-33; and of the part that is added to the angle a,
# a z P(z) with z = a^2 <= 0.617, |P| <= 1 / 6, half a step each of z (2^-25, times
# a / 6), a z (2^-26, times 1 / 6), P (2^-27, times a z = 0.485), the part itself, at most
# 0.081 (2^-28), and of P's coefficients (1 / 6: 5.0e-9 times 0.485; 1 / 120: 4e-10 times
# 0.3). A cosine's part z z Q(z), |Q| <= 1 / 24, has less of each (2 z Q 2^-25, 2^-26 / 24,
# 2^-30 and 1.3e-9 times 0.38, 2^-31). The Taylor sums leave (pi / 4)^12 / 12! at most, and
# the angle's remainder of 1e-7 is of no more than 2^-24 relative where it is used.
BOUND = (2.0**-25 + 2 * math.pi * 2.0**-33 + 0.786 / 6 * 2.0**-25 + 2.0**-26 / 6 + 0.485 * 2.0**-27
         + 2.0**-28 + 5.0e-9 * 0.485 + 4e-10 * 0.3 + 1.2e-10)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_cosines_and_sines(interleaved, inverse):
    T, rot = 6000, 64
    rng = np.random.default_rng(1)
    pos = rng.integers(-(1 << 63), (1 << 63) - 1, T, dtype=np.int64)
    pos[:3000] = rng.integers(0, 1 << 20, 3000)
    turns, _ = rotary.rotary_turns(rot)
    x = torch.zeros(T, 1, rot, device="cuda")
    first = slice(0, rot, 2) if interleaved else slice(0, rot // 2)
    second = slice(1, rot, 2) if interleaved else slice(rot // 2, rot)
    x[..., first] = 1.0
    out, none = torch.empty_like(x), torch.empty(T, 0, rot, device="cuda")
    ops.rotary_embedding(out, none.clone(), x, none, torch.from_numpy(pos).cuda(), turns,
                         interleaved, 1.0, inverse)
    at = pos.view(np.uint64)[:, None] * turns.cpu().numpy().view(np.uint64)  # of 2^64 a turn
    angle = torch.from_numpy(at.view(np.int64).astype(np.float64) * (2 * math.pi / 2.0**64)).cuda()
    assert (out[:, 0, first].double() - torch.cos(angle)).abs().max().item() <= BOUND
    sin = torch.sin(-angle if inverse else angle)
    assert (out[:, 0, second].double() - sin).abs().max().item() <= BOUND
