"""The partition of large batches (paged_decode_fwd, cross_attn_fwd): more groups
than resident work-groups, so that cut groups are noted by work-group, and the
16-row kernel over more than 64 requests of several query tokens, whose groups
are counted across windows of requests. References and tolerances as in
test_paged16_gpu.py; requests that the references leave out are checked for
being finite and, by a second call, for repeating."""

from __future__ import annotations

import pytest
import torch

from paged16_cases import (DEV, assert_close, cross, decode, make_cache, queries, reference,
                           starts_of)
from pth_flash_attn import capi

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
RESIDENT = {64: 3, 128: 2, 256: 1}  # work-groups of a compute unit


def cus():
    return torch.cuda.get_device_properties(DEV).multi_processor_count


def ragged(n, lo, hi, seed):
    return torch.randint(lo, hi + 1, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def few_of(R):
    """Requests at the edges of the windows of 64, the long one, and some others."""
    at = {0, 1, R // 2, R - 2, R - 1} | {64 * w + d for w in range(1, R // 64 + 1) for d in (-1, 0)}
    return sorted(r for r in at | set(range(0, R, max(1, R // 24))) if 0 <= r < R)


def check_requests(got, q, c, q_lens, starts, scale, pair, few):
    at = starts.tolist()
    for r in few:
        rows = slice(at[r], at[r + 1])
        want, tol = reference(q[rows], c.keys[r : r + 1], [q_lens[r]], scale, pair=pair)
        assert_close(got[rows], want, tol)
    assert not got.isnan().any()


@pytest.mark.parametrize(("D", "Hkv", "G"), [(64, 16, 4), (128, 8, 4), (128, 8, 1), (256, 4, 4),
                                             (256, 6, 5)])
@pytest.mark.parametrize("R", [65, 128, 200])
def test_decode_of_more_groups_than_work_groups(D, Hkv, G, R):
    """HND pages, so that each KV head is a group."""
    R = max(R, RESIDENT[D] * cus() // Hkv + 1)  # so many groups are cut and noted by work-group
    lens = ragged(R, 0, 700, R)
    lens[R // 2], lens[R // 2 + 1] = 5000, 0
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=BF, seed=R, layout="HND")
    q = queries(R, Hkv * G, D, BF, R)
    got = decode(c, q, D**-0.5)
    assert capi.AttnLib().last_kernel() == "p16_rows"
    check_requests(got, q, c, [1] * R, starts_of([1] * R), D**-0.5, True, few_of(R))
    assert (got[R // 2 + 1] == 0).all()
    assert torch.equal(got, decode(c, q, D**-0.5))
    # The same rows where the window cuts most of them.
    windowed = decode(c, q, D**-0.5, window=600)
    for r in few_of(R):
        want, tol = reference(q[r : r + 1], c.keys[r : r + 1], [1], D**-0.5, window=600, pair=True)
        assert_close(windowed[r : r + 1], want, tol)


@pytest.mark.parametrize("R", [63, 64, 65, 128, 130, 1000])
@pytest.mark.parametrize(("layout", "Hkv", "D"), [("NHD", 8, 64), ("NHD", 8, 128), ("NHD", 2, 128),
                                                  ("HND", 8, 128), ("NHD", 4, 256), ("NHD", 1, 64)])
def test_few_rows_of_many_requests(R, layout, Hkv, D):
    """Four query tokens of four heads: full tiles of 16 rows, one, two and four
    units side by side by the layout and the number of heads; requests without
    tokens, and without keys, among them."""
    if R == 1000 and D == 256:
        Hkv = 2  # the same team, half the cache
    G = 4
    lens = ragged(R, 0, 300, R + D)
    lens[R // 2], lens[R // 3] = 4000, 0
    q_lens = ragged(R, 0, 4, R)
    q_lens[R // 2], q_lens[0], q_lens[R - 1], q_lens[R // 3] = 4, 3, 1, 2
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=HF, seed=R, layout=layout)
    starts = starts_of(q_lens)
    q = queries(sum(q_lens), Hkv * G, D, HF, R)
    got = cross(c, q, q_lens, D**-0.5, max_q=4, starts=starts)
    assert capi.AttnLib().last_kernel() == "p16_rows"
    check_requests(got, q, c, q_lens, starts, D**-0.5, True, few_of(R))
    assert torch.equal(got, cross(c, q, q_lens, D**-0.5, max_q=4, starts=starts))


@pytest.mark.parametrize("R", [65, 130])
@pytest.mark.parametrize(("longest", "keys"), [(700, 700), (6000, 200)])
def test_few_rows_noted_by_group(R, longest, keys):
    """One KV head and few heads: fewer groups than work-groups, with more
    than 64 requests, so that the notes' places are counted across windows."""
    lens = ragged(R, 0, keys, R)
    lens[R - 1] = lens[64] = longest
    q_lens = ragged(R, 0, 2, R)
    q_lens[R - 1], q_lens[64] = 2, 1
    c = make_cache(lens, Hkv=1, D=128, block=16, dtype=BF, seed=R)
    starts = starts_of(q_lens)
    q = queries(sum(q_lens), 8, 128, BF, R)
    got = cross(c, q, q_lens, 0.09, max_q=2, starts=starts)
    assert capi.AttnLib().last_kernel() == "p16_rows"
    check_requests(got, q, c, q_lens, starts, 0.09, True, range(R))


@pytest.mark.parametrize(("D", "Hkv"), [(64, 16), (128, 8), (256, 4)])
@pytest.mark.parametrize("R", [70, 150])
def test_wide_units_cut_and_noted_by_work_group(D, Hkv, R):
    """Units of 128 rows, more than work-groups, and states past the bound up to
    which they stay whole."""
    G = 2
    R = max(R, RESIDENT[D] * cus() // Hkv + 1)
    lens = ragged(R, 0, 300, R)
    lens[R // 2], lens[R - 1], lens[1] = 3000, 1700, 0
    q_lens = ragged(R, 0, 60, R)
    q_lens[R // 2], q_lens[R - 1], q_lens[1] = 130, 9, 20
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=BF, seed=R)
    starts = starts_of(q_lens)
    q = queries(sum(q_lens), Hkv * G, D, BF, R)
    got = cross(c, q, q_lens, D**-0.5, starts=starts)
    assert capi.AttnLib().last_kernel() == "p16_wide"
    check_requests(got, q, c, q_lens, starts, D**-0.5, False, few_of(R))
    assert torch.equal(got, cross(c, q, q_lens, D**-0.5, starts=starts))
