"""Attention over a paged 16-bit cache (paged_decode_fwd, cross_attn_fwd)
against 64 bits: lengths around the tiles' edges, pages of every kind, head
layouts, windows, empty requests, padded batches. Every slot that holds no
token of a request, and every unused page, is NaN (paged16_cases.py, which
derives the tolerances)."""

from __future__ import annotations

import math

import pytest
import torch

from paged16_cases import (DEV, assert_close, cross, decode, make_cache, queries, reference,
                           starts_of, workspace)
from pth_flash_attn import capi, ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
EDGES = [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]


def last_kernel():
    return capi.AttnLib().last_kernel()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads", [(4, 1), (6, 6), (8, 2), (24, 4)])
def test_decode_edges(D, dtype, heads):
    Hq, Hkv = heads
    lens = EDGES + [0, 700]
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=dtype, seed=D + Hq)
    q = queries(len(lens), Hq, D, dtype, 1)
    got = decode(c, q, D**-0.5)
    assert last_kernel() == "p16_rows"
    assert_close(got, *reference(q, c.keys, [1] * len(lens), D**-0.5, pair=True))
    assert (got[lens.index(0)] == 0).all()


@pytest.mark.parametrize("block", [1, 7, 16, 48, 100, 528])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_pages(block, layout, D):
    lens = [5, 100, 333, 0, 1000]
    c = make_cache(lens, Hkv=2, D=D, block=block, dtype=BF, seed=block, layout=layout, pad=24)
    q = queries(len(lens), 8, D, BF, 2)
    assert_close(decode(c, q, D**-0.5), *reference(q, c.keys, [1] * 5, D**-0.5, pair=True))


@pytest.mark.parametrize("G", [1, 5, 15, 16, 17, 33, 64])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_groups(G, D):
    lens = [300, 40, 0]
    c = make_cache(lens, Hkv=2, D=D, block=32, dtype=HF, seed=G)
    q = queries(3, 2 * G, D, HF, 3)
    assert_close(decode(c, q, D**-0.5), *reference(q, c.keys, [1] * 3, D**-0.5, pair=True))


@pytest.mark.parametrize("window", [1, 15, 16, 17, 31, 100, 128, 129, 4000])
@pytest.mark.parametrize(("D", "block"), [(64, 16), (128, 48), (128, 5), (256, 16)])
def test_decode_window_with_dead_pages(window, D, block):
    """Pages wholly below the window belong to nobody: NaN."""
    lens = [1, 16, 100, 129, 1000, 1025, 3000]
    c = make_cache(lens, Hkv=2, D=D, block=block, dtype=BF, seed=window)
    for r, L in enumerate(lens):
        c.table[r, : max(0, L - window) // block] = 0
    q = queries(len(lens), 8, D, BF, 4)
    assert_close(decode(c, q, D**-0.5, window=window),
                 *reference(q, c.keys, [1] * len(lens), D**-0.5, window=window, pair=True))


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_long_and_many(D):
    """One long request among short ones, and more requests than lanes."""
    gen = torch.Generator().manual_seed(D)
    lens = torch.randint(0, 400, (150,), generator=gen).tolist()
    lens[70] = 30000
    c = make_cache(lens, Hkv=2, D=D, block=16, dtype=BF, seed=5)
    q = queries(len(lens), 4, D, BF, 5)
    got = decode(c, q, D**-0.5)
    assert_close(got, *reference(q, c.keys, [1] * 150, D**-0.5, pair=True))
    assert torch.equal(got, decode(c, q, D**-0.5))  # deterministic


@pytest.mark.parametrize("R", [64, 65, 128, 1000, 4096, 4097, 4500])
def test_many_requests(R):
    """Around 64 requests and around 64 times 64; a few tokens each."""
    gen = torch.Generator().manual_seed(R)
    lens = torch.randint(0, 40, (R,), generator=gen).tolist()
    lens[R // 2] = 3000
    c = make_cache(lens, Hkv=1, D=64, block=16, dtype=BF, seed=R)
    q = queries(R, 2, 64, BF, R)
    got = decode(c, q, 0.125)
    few = list(range(0, R, max(1, R // 40))) + [R // 2, R - 1]
    for r in few:
        assert_close(got[r : r + 1], *reference(q[r : r + 1], c.keys[r : r + 1], [1], 0.125, pair=True))
    q_lens = torch.randint(0, 12, (R,), generator=gen).tolist()
    starts = starts_of(q_lens)
    q = queries(sum(q_lens), 2, 64, BF, R + 1)
    got = cross(c, q, q_lens, 0.125, starts=starts)
    at = starts.tolist()
    for r in few:
        rows = slice(at[r], at[r + 1])
        assert_close(got[rows], *reference(q[rows], c.keys[r : r + 1], q_lens[r : r + 1], 0.125))
    assert not got.isnan().any()


def test_decode_long_alone():
    c = make_cache([131072], Hkv=2, D=128, block=16, dtype=BF, seed=6)
    q = queries(1, 8, 128, BF, 6)
    assert_close(decode(c, q, 128**-0.5), *reference(q, c.keys, [1], 128**-0.5, pair=True))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads", [(4, 1), (6, 6), (10, 2)])
def test_cross_edges(D, dtype, heads):
    Hq, Hkv = heads
    lens = EDGES + [0, 400, 500]
    q_lens = [3, 0, 128, 1, 33, 64, 17, 2, 40, 1, 65, 127, 5, 129, 31, 9, 300, 16]
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=dtype, seed=D + Hq)
    q = queries(sum(q_lens), Hq, D, dtype, 7)
    got = cross(c, q, q_lens, D**-0.5)
    assert last_kernel() == "p16_wide"
    assert_close(got, *reference(q, c.keys, q_lens, D**-0.5))


@pytest.mark.parametrize("q_max", [1, 2, 4])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cross_few_rows(q_max, D):
    lens = [0, 1500, 77, 301, 64]
    q_lens = [q_max, 1, 0, q_max, 1]
    c = make_cache(lens, Hkv=4, D=D, block=16, dtype=HF, seed=q_max)
    q = queries(sum(q_lens), 16, D, HF, 8)
    got = cross(c, q, q_lens, D**-0.5)
    assert last_kernel() == "p16_rows"
    assert_close(got, *reference(q, c.keys, q_lens, D**-0.5, pair=True))


@pytest.mark.parametrize("block", [1, 7, 16, 48, 100, 528])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_cross_pages(block, layout, D):
    lens, q_lens = [100, 333, 1000], [50, 3, 130]
    c = make_cache(lens, Hkv=2, D=D, block=block, dtype=BF, seed=block, layout=layout, pad=24)
    q = queries(sum(q_lens), 8, D, BF, 9)
    assert_close(cross(c, q, q_lens, D**-0.5), *reference(q, c.keys, q_lens, D**-0.5))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_cross_cut_units(D, dtype):
    """Few row tiles against long states: every unit is cut between work-groups."""
    lens, q_lens = [6000, 2777], [150, 70]
    c = make_cache(lens, Hkv=1, D=D, block=16, dtype=dtype, seed=10)
    q = queries(sum(q_lens), 4, D, dtype, 10)
    got = cross(c, q, q_lens, D**-0.5)
    assert_close(got, *reference(q, c.keys, q_lens, D**-0.5))
    assert torch.equal(got, cross(c, q, q_lens, D**-0.5))


@pytest.mark.parametrize("longest", [700, 1500, 2200, 6000])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_cross_few_rows_of_long_states(longest, layout):
    """Full tiles of 16 rows, cut: one, two and four units side by side, joined
    row by row and slot by slot."""
    lens, q_lens = [longest, longest // 2, 33, 0, longest - 1, 1, 17, 600], [4, 1, 3, 4, 4, 2, 4, 0]
    c = make_cache(lens, Hkv=8, D=128, block=16, dtype=BF, seed=longest, layout=layout)
    q = queries(sum(q_lens), 32, 128, BF, 13)
    got = cross(c, q, q_lens, 0.09)
    assert last_kernel() == "p16_rows"
    assert_close(got, *reference(q, c.keys, q_lens, 0.09, pair=True))


@pytest.mark.parametrize("bound", [64, 128, 129, 512, 513])
@pytest.mark.parametrize("heads", [(2, 1), (16, 4)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_bounds_at_which_groups_stay_whole(bound, heads, D):
    lens = [bound, 0, 1, bound - 1, 16, bound // 2] * 3
    c = make_cache(lens, Hkv=heads[1], D=D, block=16, dtype=BF, seed=bound)
    q = queries(len(lens), heads[0], D, BF, bound)
    assert_close(decode(c, q, D**-0.5), *reference(q, c.keys, [1] * 18, D**-0.5, pair=True))
    q_lens = [40, 3, 1, 0, 17, 130] * 3
    q = queries(sum(q_lens), heads[0], D, BF, bound)
    assert_close(cross(c, q, q_lens, D**-0.5), *reference(q, c.keys, q_lens, D**-0.5))
    # A bound above the lengths: the same rows, another partition.
    far = cross(c, q, q_lens, D**-0.5, max_len=20 * bound)
    assert_close(far, *reference(q, c.keys, q_lens, D**-0.5))


@pytest.mark.parametrize("bound", [512, 513, 1024, 1025, 1536, 1537])
@pytest.mark.parametrize(("D", "heads", "R"), [(64, (16, 16), 16), (128, (32, 8), 18),
                                               (256, (16, 4), 16), (128, (2, 1), 6)])
def test_bounds_at_which_wide_groups_stay_whole(bound, D, heads, R):
    """Units of about three quarters of the device, and of next to nothing."""
    lens = ([bound, 0, bound // 3, bound - 1, 65] * R)[:R]
    step = 128 * heads[1] // heads[0]
    q_lens = ([step, 2 * step + 1, 1, 3 * step - 1, 0, 2 * step] * R)[:R]
    c = make_cache(lens, Hkv=heads[1], D=D, block=32, dtype=HF, seed=bound)
    q = queries(sum(q_lens), heads[0], D, HF, bound)
    got = cross(c, q, q_lens, D**-0.5)
    assert last_kernel() == "p16_wide"
    assert_close(got, *reference(q, c.keys, q_lens, D**-0.5))


def test_cross_many_requests():
    gen = torch.Generator().manual_seed(11)
    lens = torch.randint(0, 200, (140,), generator=gen).tolist()
    q_lens = torch.randint(0, 60, (140,), generator=gen).tolist()
    c = make_cache(lens, Hkv=2, D=64, block=16, dtype=BF, seed=11)
    q = queries(sum(q_lens), 8, 64, BF, 11)
    assert_close(cross(c, q, q_lens, 0.125), *reference(q, c.keys, q_lens, 0.125))


@pytest.mark.parametrize("max_q", [0, 1, 10_000])
def test_cross_any_query_bound(max_q):
    """max_query_len chooses the kernel; any value is correct."""
    lens, q_lens = [100, 0, 257], [40, 3, 9]
    c = make_cache(lens, Hkv=2, D=128, block=16, dtype=BF, seed=12)
    q = queries(sum(q_lens), 8, 128, BF, 12)
    assert_close(cross(c, q, q_lens, 0.1, max_q=max_q), *reference(q, c.keys, q_lens, 0.1))


@pytest.mark.parametrize("few", [True, False])
def test_rows_of_no_request_are_left(few):
    lens, q_lens = [100, 50], [2, 1] if few else [30, 20]
    c = make_cache(lens, Hkv=2, D=128, block=16, dtype=BF, seed=13)
    T = sum(q_lens)
    q = queries(T + 5, 8, 128, BF, 13)
    out = torch.full_like(q, 7.0)
    cross(c, q, q_lens, 0.1, out=out)
    assert (out[T:] == 7.0).all()
    want, tol = reference(q[:T], c.keys, q_lens, 0.1, pair=few)
    assert_close(out[:T], want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_strided_views(D):
    """Queries cut from the fused projection's output, outputs into a wider
    buffer whose other columns stay."""
    lens, q_lens, Hq, Hkv = [90, 200, 31], [9, 40, 3], 8, 2
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, dtype=BF, seed=14)
    T = sum(q_lens)
    fused = queries(T, Hq + 2 * Hkv, D, BF, 14)
    q = fused[:, :Hq]
    buf = torch.full((T, Hq + 3, D + 16), 5.0, dtype=BF, device=DEV)
    out = buf[:, 1 : 1 + Hq, 8 : 8 + D]
    cross(c, q, q_lens, 0.1, out=out)
    assert_close(out, *reference(q, c.keys, q_lens, 0.1))
    mask = torch.ones_like(buf, dtype=torch.bool)
    mask[:, 1 : 1 + Hq, 8 : 8 + D] = False
    assert (buf[mask] == 5.0).all()
    buf.fill_(5.0)
    o = decode(c, q[:3], 0.1, out=out[:3])
    assert_close(o, *reference(q[:3], c.keys, [1] * 3, 0.1, pair=True))
    assert (buf[:3][mask[:3]] == 5.0).all() and (buf[3:] == 5.0).all()


@pytest.mark.parametrize("wide", [False, True])
def test_lengths_and_pages_out_of_range_read_nothing_outside(wide):
    """Lengths past the bound or the table are cut, negative ones are 0, page
    numbers outside the cache stand for page 0, starts outside q are brought
    into it: outputs of well-formed requests are unaffected."""
    lens = [64, 64, 64, 64]
    c = make_cache(lens, Hkv=2, D=128, block=16, dtype=BF, seed=15, spare=0)
    n = 40 if wide else 1
    q = queries(4 * n, 8, 128, BF, 15)
    c.kv[0] = 0.5
    c.lens.copy_(torch.tensor([1 << 30, -5, 64, 64], dtype=torch.int32))
    c.table[3, 1] = -1
    c.table[3, 2] = 1 << 30
    starts = starts_of([n] * 4)
    out = cross(c, q, [n] * 4, 0.1, max_len=1 << 20, max_q=n, starts=starts)
    keys = list(c.keys)
    keys[1] = (keys[1][0][:0], keys[1][1][:0])
    k3, v3 = (x.clone() for x in keys[3])
    k3[16:48], v3[16:48] = 0.5, 0.5
    keys[3] = (k3, v3)
    assert_close(out, *reference(q, keys, [n] * 4, 0.1, pair=not wide))
    if not wide:
        got = decode(c, q, 0.1, max_len=1 << 20)
        assert_close(got, *reference(q, keys, [1] * 4, 0.1, pair=True))
    bad = torch.tensor([-3, n, 2 * n, 1 << 30, 1 << 30], dtype=torch.int32, device=DEV)
    out = cross(c, q, [n] * 4, 0.1, max_len=1 << 20, max_q=n, starts=bad)
    want, tol = reference(q, keys, [n] * 4, 0.1, pair=not wide)
    assert_close(out[:2 * n], want[:2 * n], tol[:2 * n])


@pytest.mark.parametrize("n", [1, 40])
def test_infinite_and_nan_values(n):
    """A visible NaN, or a score of +inf, makes its row NaN, as the formula
    does; rows of other heads and requests are finite; scores of -inf weigh
    nothing, and a row of them alone is NaN."""
    c = make_cache([50, 50, 50, 50], Hkv=2, D=64, block=16, dtype=BF, seed=16)
    q = queries(4 * n, 2, 64, BF, 16).abs()
    q[3 * n :] = 1.0

    def put(r, pos, head, value, which):
        page = int(c.table[r, pos // 16])
        which[page, pos % 16, head] = value
        (c.keys[r][0] if which is c.k else c.keys[r][1])[pos, head] = value

    put(0, 20, 0, math.nan, c.v)
    put(1, 49, 1, math.inf, c.k)
    put(2, 3, 0, -math.inf, c.k)
    for i in range(50):
        put(3, i, 0, -math.inf, c.k)
    out = cross(c, q, [n] * 4, 0.125)
    assert out[:n, 0].isnan().all() and out[n : 2 * n, 1].isnan().all()
    assert out[3 * n :, 0].isnan().all()
    want, tol = reference(q, c.keys, [n] * 4, 0.125, pair=n == 1)
    tol = tol.nan_to_num(0.0)
    for rows, head in ((slice(0, n), 1), (slice(n, 2 * n), 0), (slice(3 * n, 4 * n), 1)):
        assert_close(out[rows, head], want[rows, head], tol[rows, head])
    # Request 2: without the key of weight 0, whose tolerance term is infinite.
    keep = [i for i in range(50) if i != 3]
    k2, v2 = c.keys[2]
    want, tol = reference(q[2 * n : 3 * n], [(k2[keep], v2[keep])], [n], 0.125, pair=n == 1)
    assert_close(out[2 * n : 3 * n, 0], want[:, 0], tol[:, 0])


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_sharp_rows(n, dtype):
    """Scores of +-hundreds: the running maximum moves far, weights vanish."""
    c = make_cache([700, 333], Hkv=1, D=128, block=16, dtype=dtype, seed=17, scale=8.0)
    q = queries(2 * n, 4, 128, dtype, 17) * 8
    assert_close(cross(c, q, [n, n], 0.3), *reference(q, c.keys, [n, n], 0.3, pair=n == 1))


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("below", [10, 20, 24, 26])
def test_one_large_weight_and_many_small(n, dtype, below):
    """30,000 keys 2^-below of the first one's weight: their sum counts. The
    first one's V is 0 and theirs 1; all numbers are powers of two, so that the
    output is x / (1 + x) rounded once, and P is exact."""
    N = 30000
    c = make_cache([N], Hkv=1, D=64, block=16, dtype=dtype, seed=31)
    k, v = torch.zeros(N, 1, 64, dtype=dtype, device=DEV), torch.ones(N, 1, 64, dtype=dtype,
                                                                      device=DEV)
    k[1:, 0, 0] = -float(below)
    v[0] = 0.0
    pos = torch.arange(N, device=DEV)
    page = c.table[0].long()[pos // 16]
    c.k[page, pos % 16], c.v[page, pos % 16] = k, v
    q = torch.zeros(n, 1, 64, dtype=dtype, device=DEV)
    q[:, :, 0] = 1.0
    got = cross(c, q, [n], math.log(2.0)).double()
    x = (N - 1) * 2.0**-below
    want = x / (1 + x)
    # ln 2 in 32 bits and its product with log2(e) (2 u), exp2 (2 u), each times
    # `below` or less, and 30,000 additions in 32 bits; the output's rounding.
    h, u = torch.finfo(dtype).eps / 2, 2.0**-24
    assert ((got - want).abs() <= want * (h + u * (4 * below + 4 + 2 * N))).all()


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB, its last pages in use."""
    block, Hkv, D = 64, 8, 128
    pages = (5 << 30) // (2 * block * Hkv * D * 2)
    kv = torch.full((pages, 2, block, Hkv, D), math.nan, dtype=BF, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(18)
    ids = [pages - 1, 3, pages - 2]
    for i in ids:
        kv[i] = torch.randn(2, block, Hkv, D, generator=gen, device=DEV).to(BF)
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    k, v = kv[:, 0], kv[:, 1]
    keys = [(k[ids].reshape(-1, Hkv, D)[:150], v[ids].reshape(-1, Hkv, D)[:150])]
    q = queries(40, 16, D, BF, 18)
    out = torch.empty_like(q)
    ops.cross_attn_fwd(out, q, k, v, table, lens, starts_of([40]), 40, 150, 0.1, workspace(D))
    assert_close(out, *reference(q, keys, [40], 0.1))
    out = torch.empty_like(q[:1])
    ops.paged_decode_fwd(out, q[:1], k, v, table, lens, 150, 0.1, workspace(D))
    assert_close(out, *reference(q[:1], keys, [1], 0.1, pair=True))
    slots = torch.tensor([(pages - 1) * block + 5, 7], device=DEV)
    new = queries(2, Hkv, D, BF, 19)
    ops.reshape_and_cache_16bit(new, new + 1, k, v, slots)
    assert torch.equal(k[pages - 1, 5], new[0]) and torch.equal(v[0, 7], (new + 1)[1])


@pytest.mark.parametrize("n", [1, 40])
def test_streams_and_two_calls_at_once(n):
    """Two calls on two streams, each with its workspace, behind work that
    delays their inputs."""
    cases = []
    for i in range(2):
        c = make_cache([900, 2000], Hkv=2, D=128, block=16, dtype=BF, seed=20 + i)
        q = queries(2 * n, 8, 128, BF, 20 + i)
        cases.append((c, q, workspace(128), torch.empty_like(q), torch.cuda.Stream()))
    a = torch.randn(2048, 2048, device=DEV)
    torch.cuda.synchronize()
    for c, q, ws, out, stream in cases:
        with torch.cuda.stream(stream):
            late = (a @ a)[0, 0] * 0 + q.float()
            cross(c, late.to(BF), [n, n], 0.1, ws=ws, out=out)
            out.add_(0)
    torch.cuda.synchronize()
    for c, q, _, out, _ in cases:
        assert_close(out, *reference(q, c.keys, [n, n], 0.1, pair=n == 1))


@pytest.mark.parametrize("n", [1, 40])
def test_graph_replays_as_lengths_change(n):
    lens = [600, 257, 1000]
    c = make_cache(lens, Hkv=2, D=128, block=16, dtype=BF, seed=22)
    q = queries(3 * n, 8, 128, BF, 22)
    ws, out, starts = workspace(128), torch.empty_like(q), starts_of([n] * 3)
    call = lambda: cross(c, q, [n] * 3, 0.1, ws=ws, out=out, starts=starts)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for now in ([600, 257, 1000], [1, 0, 999], [64, 128, 16], [600, 200, 3]):
        c.lens.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        call()
        torch.cuda.synchronize()
        assert torch.equal(replayed, out)
        keys = [(k[:L], v[:L]) for (k, v), L in zip(c.keys, now)]
        assert_close(out, *reference(q, keys, [n] * 3, 0.1, pair=n == 1))


def test_graphs_share_a_workspace():
    """Captured calls of other shapes, head sizes and kernels leave nothing in
    the workspace that the next one reads."""
    ws = torch.full((max(workspace(D).numel() for D in (64, 128, 256)),), math.nan, device=DEV)
    graphs = []
    for i, (D, lens, n) in enumerate([(128, [3000, 40, 0], 1), (64, [2000, 1999], 50),
                                      (256, [700], 4), (64, [800] * 9, 3)]):
        c = make_cache(lens, Hkv=4, D=D, block=16, dtype=BF, seed=40 + i)
        q = queries(len(lens) * n, 16, D, BF, 40 + i)
        out, starts = torch.empty_like(q), starts_of([n] * len(lens))
        want = cross(c, q, [n] * len(lens), 0.1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cross(c, q, [n] * len(lens), 0.1, ws=ws, out=out, starts=starts)
        graphs.append((graph, out, want, (c, q, starts)))
    for order in ([0, 1, 2, 3], [3, 1, 0, 2], [2, 2, 1, 0, 3]):
        for i in order:
            graphs[i][1].fill_(math.nan)
            graphs[i][0].replay()
        torch.cuda.synchronize()
        for _, out, want, _ in graphs:
            assert torch.equal(out, want)


def test_compile_traces_and_opcheck():
    c = make_cache([60, 30], Hkv=2, D=64, block=16, dtype=BF, seed=23)
    q, ws = queries(2, 4, 64, BF, 23), workspace(64)
    args = (torch.empty_like(q), q, c.k, c.v, c.table, c.lens, 60, 0.125, ws.fill_(0.0), 0)
    torch.library.opcheck(torch.ops.pth_flash_attn.paged_decode_fwd.default, args,
                          test_utils=("test_schema", "test_faketensor"))
    args = (torch.empty_like(q), q, c.k, c.v, c.table, c.lens, starts_of([1, 1]), 1, 60, 0.125, ws)
    torch.library.opcheck(torch.ops.pth_flash_attn.cross_attn_fwd.default, args,
                          test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("n", [1, 24, 200])
def test_out_is_q(n):
    """Whole and cut units, one and several waves of a unit, in place."""
    for lens, block in (([700, 33, 0, 129], 16), ([9000, 33, 0, 4000], 48)):
        c = make_cache(lens, Hkv=2, D=128, block=block, dtype=BF, seed=n)
        q = queries(4 * n, 8, 128, BF, n)
        both = q.clone()
        if n == 1:
            assert torch.equal(decode(c, both, 0.1, out=both), decode(c, q, 0.1))
        else:
            assert torch.equal(cross(c, both, [n] * 4, 0.1, out=both), cross(c, q, [n] * 4, 0.1))


def test_empty_batches():
    c = make_cache([10], Hkv=1, D=64, block=16, dtype=BF, seed=24)
    q = queries(0, 4, 64, BF, 24)
    none = c.lens[:0]
    decode(c, q, 0.1, lens=none, table=c.table[:0])
    out = torch.full((3, 4, 64), 2.0, dtype=BF, device=DEV)
    ops.cross_attn_fwd(out, queries(3, 4, 64, BF, 24), c.k, c.v, c.table, c.lens,
                       starts_of([0]), 0, 10, 0.1, workspace(64))
    torch.cuda.synchronize()
    assert (out == 2.0).all()


def test_workspace_and_device_refusals():
    c = make_cache([10], Hkv=1, D=64, block=16, dtype=BF, seed=25)
    q = queries(1, 4, 64, BF, 25)
    with pytest.raises(RuntimeError, match="ws must be 16-byte aligned and hold"):
        decode(c, q, 0.1, ws=workspace(64)[4:])
    with pytest.raises(RuntimeError, match="ws must be 16-byte aligned and hold"):
        decode(c, q, 0.1, ws=torch.empty(0, device=DEV))
    with pytest.raises(RuntimeError, match="all tensors must be on the device of q"):
        decode(c, q, 0.1, lens=c.lens.cpu())
    with pytest.raises(RuntimeError, match="16-byte aligned rows"):
        big = torch.zeros(1, 4, 72, dtype=BF, device=DEV)
        decode(c, big[..., 4:68], 0.1, out=torch.empty_like(q))
    with pytest.raises(RuntimeError, match="out must not overlap an input"):
        decode(c, q, 0.1, out=c.kv.view(-1)[:256].view(1, 4, 64))
