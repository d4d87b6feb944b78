"""paged_attn_fp8_fwd against attention in 64 bits, on both kernels."""

from __future__ import annotations

import math

import pytest
import torch

from fp8_cases import (FP8, NAN_CODE, SPAN, assert_close, attend, make_cache, queries, reference,
                       starts_of, workspace)
from pth_flash_attn import capi, ops

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
# max_query_len: the kernel of 16-row units, of 128-row units; of both, each for its
# requests, where more than eight of them could have FAR keys.
FEW, MANY, BOTH = 1, 17, 1 << 20
FAR = 1 << 17


def check(c, q, q_lens, scale, kernel=None, **kw):
    if kernel is not None:
        kw["max_q"] = kernel
    out = attend(c, q, q_lens, scale, **kw)
    ref = {k: kw[k] for k in ("window", "causal") if k in kw}
    G = q.shape[1] // c.k.shape[2]
    many = (max(q_lens) if kernel is None else kernel) * G > 16 and not kw.get("decode")
    assert capi.AttnLib().last_kernel() == ("f8_wide" if many and kernel != BOTH else "f8_rows")
    want, tol = reference(q, c.keys, q_lens, scale, single=many and q.dtype == BF, **ref)
    assert_close(out, want, tol)
    return out


@pytest.mark.parametrize("kernel", [FEW, MANY, BOTH])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize(("layout", "block"), [("NHD", 16), ("HND", 32), ("NHD", 48), ("HND", 816)])
def test_mixed_lengths(kernel, dtype, D, layout, block):
    """Decodes, drafts, prompts, an empty request, tokens without a place among the keys."""
    q_lens = [1, 3, 0, 17, 1, 40, 2, 70, 5]
    lens = [1, 3, 5, 100, 900, 40, 0, 333, 3]
    far = kernel == BOTH
    c = make_cache(lens, Hkv=2, D=D, block=block, seed=D + block, layout=layout,
                   width=FAR // block + 1 if far else 60)
    q = queries(sum(q_lens), 8, D, dtype, 1)
    check(c, q, q_lens, 0.3 / math.sqrt(D), kernel, max_len=FAR if far else None)


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 700])
@pytest.mark.parametrize(("D", "dtype"), [(64, BF), (128, HF), (256, BF)])
def test_windows(kernel, window, D, dtype):
    q_lens = [1, 4, 33, 130, 1]
    lens = [1, 260, 33, 700, 1500]
    c = make_cache(lens, Hkv=1, D=D, block=32, seed=window)
    q = queries(sum(q_lens), 4, D, dtype, 2)
    check(c, q, q_lens, 1 / math.sqrt(D), kernel, window=window)


@pytest.mark.parametrize("window", [0, 3000])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompts_and_decodes_in_a_batch(window, dtype):
    """Each kernel leaves the other's rows alone, and rows of no request stay; a
    captured call follows requests that change from one to the other."""
    q_lens = [1, 60, 1, 4, 5, 1, 0, 1, 130, 1, 2, 1]
    lens = [700, 60, 33, 4, 500, 1, 9, 0, 3400, 64, 1, 5000]
    c = make_cache(lens, Hkv=32, D=128, block=16, seed=77)
    q = queries(sum(q_lens) + 3, 64, 128, dtype, 77)
    out = check(c, q, q_lens, 0.1, BOTH, window=window)
    assert out[-3:].isnan().all() and not out[:-3].isnan().any()
    starts, ws, out = starts_of(q_lens), workspace(128), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            attend(c, q, q_lens, 0.1, max_q=BOTH, window=window, starts=starts, ws=ws, out=out)
        for new in (q_lens, q_lens[::-1], [17] * 12, [0] * 12, [1] * 12):
            starts.copy_(starts_of(new))
            out.fill_(7.0)
            graph.replay()
            eager = torch.full_like(q, 7.0)
            attend(c, q, new, 0.1, max_q=BOTH, window=window, out=eager)
            side.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize(("Hq", "Hkv"), [(1, 1), (5, 1), (40, 8), (24, 4), (64, 1), (7, 7), (34, 2)])
def test_head_groups(kernel, Hq, Hkv):
    q_lens, lens = [1, 9, 30], [77, 200, 41]
    c = make_cache(lens, Hkv=Hkv, D=64, block=16, seed=Hq)
    q = queries(sum(q_lens), Hq, 64, BF, 3)
    check(c, q, q_lens, 0.125, kernel)


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_not_causal(kernel, D):
    q_lens, lens = [1, 6, 50, 3], [9, 300, 20, 0]
    c = make_cache(lens, Hkv=2, D=D, block=16, seed=4)
    q = queries(sum(q_lens), 4, D, BF, 4)
    check(c, q, q_lens, 0.1, kernel, causal=False)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize(("lens", "Hkv"), [([1], 1), ([20000], 1), ([5000, 1, 0, 17, 9000], 4),
                                           ([600] * 70, 2), ([1000 + 37 * i for i in range(20)], 8)])
def test_decode(D, dtype, lens, Hkv):
    """One token per request, with and without starts; keys cut between work-groups."""
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, seed=5)
    q = queries(len(lens), 4 * Hkv, D, dtype, 5)
    ones = [1] * len(lens)
    a = check(c, q, ones, 1 / math.sqrt(D), decode=True)
    b = check(c, q, ones, 1 / math.sqrt(D), max_q=1)
    assert torch.equal(a, b)
    check(c, q, ones, 1 / math.sqrt(D), decode=True, window=333)
    check(c, q, ones, 1 / math.sqrt(D), decode=True, causal=False)


@pytest.mark.parametrize(("D", "dtype"), [(64, HF), (128, BF), (128, HF), (256, BF)])
@pytest.mark.parametrize(("q_lens", "lens"), [([300], [9000]), ([128, 33, 1], [6000, 3000, 5000]),
                                              ([700, 700], [700, 2000])])
def test_long_chunks(D, dtype, q_lens, lens):
    """128-row units whose keys are cut between work-groups."""
    c = make_cache(lens, Hkv=2, D=D, block=16, seed=6)
    q = queries(sum(q_lens), 8, D, dtype, 6)
    out = check(c, q, q_lens, 1 / math.sqrt(D), MANY)
    check(c, q, q_lens, 1 / math.sqrt(D), MANY, window=1000)
    assert torch.equal(out, attend(c, q, q_lens, 1 / math.sqrt(D), max_q=MANY))


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize(("reqs", "Hkv"), [(3, 3), (2, 4), (33, 1), (70, 2)])
def test_many_prompts(reqs, Hkv, window):
    """Units left whole, in the orders of their row tiles and KV heads, requests without
    tokens among them; more than a wave's lanes of requests."""
    q_lens = [[0, 40, 300, 17, 129][(3 * i) % 5] if i else 260 for i in range(reqs)]
    lens = [n + (50 * i) % 350 for i, n in enumerate(q_lens)]
    c = make_cache(lens, Hkv=Hkv, D=64, block=16, seed=reqs)
    q = queries(sum(q_lens), 4 * Hkv, 64, BF, reqs)
    check(c, q, q_lens, 0.125, MANY, window=window)


@pytest.mark.parametrize(("causal", "window"), [(True, 0), (True, 600), (False, 0)])
@pytest.mark.parametrize(("D", "Hq", "Hkv"), [(64, 15, 3), (128, 8, 8), (256, 8, 2)])
def test_ragged_prompts(D, Hq, Hkv, causal, window):
    """Units that go by the keys that they see: prompts alone and behind long prefixes,
    tokens before the first key, lengths that tie."""
    q_lens = [200, 33, 900, 17, 450, 0, 60]
    lens = [3000, 33, 900, 2500, 2733, 5000, 20]
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, seed=D)
    q = queries(sum(q_lens), Hq, D, BF, D)
    check(c, q, q_lens, 1 / math.sqrt(D), MANY, causal=causal, window=window)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize(("reqs", "Hkv", "D"), [(1, 1, 128), (12, 2, 64), (180, 8, 256)])
def test_short_prompts(reqs, Hkv, D, causal):
    """No request longer than a tile: few that are left whole, many that are not."""
    q_lens = [17 + i % 9 for i in range(reqs)]
    lens = [n + (5 * i) % 36 for i, n in enumerate(q_lens)]
    c = make_cache(lens, Hkv=Hkv, D=D, block=16, seed=reqs)
    q = queries(sum(q_lens), Hkv, D, BF, reqs)
    check(c, q, q_lens, 1 / math.sqrt(D), MANY, causal=causal)


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_peaked_and_wide_scores(kernel, dtype):
    """Scores of some hundred, block scales 2^20 apart, and values near the
    largest that the format has."""
    q_lens, lens, D = [2, 20], [300, 90], 128
    c = make_cache(lens, Hkv=1, D=D, block=16, seed=8, spread=20)
    q = queries(sum(q_lens), 4, D, dtype, 8)
    check(c, q, q_lens, 0.02, kernel)
    if dtype == BF:
        big = make_cache(lens, Hkv=1, D=D, block=16, seed=9)
        big.vs[big.vs < 200] += 246 - 122
        big.keys = [(k, v * 2.0**124) for k, v in big.keys]
        out = attend(big, q, q_lens, 0.1, max_q=kernel)
        want, tol = reference(q, big.keys, q_lens, 0.1, single=True)
        assert_close(out, want, tol)


@pytest.mark.parametrize("kernel", [FEW, MANY])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 6])
def test_nan_reaches_the_rows_that_see_it(kernel, dtype, D, window):
    """A NaN in V spoils its column of the rows that see its key, one in K those
    rows; rows before it, and behind the window, stay as they are."""
    q_lens, lens = [12, 4, 40], [50, 4, 200]
    c = make_cache(lens, Hkv=1, D=D, block=16, seed=10)
    for r, pos, col, cache, j in ((0, 44, 5, c.v, 1), (0, 47, D - 1, c.k, 0), (1, 3, 0, c.v, 1),
                                  (2, 199, 33, c.v, 1), (2, 180, 34, c.v, 1), (2, 165, 1, c.k, 0)):
        page = int(c.table[r, pos // 16])
        cache.view(torch.uint8)[page, pos % 16, 0, col] = 0x80 | NAN_CODE
        c.keys[r][j][pos, 0, col] = math.nan
    q = queries(sum(q_lens), 3, D, dtype, 11)
    out = check(c, q, q_lens, 0.1, kernel, window=window)
    assert not out[:6].isnan().any() and out[6, :, 5].isnan().all()


def test_infinite_and_nan_queries():
    c = make_cache([100, 100], Hkv=1, D=64, block=16, seed=12)
    for kernel in (FEW, MANY):
        q = queries(40, 1, 64, BF, 13)
        want, tol = reference(q, c.keys, [20, 20], 0.1, single=kernel == MANY)
        q[3, 0, 5], q[25, 0, 0] = math.nan, math.inf
        out = attend(c, q, [20, 20], 0.1, max_q=kernel)
        rest = [i for i in range(40) if i not in (3, 25)]
        assert out[3].isnan().all()
        assert_close(out[rest], want[rest], tol[rest])


@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_bounds(kernel):
    """Lengths cut at max_seq_len and at the table's reach, negative ones, page
    numbers outside the cache, starts out of order: nothing is read or written
    outside, rows of no request stay."""
    lens = [100, 64, 30]
    c = make_cache(lens, Hkv=2, D=64, block=16, seed=14)
    q = queries(30, 4, 64, BF, 14)
    q_lens = [5, 3, 2]
    # Cut at max_len: the tokens are then the last of the keys that are left.
    short = [(k[:40], v[:40]) for k, v in c.keys]
    out = attend(c, q, q_lens, 0.1, max_q=kernel, max_len=40)
    want, tol = reference(q, short, q_lens, 0.1, single=kernel == MANY)
    assert_close(out, want, tol)
    # Cut at the table's reach.
    table = c.table[:, :2].contiguous()
    out = attend(c, q, q_lens, 0.1, max_q=kernel, table=table, max_len=1000)
    short = [(k[:32], v[:32]) for k, v in c.keys]
    want, tol = reference(q, short, q_lens, 0.1, single=kernel == MANY)
    assert_close(out, want, tol)
    lens_bad = torch.tensor([-5, 64, -(1 << 31)], dtype=torch.int32, device="cuda")
    out = attend(c, q, q_lens, 0.1, max_q=kernel, lens=lens_bad)
    assert not out[:5].any() and not out[8:10].any() and out[10:].isnan().all()
    wild = c.table.clone()
    wild[0, 1], wild[1, 0], wild[2, 0] = -7, 1 << 30, c.k.shape[0]
    attend(c, q, q_lens, 0.1, max_q=kernel, table=wild)
    for starts in ([0, 20, 10, 30], [5, 3, 2, 1], [-(1 << 31), 4, 1 << 30, 7], [0, 0, 0, 0]):
        attend(c, q, q_lens, 0.1, max_q=kernel,
               starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    none = attend(c, q, [0, 0, 0], 0.1, max_q=kernel)
    assert none.isnan().all()


def test_no_pages_no_requests():
    c = make_cache([3, 4], Hkv=1, D=64, block=16, seed=15)
    q = queries(2, 1, 64, BF, 15)
    out = attend(c, q, [1, 1], 0.1, table=c.table[:, :0], max_len=10)
    assert not out.any()
    out = attend(c, q, [1, 1], 0.1, max_len=0)
    assert not out.any()
    e = attend(c, q[:0], [], 0.1, table=c.table[:0], lens=c.lens[:0])
    assert e.shape[0] == 0


def test_strides_and_query_in_place():
    """Rows cut from a wider buffer, the output into the queries."""
    c = make_cache([70, 500], Hkv=2, D=128, block=16, seed=16, pad=64)
    wide = queries(40, 12, 128, BF, 16)
    q = wide[:, 2:10]
    for kernel in (FEW, MANY):
        buf = wide.clone()
        mine = buf[:, 2:10]
        want, tol = reference(q, c.keys, [10, 30], 0.1, single=kernel == MANY)
        out = attend(c, mine, [10, 30], 0.1, max_q=kernel, out=mine)
        assert_close(out, want, tol)
        assert torch.equal(buf[:, :2], wide[:, :2]) and torch.equal(buf[:, 10:], wide[:, 10:])


@pytest.mark.parametrize("kernel", [FEW, MANY])
def test_captured_replays(kernel):
    """A captured call follows the lengths, two graphs share the workspace, and every
    replay equals the eager call bit for bit."""
    c = make_cache([3000, 700, 64], Hkv=2, D=64, block=16, seed=17)
    q = queries(24, 8, 64, BF, 17)
    ws, out, other = workspace(64), torch.empty_like(q), torch.empty_like(q)
    lens, starts = c.lens.clone(), starts_of([8, 8, 8])
    side = torch.cuda.Stream()

    def call(dst, w):
        attend(c, q, [8, 8, 8], 0.1, window=w, out=dst, ws=ws, lens=lens, starts=starts,
               max_q=kernel)

    with torch.cuda.stream(side):
        call(out, 0)
        side.synchronize()
        graphs = []
        for dst, w in ((out, 0), (other, 100)):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                call(dst, w)
            graphs.append(g)
        for new, st in (([3000, 700, 64], [8, 8, 8]), ([10, 0, 30], [8, 1, 3]), ([2999, 1, 33], [1, 0, 20])):
            lens.copy_(torch.tensor(new))
            starts.copy_(starts_of(st))
            for g, dst, w in ((graphs[0], out, 0), (graphs[1], other, 100)):
                dst.fill_(7.0)
                g.replay()
                eager = torch.full_like(q, 7.0)
                call(eager, w)
                side.synchronize()
                assert torch.equal(dst, eager)


def test_large_pool():
    """Codes behind 2^32 bytes."""
    D, Hkv, block = 128, 8, 16
    page = 2 * block * Hkv * D
    pages = (1 << 32) // page + 40
    codes = torch.zeros(pages, 2, block, Hkv, D, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(2, pages, 1, Hkv, dtype=torch.uint8, device="cuda")
    k, v = codes[:, 0].view(FP8), codes[:, 1].view(FP8)
    far = torch.arange(pages - 20, pages, device="cuda")
    T = 20 * SPAN
    key, value = (queries(T, Hkv, D, BF, s) for s in (18, 19))
    slots = (far[:, None] * block + torch.arange(block, device="cuda")).reshape(-1)
    ops.reshape_and_cache_fp8(key, value, k, v, scale[0], scale[1], slots)
    table = far.to(torch.int32)[None].contiguous()
    back = [torch.empty_like(key) for _ in range(2)]
    ops.gather_cache_fp8(*back, k, v, scale[0], scale[1], table, starts_of([T]))
    for a, b in zip(back, (key, value)):
        assert (a.double() - b.double()).abs().max().item() <= 2.0**-4 * b.abs().max().item()
    q = queries(2, 16, D, BF, 20)
    out = torch.empty_like(q)
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    ops.paged_attn_fp8_fwd(out, q, k, v, scale[0], scale[1], table, lens, starts_of([2]), 2, T, 0.1,
                           workspace(D))
    want, tol = reference(q, [(back[0].double(), back[1].double())], [2], 0.1)
    assert_close(out, want, tol)
    assert not codes[: pages - 20].any()
