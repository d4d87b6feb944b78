"""Rotary positions and the ops of an 8-bit cache together, as a serving loop
uses them: a step's tables, its queries and keys rotated in place, the write,
attention, and the cache read back; prompts, then decodes; eager, captured, on
another stream, under opcheck and torch.compile."""

from __future__ import annotations

import pytest
import torch

from fp8_cases import DEV, assert_close, make_cache, queries, reference, starts_of, workspace
from pth_flash_attn import ops, rotary
from pth_flash_attn.cache import fp8_cache

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16
I32 = dict(dtype=torch.int32, device=DEV)
OPS = torch.ops.pth_flash_attn
HQ, HKV, BLOCK, PAGES, WIDTH, MOST = 8, 2, 32, 40, 8, 256
PROMPTS = [70, 1, 33, 100]


class Loop:
    """One layer's buffers; every step has at most T tokens of R requests."""

    def __init__(self, D, dtype, layout, interleaved):
        self.D, self.R, self.interleaved = D, len(PROMPTS), interleaved
        self.gen = torch.Generator(device=DEV).manual_seed(D)
        self.cache = fp8_cache(PAGES, BLOCK, HKV, D, layout=layout)
        R, T = self.R, sum(PROMPTS) + 5  # five rows of padding
        self.table = torch.zeros(R, WIDTH, **I32)
        self.slots = torch.zeros(T, dtype=torch.int64, device=DEV)
        self.seq, self.starts = torch.zeros(R, **I32), torch.zeros(R + 1, **I32)
        self.pool, self.pool_in = torch.zeros(2, **I32), torch.zeros(2, **I32)
        self.ctx, self.new = torch.zeros(R, **I32), torch.zeros(R, **I32)
        self.free = torch.randperm(PAGES - 1, generator=self.gen, device=DEV).to(torch.int32) + 1
        self.qkv = torch.zeros(T, (HQ + 2 * HKV) * D, dtype=dtype, device=DEV)
        self.pos = torch.zeros(T, dtype=torch.int64, device=DEV)
        self.out = torch.zeros(T, HQ, D, dtype=dtype, device=DEV)
        self.turns, self.scale = rotary.rotary_turns(D // 2, scaling="ramp", factor=4.0)
        self.ws = workspace(D)

    def split(self):
        T, D = self.qkv.shape[0], self.D
        q, k, v = self.qkv.split([HQ * D, HKV * D, HKV * D], dim=1)
        return q.view(T, HQ, D), k.view(T, HKV, D), v.view(T, HKV, D)

    def feed(self, new):
        """The next step's tokens, on the host's side of the program."""
        self.ctx.copy_(self.seq)
        self.pool_in.copy_(self.pool)
        self.new.copy_(torch.tensor(new))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.gen, device=DEV))
        at = torch.cat([self.ctx[r] + torch.arange(n, device=DEV) for r, n in enumerate(new)])
        self.pos.zero_()
        self.pos[: len(at)] = at

    def step(self, max_q):
        q, k, v = self.split()
        ops.build_step_tables(self.table, self.slots, self.seq, self.starts, self.pool, self.ctx,
                              self.new, self.free, self.pool_in, BLOCK)
        ops.rotary_embedding(q, k, q, k, self.pos, self.turns, self.interleaved, self.scale)
        ops.reshape_and_cache_fp8(k, v, *self.cache, self.slots)
        ops.paged_attn_fp8_fwd(self.out, q, *self.cache, self.table, self.seq, self.starts, max_q,
                               MOST, 0.1, self.ws)

    def read(self):
        """Per request (K, V) of all its tokens, as the cache holds them."""
        lens = self.seq.tolist()
        rows = [torch.empty(sum(lens), HKV, self.D, device=DEV) for _ in range(2)]
        ops.gather_cache_fp8(*rows, *self.cache, self.table, starts_of(lens))
        return list(zip(*(x.double().split(lens) for x in rows)))


STEPS = [PROMPTS, [1, 1, 1, 1], [1, 0, 4, 1], [1, 1, 0, 30]]


@pytest.mark.parametrize(("D", "dtype", "layout", "interleaved"), [
    (64, BF, "NHD", False), (128, HF, "HND", True), (256, BF, "HND", False)])
def test_prompts_and_decodes(D, dtype, layout, interleaved):
    loop = Loop(D, dtype, layout, interleaved)
    history = [[] for _ in PROMPTS]
    for new in STEPS:
        loop.feed(new)
        loop.step(max(new))
        q, k, v = loop.split()  # rotated in place
        keys, T = loop.read(), sum(new)
        many = max(new) * HQ // HKV > 16
        want, tol = reference(q[:T], keys, new, 0.1, single=many and dtype == BF)
        assert_close(loop.out[:T], want, tol)
        t = 0
        for r, n in enumerate(new):
            history[r] += [(k[t + i].double(), v[t + i].double()) for i in range(n)]
            t += n
        for r, (kk, vv) in enumerate(keys):
            for got, j in ((kk, 0), (vv, 1)):
                true = torch.stack([h[j] for h in history[r]])
                # A code is off by half a step, 2^-4 of the value, each time it is
                # rounded (twice or more only below 2^-6 of the scale), or by half the
                # smallest step, 2^-10, in units of a scale at most 2^-7 of the largest.
                top = true.abs().amax().item()
                assert ((got - true).abs() <= 2.0**-4 * true.abs() + 4 * 2.0**-10 * 2.0**-7 * top).all()
    assert loop.seq.tolist() == [sum(s[r] for s in STEPS) for r in range(4)]


def test_captured_step():
    """A whole step in a graph, replayed as lengths and tokens change, against the
    eager step of another loop, bit for bit; on a stream of its own."""
    a, b = Loop(64, BF, "NHD", False), Loop(64, BF, "NHD", False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in (a, b):
            x.feed(PROMPTS)
            x.step(100)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        a.feed([1, 1, 1, 1])
        with torch.cuda.graph(graph, stream=side):
            a.step(4)
        b.feed([1, 1, 1, 1])
        for new in ([1, 1, 1, 1], [1, 0, 4, 1], [1, 1, 1, 0], [2, 3, 1, 0]):
            if new != [1, 1, 1, 1]:
                a.feed(new)
                b.feed(new)
            graph.replay()
            b.step(4)
            side.synchronize()
            T = sum(new)
            assert torch.equal(a.out[:T], b.out[:T]) and a.out[:T].abs().max() > 0
            assert torch.equal(a.seq, b.seq)
            for s, t in zip(a.cache, b.cache):
                assert torch.equal(s.view(torch.uint8), t.view(torch.uint8))


def test_opcheck():
    D = 64
    q, k = queries(5, HQ, D, BF, 1), queries(5, HKV, D, BF, 2)
    turns, _ = rotary.rotary_turns(D)
    pos = torch.arange(5, device=DEV)
    torch.library.opcheck(OPS.rotary_embedding.default, (
        torch.zeros_like(q), torch.zeros_like(k), q, k, pos, turns, False, 1.0, False))
    # opcheck's other utilities compare tensors in ways that 8-bit floating types lack.
    c = make_cache([60, 30], Hkv=HKV, D=D, block=16, seed=23)
    slots = torch.tensor([16, -1, 20, 21, 40], device=DEV)
    torch.library.opcheck(OPS.gather_cache_fp8.default, (
        torch.zeros_like(k), torch.zeros_like(k), *c.views, c.table, starts_of([2, 3]), None),
        test_utils=("test_faketensor",))
    torch.library.opcheck(OPS.paged_attn_fp8_fwd.default, (
        torch.zeros_like(q), q, *c.views, c.table, c.lens, starts_of([3, 2]), 3, 60, 0.125,
        workspace(D).fill_(0.0), 0, True), test_utils=("test_faketensor",))
    torch.library.opcheck(OPS.reshape_and_cache_fp8.default, (k, k, *c.views, slots),
                          test_utils=("test_faketensor",))


def compiled_step(codes, scale, table, slots, seq, starts, pool, out, ctx, new, free, pool_in, q, k,
                  v, pos, turns, ws):
    k_cache, v_cache = codes[:, 0].view(torch.float8_e4m3fn), codes[:, 1].view(torch.float8_e4m3fn)
    ops.build_step_tables(table, slots, seq, starts, pool, ctx, new, free, pool_in, 16)
    qr, kr = torch.empty_like(q), torch.empty_like(k)
    ops.rotary_embedding(qr, kr, q, k, pos, turns)
    ops.reshape_and_cache_fp8(kr, v, k_cache, v_cache, scale[0], scale[1], slots)
    ops.paged_attn_fp8_fwd(out, qr, k_cache, v_cache, scale[0], scale[1], table, seq, starts, 3, 64,
                           0.125, ws)
    return out * 2


def test_compiled_step_equals_eager():
    D, R = 64, 3
    turns, _ = rotary.rotary_turns(D)

    def state():
        new = torch.tensor([1, 3, 2], **I32)
        return [torch.zeros(8, 2, 16, HKV, D, dtype=torch.uint8, device=DEV),
                torch.zeros(2, 8, 1, HKV, dtype=torch.uint8, device=DEV), torch.zeros(R, 4, **I32),
                torch.zeros(6, dtype=torch.int64, device=DEV), torch.zeros(R, **I32),
                torch.zeros(R + 1, **I32), torch.zeros(2, **I32),
                torch.zeros(6, HQ, D, dtype=BF, device=DEV), torch.zeros(R, **I32), new,
                torch.arange(1, 8, **I32), torch.zeros(2, **I32), queries(6, HQ, D, BF, 1),
                queries(6, HKV, D, BF, 2), queries(6, HKV, D, BF, 3),
                torch.tensor([0, 0, 1, 2, 0, 1], device=DEV), turns, workspace(D).fill_(0.0)]

    a, b = state(), state()
    x = torch.compile(compiled_step, backend="aot_eager", fullgraph=True)(*a)
    y = compiled_step(*b)
    torch.cuda.synchronize()
    assert torch.equal(x, y) and x.abs().max() > 0
    for s, t in zip(a[:8], b[:8]):
        assert torch.equal(s, t)


def test_two_streams_at_once():
    """Calls on two streams that may run at the same time, a workspace each."""
    c = make_cache([3000, 900], Hkv=HKV, D=64, block=16, seed=3)
    q = queries(6, HQ, 64, BF, 3)
    want = torch.empty_like(q)
    args = (*c.views, c.table, c.lens, starts_of([2, 4]), 4, 3000, 0.1)
    ops.paged_attn_fp8_fwd(want, q, *args, workspace(64))
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, spaces = [torch.zeros_like(q) for _ in range(2)], [workspace(64) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w in zip(streams, outs, spaces):
            with torch.cuda.stream(s):
                ops.paged_attn_fp8_fwd(o, q, *args, w)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
