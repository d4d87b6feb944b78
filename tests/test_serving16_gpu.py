"""The ops of a 16-bit cache together, as a serving loop uses them: the tables of
an encoder's states and of each decode step, the writes, attention over the
decoder's own cache and over the encoder's; eager, and as a captured graph of
two steps that hand lengths and the pool's cursor to each other."""

from __future__ import annotations

import pytest
import torch

from paged16_cases import DEV, assert_close, reference, workspace
from pth_flash_attn import ops
from pth_flash_attn.cache import paged16_views

pytestmark = pytest.mark.gpu
HQ, HKV, BLOCK, WIDTH, PAGES = 8, 2, 16, 8, 64
ENC = [37, 0, 150, 9]
I32 = dict(dtype=torch.int32, device=DEV)


class Loop:
    """Buffers of one model layer with self and cross attention; request 3 of 5
    brings no token in odd steps, request 4 is padding."""

    def __init__(self, D, dtype, seed, layout):
        self.D, self.dtype, self.R = D, dtype, 5
        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        shape = (PAGES, 2, BLOCK, HKV, D) if layout == "NHD" else (PAGES, 2, HKV, BLOCK, D)
        nan = float("nan")
        self.self_kv = torch.full(shape, nan, dtype=dtype, device=DEV)
        self.enc_kv = torch.full(shape, nan, dtype=dtype, device=DEV)
        self.self_views = paged16_views(self.self_kv, layout=layout)
        self.enc_views = paged16_views(self.enc_kv, layout=layout)
        R = self.R
        self.table = torch.zeros(R, WIDTH, **I32)
        self.enc_table = torch.zeros(R, 12, **I32)
        self.lens = [torch.zeros(R, **I32), torch.zeros(R, **I32)]
        self.pool = [torch.zeros(2, **I32), torch.zeros(2, **I32)]
        self.new = [torch.tensor([1, 1, 1, 1, 0], **I32), torch.tensor([1, 1, 1, 0, 0], **I32)]
        self.free = torch.randperm(PAGES - 1, generator=self.gen, device=DEV).to(torch.int32) + 1
        self.slots = torch.zeros(R, dtype=torch.int64, device=DEV)
        self.starts = torch.zeros(R + 1, **I32)
        self.enc_lens = torch.zeros(R, **I32)
        self.ws, self.ws2 = workspace(D), workspace(D)
        # Row t of the step's projections belongs to the t-th token; attention
        # of one token per request reads row r, so every request has its row.
        self.qkv = [torch.zeros(R, HQ + 2 * HKV, D, dtype=dtype, device=DEV) for _ in range(2)]
        self.out = [torch.zeros(R, HQ, D, dtype=dtype, device=DEV) for _ in range(2)]
        self.cross = [torch.zeros(R, HQ, D, dtype=dtype, device=DEV) for _ in range(2)]
        self.history = [[] for _ in range(R)]
        self.encode()

    def encode(self):
        """All encoder states, in one step of their own tables."""
        T = sum(ENC)
        self.enc_k = torch.randn(T, HKV, self.D, generator=self.gen, device=DEV)
        self.enc_v = torch.randn(T, HKV, self.D, generator=self.gen, device=DEV)
        slots = torch.zeros(T + 3, dtype=torch.int64, device=DEV)
        starts, pool = torch.zeros(self.R + 1, **I32), torch.zeros(2, **I32)
        free = torch.arange(PAGES - 1, 0, -1, **I32)
        ops.build_step_tables(self.enc_table, slots, self.enc_lens, starts, pool,
                              torch.zeros(self.R, **I32), torch.tensor(ENC + [0], **I32), free,
                              torch.zeros(2, **I32), BLOCK)
        pad = torch.zeros(3, HKV, self.D, device=DEV)
        ops.reshape_and_cache_16bit(torch.cat([self.enc_k, pad]), torch.cat([self.enc_v, pad]),
                                    *self.enc_views, slots)
        assert self.enc_lens.tolist() == ENC + [0]
        at, self.enc_keys = 0, []
        for n in ENC + [0]:
            self.enc_keys.append((self.enc_k[at : at + n].to(self.dtype),
                                  self.enc_v[at : at + n].to(self.dtype)))
            at += n

    def step(self, i):
        """Step i (0 or 1 of the pair): tokens are packed in request order, and
        here every active request's index is its token's, as requests 0..3."""
        q, k, v = self.qkv[i].split([HQ, HKV, HKV], dim=1)
        ops.build_step_tables(self.table, self.slots, self.lens[1 - i], self.starts,
                              self.pool[1 - i], self.lens[i], self.new[i], self.free,
                              self.pool[i], BLOCK)
        ops.reshape_and_cache_16bit(k, v, *self.self_views, self.slots)
        ops.paged_decode_fwd(self.out[i], q, *self.self_views, self.table, self.lens[1 - i],
                             WIDTH * BLOCK, 0.1, self.ws)
        ops.cross_attn_fwd(self.cross[i], q, *self.enc_views, self.enc_table, self.enc_lens,
                           self.starts, 1, 12 * BLOCK, 0.1, self.ws2)

    def feed(self, i):
        self.qkv[i].copy_(torch.randn(self.qkv[i].shape, generator=self.gen, device=DEV))

    def check(self, i):
        new = self.new[i].tolist()
        q, k, v = self.qkv[i].split([HQ, HKV, HKV], dim=1)
        for r in range(self.R):
            if new[r]:
                self.history[r].append((k[r].clone(), v[r].clone()))
        none = torch.zeros(0, HKV, self.D, dtype=self.dtype, device=DEV)
        keys = [(torch.stack([a for a, _ in h]), torch.stack([b for _, b in h])) if h
                else (none, none) for h in self.history]
        assert_close(self.out[i], *reference(q, keys, [1] * self.R, 0.1, pair=True))
        T = sum(new)
        want, tol = reference(q[:T], self.enc_keys, new, 0.1, pair=True)
        assert_close(self.cross[i][:T], want, tol)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_eager_loop(D, dtype, layout):
    loop = Loop(D, dtype, D, layout)
    for n in range(40):
        loop.feed(n & 1)
        loop.step(n & 1)
        loop.check(n & 1)
    assert loop.lens[0].tolist() == [40, 40, 40, 20, 0]
    assert loop.pool[0].tolist() == [3 * 3 + 2, 0]
    assert loop.self_kv[0].isnan().all() and loop.enc_kv[0].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
def test_captured_pair_of_steps(D):
    loop = Loop(D, torch.bfloat16, 7, "NHD")
    state = [loop.table, loop.self_kv, *loop.lens, *loop.pool]
    before = [t.clone() for t in state]
    for i in (0, 1):
        loop.step(i)
    torch.cuda.synchronize()
    for t, b in zip(state, before):
        t.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in (0, 1):
            loop.step(i)
    for _ in range(15):
        loop.feed(0)
        loop.feed(1)
        graph.replay()
        torch.cuda.synchronize()
        loop.check(0)
        loop.check(1)
    assert loop.lens[0].tolist() == [30, 30, 30, 15, 0]


def test_a_pool_that_runs_out():
    """Refused requests keep their lengths and attend to what they have."""
    loop = Loop(64, torch.bfloat16, 9, "NHD")
    loop.free = loop.free[:5].contiguous()
    for n in range(32):
        loop.feed(n & 1)
        loop.step(n & 1)
        if n < 16:
            loop.check(n & 1)
    # Requests 0..3 took one page each, request 0 the fifth at its 17th token;
    # 1 and 2 stay at 16 tokens, 3 has brought 16 by now.
    assert loop.lens[0].tolist() == [32, 16, 16, 16, 0]
    assert loop.pool[0].tolist() == [5, 2]
    assert not loop.out[1].isnan().any()
