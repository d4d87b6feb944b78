"""The 16-bit cache's ops under opcheck and torch.compile: a whole step (tables,
write, decode, cross attention) traced without graph breaks gives the eager
step's tensors bitwise, in place where the ops write in place."""

from __future__ import annotations

import pytest
import torch

from paged16_cases import DEV, make_cache, queries, starts_of, workspace
from pth_flash_attn import ops
from pth_flash_attn.cache import paged16_views

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
I32 = dict(dtype=torch.int32, device=DEV)
OPS = torch.ops.pth_flash_attn
HQ, HKV, D, BLOCK, PAGES = 8, 2, 64, 16, 24


def tables_args(R=3):
    return (torch.zeros(R, 4, **I32), torch.zeros(9, dtype=torch.int64, device=DEV),
            torch.zeros(R, **I32), torch.zeros(R + 1, **I32), torch.zeros(2, **I32),
            torch.tensor([3, 0, 16][:R], **I32), torch.tensor([1, 5, 1][:R], **I32),
            torch.arange(1, 9, **I32), torch.zeros(2, **I32), BLOCK)


def test_opcheck_tables():
    torch.library.opcheck(OPS.build_step_tables.default, tables_args())


@pytest.mark.parametrize("one_buffer", [False, True])
def test_opcheck_writer(one_buffer):
    """Caches of two buffers, and the two views of one."""
    kv = torch.zeros(4, 2, BLOCK, HKV, D, dtype=BF, device=DEV)
    k, v = paged16_views(kv)
    if not one_buffer:
        k, v = k.contiguous(), v.contiguous()
    args = (queries(5, HKV, D, BF, 1), queries(5, HKV, D, BF, 2), k, v,
            torch.tensor([3, -1, 20, 21, 40], device=DEV))
    torch.library.opcheck(OPS.reshape_and_cache_16bit.default, args)


def test_opcheck_attention():
    c = make_cache([60, 30], Hkv=HKV, D=D, block=BLOCK, dtype=BF, seed=23)
    q, ws = queries(2, HQ, D, BF, 23), workspace(D).fill_(0.0)
    torch.library.opcheck(OPS.paged_decode_fwd.default, (
        torch.zeros_like(q), q, c.k, c.v, c.table, c.lens, 60, 0.125, ws, 0))
    torch.library.opcheck(OPS.cross_attn_fwd.default, (
        torch.zeros_like(q), q, c.k, c.v, c.table, c.lens, starts_of([1, 1]), 1, 60, 0.125, ws))


class State:
    """A step's buffers; `free` hands page 1 on out in order."""

    def __init__(self, R):
        self.R = R
        gen = torch.Generator(device=DEV).manual_seed(R)
        self.kv = torch.zeros(PAGES, 2, BLOCK, HKV, D, dtype=BF, device=DEV)
        self.table, self.slots = torch.zeros(R, 4, **I32), torch.zeros(R, dtype=torch.int64,
                                                                       device=DEV)
        self.seq, self.starts, self.pool = (torch.zeros(n, **I32) for n in (R, R + 1, 2))
        self.ctx, self.new, self.pool_in = (torch.zeros(n, **I32) for n in (R, R, 2))
        self.new.fill_(1)
        self.free = torch.arange(1, PAGES, **I32)
        self.qkv = torch.randn(R, HQ + 2 * HKV, D, generator=gen, device=DEV).to(BF)
        self.enc = make_cache([70 + i for i in range(R)], Hkv=HKV, D=D, block=BLOCK, dtype=BF,
                              seed=R)
        self.out, self.ws = torch.zeros(R, HQ, D, dtype=BF, device=DEV), workspace(D).fill_(0.0)

    def tensors(self):
        return (self.kv, self.table, self.slots, self.seq, self.starts, self.pool, self.out)


def step(kv, table, slots, seq, starts, pool, out, ctx, new, free, pool_in, qkv, enc_k, enc_v,
         enc_table, enc_lens, ws):
    k_cache, v_cache = paged16_views(kv)
    q, k, v = qkv.split([HQ, HKV, HKV], dim=1)
    ops.build_step_tables(table, slots, seq, starts, pool, ctx, new, free, pool_in, BLOCK)
    ops.reshape_and_cache_16bit(k, v, k_cache, v_cache, slots)
    ops.paged_decode_fwd(out, q, k_cache, v_cache, table, seq, 64, 0.125, ws)
    own = out * 2
    # In place: the first layer's output is the second's query.
    ops.cross_attn_fwd(out, out, enc_k, enc_v, enc_table, enc_lens, starts, 1, 100, 0.125, ws)
    return own + out


def call(f, s):
    e = s.enc
    return f(*s.tensors(), s.ctx, s.new, s.free, s.pool_in, s.qkv, e.k, e.v, e.table, e.lens, s.ws)


@pytest.mark.parametrize("R", [1, 3, 7])
def test_compiled_step_equals_eager(R):
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    a, b = State(R), State(R)
    for n in range(3):
        x, y = call(compiled, a), call(step, b)
        torch.cuda.synchronize()
        assert torch.equal(x, y) and x.abs().max() > 0
        for s, t in zip(a.tensors(), b.tensors()):
            assert torch.equal(s, t)
        for s in (a, b):  # the next step
            s.ctx.copy_(s.seq)
            s.pool_in.copy_(s.pool)
            s.qkv.add_(0.25 * n + 0.5)
    assert a.seq.tolist() == [3] * R and a.pool.tolist() == [R, 0]
