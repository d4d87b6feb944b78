"""reshape_and_cache_fp8 and gather_cache_fp8: bit for bit, and their refusals."""

from __future__ import annotations

import math

import pytest
import torch

from fp8_cases import (FP8, SPAN, assert_codes, exponent_for, make_cache, power, starts_of, storage,
                       write_reference)
from pth_flash_attn import ops
from pth_flash_attn.cache import fp8_cache

needs_op = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def source(T, Hkv, D, dtype, seed, odd=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    row = 2 * Hkv * D + (9 if odd else 8)
    data = torch.randn(T, row, generator=gen, device="cuda")
    # Values over some binades, tokens and channels of their own size.
    data *= torch.exp2(torch.randint(-6, 7, (T, 1), generator=gen, device="cuda").float())
    data *= torch.exp2(torch.randint(-3, 4, (1, row), generator=gen, device="cuda").float())
    at = 1 if odd else 0
    data = data.to(dtype)
    return (data[:, at : at + Hkv * D].view(T, Hkv, D),
            data[:, at + Hkv * D : at + 2 * Hkv * D].view(T, Hkv, D))


def filled(pages, block, Hkv, D, layout, seed, pad=0):
    """A cache of any codes (NaN among them) and exponents, 0 and those above 246
    among them."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes, k, v, ks, vs = storage(pages, block, Hkv, D, layout, fill=0, pad=pad)
    codes.copy_(torch.randint(0, 256, codes.shape, generator=gen, device="cuda").to(torch.uint8))
    for s in (ks, vs):
        s.copy_(torch.randint(100, 140, s.shape, generator=gen, device="cuda").to(torch.uint8))
        s.view(-1)[::7] = 0
        s.view(-1)[3::29] = 255
    return codes, k, v, ks, vs


def check_write(key, value, cache, slots):
    codes, k, v, ks, vs = cache
    want = write_reference(key, value, k, v, ks, vs, slots)
    before = codes.clone()
    ops.reshape_and_cache_fp8(key, value, k, v, ks, vs, slots)
    assert_codes(k.view(torch.uint8), want[0])
    assert_codes(v.view(torch.uint8), want[1])
    assert torch.equal(ks.cpu(), want[2]) and torch.equal(vs.cpu(), want[3])
    return before


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("odd", [False, True])
def test_write(D, dtype, layout, odd):
    """Blocks begun, continued, filled, in part and out of order; ``odd``: source
    rows off 16-byte addresses, pages of 48 slots with a gap behind each."""
    block, Hkv, pages = (48, 3, 9) if odd else (16, 2, 24)
    key, value = source(150, Hkv, D, dtype, D, odd)
    gen = torch.Generator(device="cuda").manual_seed(D + odd)
    slots = torch.randperm(pages * block, generator=gen, device="cuda")[:150]
    slots[40:100] = torch.arange(60, device="cuda") + 5 * SPAN + 3  # a run
    slots[[3, 30, 120]] = torch.tensor([-1, pages * block, 1 << 40], device="cuda")
    check_write(key, value, filled(pages, block, Hkv, D, layout, 7, 16 * odd), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 63, 129, 1000, 5000])
def test_orders(T):
    """Tokens of a block anywhere in the call, slots given twice (the last one
    counts), more tokens than a work-group takes."""
    Hkv, D, block = 2, 64, 32
    key, value = source(T, Hkv, D, BF, T)
    pages = max(2, T // 24)
    gen = torch.Generator(device="cuda").manual_seed(T)
    slots = torch.randint(-3, pages * block + 3, (T,), generator=gen, device="cuda")
    check_write(key, value, filled(pages, block, Hkv, D, "NHD", T), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("odd", [False, True])
def test_write_many(D, dtype, odd):
    """As many tokens as give a work-group all heads: runs of blocks, their tokens in
    order but for some that stand elsewhere in the call, padding between."""
    block, Hkv, T = (48, 3, 4997) if odd else (16, 1, 4200)
    key, value = source(T, Hkv, D, dtype, D + 1, odd)
    pages = T // block + 9
    gen = torch.Generator(device="cuda").manual_seed(D + odd)
    slots = torch.arange(T, device="cuda") + 21
    moved = torch.randperm(T, generator=gen, device="cuda")[:200]
    slots[moved] = slots[moved.roll(1)]
    slots[77::501] = -1
    slots[78::503] = slots[5]
    check_write(key, value, filled(pages, block, Hkv, D, "HND" if odd else "NHD", 8, 16 * odd), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T", [40, 1500, 4095, 4096])
def test_first_row_not_finite(D, dtype, T):
    """The first token's row is infinite and NaN: blocks with fewer tokens than slots keep
    it out, and their other values are of the largest finite size here and there."""
    key, value = source(T, 3, D, dtype, D + T)
    key[0], value[0] = math.nan, -math.inf
    big = torch.finfo(dtype).max
    key[5::97, 1, 3], value[7::101, 2, 1] = big, -big
    slots = torch.arange(T, device="cuda") * 5 // 2 + 3  # six or seven of a block's slots
    check_write(key, value, filled(T * 5 // 32 + 2, 16, 3, D, "NHD", T), slots)


@pytest.mark.gpu
def test_write_longest_runs():
    """The most tokens of a work-group, each in a block of its own."""
    T = 34000
    key, value = source(T, 1, 64, BF, 12)
    slots = 16 * torch.randperm(T, generator=torch.Generator().manual_seed(1)).cuda() + 3
    check_write(key, value, filled(T, 16, 1, 64, "NHD", 9), slots)


@pytest.mark.gpu
def test_growth_and_begin():
    """A block's scale grows with its tokens and not back; its first slot begins
    it anew."""
    D, Hkv = 64, 1
    k, v, ks, vs = fp8_cache(2, 16, Hkv, D)
    sizes = [1.0, 1.0, 3.0, 1000.0, 1e-3, 5e4, 1.0]
    held = []
    for i, size in enumerate(sizes):
        x = torch.full((1, Hkv, D), size, device="cuda")
        ops.reshape_and_cache_fp8(x, -x, k, v, ks, vs, torch.tensor([16 + i], device="cuda"))
        held.append(int(ks[1, 0, 0]))
    need = [int(exponent_for(torch.tensor(s, dtype=torch.float64))) for s in sizes]
    assert held == [max(need[: i + 1]) for i in range(len(sizes))]
    x = k[1, : len(sizes), 0].double() * power(ks[1, 0, 0])
    # Each was rounded once or, when the block grew, again: a step each, of 2^-4 of
    # the value or half the smallest code in the final scale.
    for i, size in enumerate(sizes):
        step = max(2.0**-4 * size * 2, 2.0**-9 * 2.0 ** (held[-1] - 127))
        assert (x[i] - size).abs().max().item() <= step
    one = torch.ones(1, Hkv, D, device="cuda")
    rest = k[1, 1:].view(torch.uint8).clone()
    ops.reshape_and_cache_fp8(one, one, k, v, ks, vs, torch.tensor([16], device="cuda"))
    assert int(ks[1, 0, 0]) == need[0] and (k[1, 0].float() == 256.0).all()
    assert torch.equal(k[1, 1:].view(torch.uint8), rest)
    assert int(ks[0, 0, 0]) == 0 and not k[0].view(torch.uint8).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_extremes(dtype):
    """Zeros, infinities, NaN, the type's smallest and largest values, and those at
    the edge of a binade's codes, each in a block of its own beside ones."""
    info = torch.finfo(dtype)
    tiny = float(torch.tensor(info.smallest_normal / 2**3).to(dtype))
    vals = [0.0, -0.0, math.inf, -math.inf, math.nan, tiny, info.smallest_normal, info.max, info.min,
            448.0, 449.0, 450.0, 464.0, 1.75, 1.7578125, 2.0**-9, 1e-7, 3e-39, 1e38]
    D, n = 64, len(vals)
    x = torch.zeros(2 * n, 1, D, dtype=torch.float64)
    x[:n, 0] = torch.tensor(vals, dtype=torch.float64)[:, None]  # alone
    x[n:, 0, 1] = torch.tensor(vals, dtype=torch.float64)  # beside zeros and a one
    x[n:, 0, 0] = 1.0
    x = x.to(dtype).cuda()
    slots = torch.arange(2 * n, device="cuda") * 16
    check_write(x, -x, filled(2 * n, 16, 1, D, "NHD", 1), slots)
    check_write(x, -x, filled(2 * n, 16, 1, D, "NHD", 2), slots + 5)


@pytest.mark.gpu
def test_write_nothing():
    cache = filled(2, 16, 1, 64, "NHD", 3)
    e = torch.empty(0, 1, 64, dtype=BF, device="cuda")
    check_write(e, e, cache, torch.empty(0, dtype=torch.int64, device="cuda"))
    x = torch.ones(3, 1, 64, dtype=BF, device="cuda")
    check_write(x, x, cache, torch.tensor([-1, 32, -(1 << 62)], device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
def test_gather(D, dtype, layout):
    """Each value rounded once; requests of no tokens, from inside blocks, behind
    their pages; rows of no request untouched."""
    lens = [5, 0, 77, 1, 130]
    c = make_cache(lens, Hkv=3, D=D, block=32, seed=D, layout=layout, spread=40, pad=16)
    first = [0, 0, 33, 0, 17]
    n = [5, 0, 44, 1, 100]
    starts = starts_of(n) + 2
    T = sum(n) + 5
    outs = [torch.full((T, 3, D), 7.0, dtype=dtype, device="cuda") for _ in range(2)]
    ops.gather_cache_fp8(*outs, *c.views, c.table, starts,
                         torch.tensor(first, dtype=torch.int32, device="cuda"))
    for out, j in ((outs[0], 0), (outs[1], 1)):
        want = torch.cat([c.keys[r][j][first[r] : first[r] + n[r]] for r in range(5)])
        assert torch.equal(out[2 : 2 + len(want)], want.to(dtype))
        assert (out[:2] == 7).all() and (out[2 + len(want) :] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [(2100, 1, 2095), (4000, 0, 4999, 3)])
def test_gather_many(n):
    """Work-groups of more rows, which requests end inside of."""
    first = [3 + 16 * r for r in range(len(n))]
    c = make_cache([a + b for a, b in zip(first, n)], Hkv=3, D=64, block=16, seed=5, spread=40)
    outs = [torch.full((sum(n) + 1, 3, 64), 7.0, dtype=BF, device="cuda") for _ in range(2)]
    ops.gather_cache_fp8(*outs, *c.views, c.table, starts_of(n),
                         torch.tensor(first, dtype=torch.int32, device="cuda"))
    for out, j in ((outs[0], 0), (outs[1], 1)):
        want = torch.cat([c.keys[r][j][first[r] :] for r in range(len(n))])
        assert torch.equal(out[:-1], want.to(BF)) and (out[-1] == 7).all()


@pytest.mark.gpu
def test_gather_bounds():
    """Zeros where the table holds no page of the cache; scales at both ends."""
    c = make_cache([64], Hkv=1, D=64, block=16, seed=3)
    table = c.table.clone()
    table[0, 1], table[0, 2] = -1, c.k.shape[0]
    c.ks[table[0, 3].long()] = 0
    c.vs[table[0, 3].long()] = 255
    outs = [torch.full((100, 1, 64), 7.0, device="cuda") for _ in range(2)]
    starts = torch.tensor([0, 100], dtype=torch.int32, device="cuda")
    first = torch.tensor([-10], dtype=torch.int32, device="cuda")
    ops.gather_cache_fp8(*outs, *c.views, table, starts, first)
    kd, vd = (x.clone() for x in c.keys[0])
    kd[16:] = 0
    assert torch.equal(outs[0][10:74], kd.float())
    vd[16:48] = 0
    page = int(table[0, 3])
    vd[48:] = c.v[page].double() * power(torch.tensor(246, device="cuda"))
    assert torch.equal(outs[1][10:74], vd.float())
    for o in outs:
        assert not o[:10].any() and not o[74:].any()
    ops.gather_cache_fp8(*outs, *c.views, table, starts)  # from the first token on
    assert torch.equal(outs[0][:64], kd.float()) and not outs[0][64:].any()
    none = outs[0].clone()
    ops.gather_cache_fp8(outs[0][:0], outs[1][:0], *c.views, table, starts)
    ops.gather_cache_fp8(*outs, *c.views, table[:0], starts[:1])
    assert torch.equal(outs[0], none)


def _cpu(T=4):
    k, v, ks, vs = fp8_cache(2, 32, 2, 64, device="cpu")
    x = torch.zeros(T, 2, 64, dtype=BF)
    return dict(key=x, value=x.clone(), k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)


BOTH = [
    (lambda a: {}, "computes on CUDA tensors only"),
    (lambda a: dict(key=a["key"][0]), "must be 3-D"),
    (lambda a: dict(value=a["value"][:3]), "must have the same shape"),
    (lambda a: dict(key=a["key"][..., :32], value=a["value"][..., :32]), "k_cache and v_cache must be"),
    (lambda a: dict(key=a["key"][..., :32], value=a["value"][..., :32], k_cache=a["k_cache"][..., :32],
                    v_cache=a["v_cache"][..., :32]), "head size must be"),
    (lambda a: dict(k_cache=a["k_cache"].view(torch.uint8)), "must be float8_e4m3fn"),
    (lambda a: dict(k_cache=a["k_cache"][:0], v_cache=a["v_cache"][:0]), "must not be empty"),
    (lambda a: dict(k_cache=a["k_cache"][:, :24], v_cache=a["v_cache"][:, :24]), "multiple of 16"),
    (lambda a: dict(k_scale=a["k_scale"].float()), "k_scale and v_scale must be"),
    (lambda a: dict(v_scale=a["v_scale"][:, :1]), "k_scale and v_scale must be"),
    (lambda a: dict(key=a["key"][:, :1], value=a["value"][:, :1]), "the cache's heads"),
    (lambda a: dict(key=a["key"].double(), value=a["value"].double()), "must both be float32"),
    (lambda a: dict(key=torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)), "stride 1"),
]


@needs_op
@pytest.mark.parametrize(("change", "message"), BOTH + [
    (lambda a: dict(slot_mapping=a["slot_mapping"].int()), "slot_mapping must be"),
    (lambda a: dict(slot_mapping=a["slot_mapping"][:3]), "slot_mapping must be"),
    (lambda a: dict(k_cache=a["k_cache"][:, :, :1].expand_as(a["k_cache"])), "overlap themselves"),
])
def test_write_refusals(change, message):
    args = dict(_cpu(), slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.reshape_and_cache_fp8(**args)
    if "CUDA" not in message:
        with pytest.raises(RuntimeError, match=message):
            ops.ops8.reshape_and_cache_fp8_fake(**args)


@needs_op
@pytest.mark.parametrize(("change", "message"), BOTH + [
    (lambda a: dict(row_start_loc=a["row_start_loc"].long()), "row_start_loc must be"),
    (lambda a: dict(row_start_loc=a["row_start_loc"][:0]), "row_start_loc must be"),
    (lambda a: dict(block_table=a["block_table"][:1]), "block_table must be"),
    (lambda a: dict(block_table=a["block_table"].t().contiguous().t()), "block_table must be"),
    (lambda a: dict(first=torch.zeros(3, dtype=torch.int32)), "first must be"),
    (lambda a: dict(first=torch.zeros(2, dtype=torch.int64)), "first must be"),
    (lambda a: dict(value=a["value"][:1].expand_as(a["value"])), "overlap themselves"),
])
def test_gather_refusals(change, message):
    args = dict(_cpu(), block_table=torch.zeros(2, 3, dtype=torch.int32),
                row_start_loc=torch.zeros(3, dtype=torch.int32))
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.gather_cache_fp8(**args)
    if "CUDA" not in message:
        with pytest.raises(RuntimeError, match=message):
            ops.ops8.gather_cache_fp8_fake(**args)


@needs_op
def test_shared_memory_refused():
    a = dict(_cpu(), slot_mapping=torch.zeros(4, dtype=torch.int64))
    one = torch.zeros(2, 2, 32, 2, 64, dtype=torch.uint8).view(FP8)
    scale = torch.zeros(2, 2, 2, 2, dtype=torch.uint8)
    for bad, message in (
            (dict(k_cache=one[:, 0], v_cache=one[:, 0]), "share no memory"),
            (dict(k_scale=scale[0], v_scale=scale[0]), "scales must not overlap"),
            (dict(k_cache=one[:, 0], key=one.view(-1)[:1024].view(BF).view(4, 2, 64)),
             "must not overlap an input")):
        with pytest.raises(RuntimeError, match=message):
            ops.reshape_and_cache_fp8(**{**a, **bad})
    g = dict(_cpu(), block_table=torch.zeros(2, 3, dtype=torch.int32),
             row_start_loc=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="share no memory"):
        ops.gather_cache_fp8(**{**g, "value": g["key"]})
    with pytest.raises(RuntimeError, match="must not overlap an input"):
        ops.gather_cache_fp8(**{**g, "row_start_loc": g["key"].view(-1).view(torch.int32)[:3]})


@pytest.mark.gpu
def test_unaligned_rows_refused():
    flat = torch.zeros(2 * 2 * 16 * 64 + 8, dtype=torch.uint8, device="cuda")
    kv = flat[8:].view(2, 2, 16, 1, 64).view(FP8)
    scale = torch.zeros(2, 2, 1, 1, dtype=torch.uint8, device="cuda")
    x = torch.zeros(1, 1, 64, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="16-byte aligned rows"):
        ops.reshape_and_cache_fp8(x, x, kv[:, 0], kv[:, 1], scale[0], scale[1],
                                  torch.tensor([1], device="cuda"))
    k, v, ks, vs = fp8_cache(2, 16, 1, 64)
    y = torch.zeros(68, dtype=BF, device="cuda")[4:].view(1, 1, 64)
    with pytest.raises(RuntimeError, match="16-byte aligned rows"):
        ops.gather_cache_fp8(y, x, k, v, ks, vs, torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
                             torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
