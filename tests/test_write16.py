"""reshape_and_cache_16bit: the cache's bytes, and its refusals."""

from __future__ import annotations

import math

import pytest
import torch

from pth_flash_attn import ops
from pth_flash_attn.cache import paged16_views

needs_op = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def cache(pages, block, Hkv, D, dtype, layout, device="cuda"):
    inner = (block, Hkv, D) if layout == "NHD" else (Hkv, block, D)
    kv = torch.full((pages, 2, *inner), 3.0, dtype=dtype, device=device)
    return kv, *paged16_views(kv, layout=layout)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize(("src", "dst"), [(BF, BF), (HF, HF), (F32, BF), (F32, HF)])
@pytest.mark.parametrize("layout", ["NHD", "HND"])
@pytest.mark.parametrize("odd", [False, True])
def test_bytes(D, src, dst, layout, odd):
    """Every written value, every other byte untouched; ``odd``: source rows
    off 16-byte addresses, pages of 7 slots, 3 heads."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    T, Hkv, block, pages = 61, 3, 7 if odd else 16, 12
    wide = 1e30 if dst == BF else 1e3
    data = torch.randn(T, 2 * Hkv * D + 9, generator=gen, device="cuda") * wide
    data[0, :40] = torch.tensor([math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-41, 65519.9, 65520.0],
                                device="cuda").repeat(5)
    data = data.to(src)
    at = 1 if odd else 0
    row = 2 * Hkv * D + (9 if odd else 0)
    data = data if odd else data[:, :row].contiguous()
    key = data[:, at : at + Hkv * D].view(T, Hkv, D)
    value = data[:, at + Hkv * D : at + 2 * Hkv * D].view(T, Hkv, D)
    kv, k, v = cache(pages, block, Hkv, D, dst, layout)
    slots = torch.randperm(pages * block, generator=gen, device="cuda")[:T]
    slots[[3, 30]] = -1
    slots[[5, 31]] = torch.tensor([pages * block, 1 << 40], device="cuda")
    want = kv.clone()
    wk, wv = paged16_views(want, layout=layout)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * block:
            wk[s // block, s % block] = key[t].to(dst)
            wv[s // block, s % block] = value[t].to(dst)
    ops.reshape_and_cache_16bit(key, value, k, v, slots)
    assert torch.equal(kv.isnan(), want.isnan())
    nan = want.isnan()
    assert torch.equal(kv.masked_fill(nan, 0).view(torch.int16),
                       want.masked_fill(nan, 0).view(torch.int16))


@pytest.mark.gpu
def test_no_tokens_and_one():
    kv, k, v = cache(2, 16, 1, 64, BF, "NHD")
    e = torch.empty(0, 1, 64, dtype=BF, device="cuda")
    ops.reshape_and_cache_16bit(e, e, k, v, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert (kv == 3).all()
    x = torch.ones(1, 1, 64, dtype=BF, device="cuda")
    ops.reshape_and_cache_16bit(x, 2 * x, k, v, torch.tensor([17], device="cuda"))
    assert (k[1, 1] == 1).all() and (v[1, 1] == 2).all() and (kv == 3).sum() == kv.numel() - 128


def _cpu(D=64, T=4, Hkv=2):
    kv, k, v = cache(2, 16, Hkv, D, BF, "NHD", "cpu")
    x = torch.zeros(T, Hkv, D, dtype=BF)
    return dict(key=x, value=x.clone(), k_cache=k, v_cache=v,
                slot_mapping=torch.zeros(T, dtype=torch.int64))


@needs_op
@pytest.mark.parametrize(("change", "message"), [
    (lambda a: {}, "computes on CUDA tensors only"),
    (lambda a: dict(key=a["key"][0]), "must be 3-D"),
    (lambda a: dict(value=a["value"][:3]), "must have the same shape"),
    (lambda a: dict(key=a["key"][..., :32], value=a["value"][..., :32]), "head size must be"),
    (lambda a: dict(k_cache=a["k_cache"][..., :1, :]), "k_cache and v_cache must be"),
    (lambda a: dict(k_cache=a["k_cache"].half()), "must both be bfloat16 or float16"),
    (lambda a: dict(key=a["key"].half(), value=a["value"].half()), "float32 or have the dtype"),
    (lambda a: dict(key=a["key"].float()), "float32 or have the dtype"),
    (lambda a: dict(slot_mapping=a["slot_mapping"].int()), "slot_mapping must be"),
    (lambda a: dict(slot_mapping=a["slot_mapping"][:3]), "slot_mapping must be"),
    (lambda a: dict(k_cache=a["k_cache"][:0], v_cache=a["v_cache"][:0]), "must not be empty"),
    (lambda a: dict(key=torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)), "stride 1"),
])
def test_refusals(change, message):
    args = _cpu()
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.reshape_and_cache_16bit(**args)
    if "CUDA" not in message:
        with pytest.raises(RuntimeError, match=message):
            ops.ops16.reshape_and_cache_16bit_fake(**args)


@pytest.mark.gpu
def test_unaligned_cache_is_refused():
    flat = torch.zeros(2 * 2 * 16 * 64 + 4, dtype=BF, device="cuda")
    kv = flat[4:].view(2, 2, 16, 1, 64)
    x = torch.zeros(1, 1, 64, dtype=BF, device="cuda")
    with pytest.raises(RuntimeError, match="16-byte aligned rows"):
        ops.reshape_and_cache_16bit(x, x, kv[:, 0], kv[:, 1], torch.tensor([1], device="cuda"))


@needs_op
def test_cache_that_overlaps_itself_is_refused():
    args = _cpu()
    for bad in (dict(k_cache=args["k_cache"][:, :, :1].expand_as(args["k_cache"])),
                dict(v_cache=args["v_cache"][:1].expand_as(args["v_cache"]))):
        for f in (ops.reshape_and_cache_16bit, ops.ops16.reshape_and_cache_16bit_fake):
            with pytest.raises(RuntimeError, match="must not overlap themselves"):
                f(**{**args, **bad})
