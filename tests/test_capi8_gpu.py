"""The C entries of rotary positions and the 8-bit floating cache on data: what the
structs' fields say is what the torch ops do, bit for bit, over strided tensors."""

from __future__ import annotations

import math

import pytest
import torch

from fp8_cases import make_cache, queries, starts_of, storage, workspace
from pth_flash_attn import capi, ops, rotary

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def call(what, args):
    lib = capi.AttnLib()
    torch.cuda.synchronize()
    lib.check(getattr(lib, what)(args, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()


def cut(T, H, D, dtype, seed, before=1, behind=2):
    """Rows of a wider buffer: [T, H, D] with strides of their own."""
    return queries(T, before + H + behind, D, dtype, seed)[:, before : before + H]


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize(("interleaved", "inverse", "scale", "rot", "Hkv"), [
    (False, False, 1.0, 64, 2), (True, False, 1.25, 48, 1), (False, True, 0.5, 20, 3),
    (True, True, 1.0, 64, 0)])
def test_rotary(dtype, interleaved, inverse, scale, rot, Hkv):
    q, k = cut(37, 5, 64, dtype, 1), cut(37, Hkv, 64, dtype, 2, before=2)
    turns, _ = rotary.rotary_turns(rot)
    pos = torch.arange(37, device="cuda") * 1009
    outs = []
    for via in ("op", "c"):
        q_out = torch.full_like(queries(37, 9, 64, dtype, 3), math.nan)
        k_out = torch.full((37, Hkv + 1, 64), math.nan, dtype=dtype, device="cuda")
        a, b = q_out[:, 3:8], k_out[:, 1:]
        if via == "op":
            ops.rotary_embedding(a, b, q, k, pos, turns, interleaved, scale, inverse)
        else:
            call("rotary", capi.rotary_args(q_out=a, k_out=b, q=q, k=k, positions=pos, turns=turns,
                                            interleaved=interleaved, scale=scale, inverse=inverse))
        assert not a.isnan().any() and q_out[:, :3].isnan().all() and q_out[:, 8:].isnan().all()
        outs.append((a.clone(), b.clone()))
    assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize(("D", "layout", "block"), [(64, "NHD", 16), (128, "HND", 48), (256, "NHD", 32)])
def test_write_and_gather(dtype, D, layout, block):
    T, Hkv, pages = 61, 3, 9
    key, value = cut(T, Hkv, D, dtype, 4), cut(T, Hkv, D, dtype, 5, before=0, behind=1)
    slots = torch.arange(T, device="cuda") + block + 3
    slots[::7] = -1
    table = torch.arange(1, pages, dtype=torch.int32, device="cuda").repeat(2, 1)[:, : pages - 2]
    starts = starts_of([20, 41])
    first = torch.tensor([3, 5], dtype=torch.int32, device="cuda")
    got = []
    for via in ("op", "c"):
        codes, k, v, ks, vs = storage(pages, block, Hkv, D, layout, fill=0, pad=32)
        ks.zero_(), vs.zero_()
        cache = dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)
        rows = [torch.full((T + 2, Hkv + 1, D), 7.0, dtype=dtype, device="cuda") for _ in range(4)]
        views = [x[:, 1:] for x in rows]
        if via == "op":
            ops.reshape_and_cache_fp8(key, value, **cache, slot_mapping=slots)
            ops.gather_cache_fp8(*views[:2], **cache, block_table=table, row_start_loc=starts,
                                 first=first)
            ops.gather_cache_fp8(*views[2:], **cache, block_table=table, row_start_loc=starts)
        else:
            call("write_f8", capi.write_f8_args(key=key, value=value, slot_mapping=slots, **cache))
            common = dict(block_table=table, row_start_loc=starts, **cache)
            call("gather_f8", capi.gather_f8_args(key=views[0], value=views[1], first=first, **common))
            call("gather_f8", capi.gather_f8_args(key=views[2], value=views[3], **common))
        assert ks.any() and vs.any() and views[0][:T].any()
        assert all((x[T:] == 7.0).all() and (x[:, 0] == 7.0).all() for x in rows)
        got.append((codes.clone(), ks.clone(), vs.clone(), *rows))
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize(("D", "layout", "block"), [(64, "NHD", 16), (128, "HND", 48), (256, "NHD", 32)])
@pytest.mark.parametrize("kw", [dict(), dict(window=70), dict(causal=False), dict(decode=True),
                                dict(decode=True, window=33), dict(max_query_len=1)])
def test_attention(dtype, D, layout, block, kw):
    kw = dict(kw)
    decode = kw.pop("decode", False)
    q_lens = [1, 1, 1] if decode else [3, 40, 1]
    lens = [300, 41, 2000]
    c = make_cache(lens, Hkv=2, D=D, block=block, seed=D, layout=layout, width=140, pad=16)
    T = sum(q_lens)
    q = cut(T, 8, D, dtype, 6)
    starts = None if decode else starts_of(q_lens)
    most = kw.pop("max_query_len", max(q_lens))
    got = []
    for via in ("op", "c"):
        buf = torch.full((T, 10, D), math.nan, dtype=dtype, device="cuda")
        out, ws = buf[:, 1:9], workspace(D)
        if via == "op":
            ops.paged_attn_fp8_fwd(out, q, *c.views, c.table, c.lens, starts, most, 2000, 0.1, ws, **kw)
        else:
            call("paged_f8", capi.paged_f8_args(
                q=q, out=out, block_table=c.table, kv_lens=c.lens, max_kv_len=2000,
                softmax_scale=0.1, ws=ws, query_start_loc=starts, max_query_len=most,
                k_cache=c.k, v_cache=c.v, k_scale=c.ks, v_scale=c.vs, **kw))
        assert not out.isnan().any() and buf[:, 0].isnan().all() and buf[:, 9].isnan().all()
        got.append(out.clone())
    assert torch.equal(*got)
