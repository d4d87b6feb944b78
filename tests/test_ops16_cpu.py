"""Refusals of the attention ops of a 16-bit cache on CPU tensors: the op and its
fake, with the same messages."""

from __future__ import annotations

import pytest
import torch

from pth_flash_attn import ops, ops16
from pth_flash_attn.cache import paged16_views

pytestmark = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
BF, HF, I32 = torch.bfloat16, torch.float16, torch.int32


def _args(R=2, Hq=4, Hkv=2, D=64):
    kv = torch.zeros(5, 2, 16, Hkv, D, dtype=BF)
    k, v = paged16_views(kv)
    q = torch.zeros(R, Hq, D, dtype=BF)
    return dict(out=torch.zeros_like(q), q=q, k_cache=k, v_cache=v,
                block_table=torch.zeros(R, 3, dtype=I32), lens=torch.ones(R, dtype=I32),
                max_len=40, softmax_scale=0.1, ws=torch.zeros(64))


def _decode(a, fake=False):
    f = ops16.paged_decode_fwd_fake if fake else ops.paged_decode_fwd
    f(a["out"], a["q"], a["k_cache"], a["v_cache"], a["block_table"], a["lens"], a["max_len"],
      a["softmax_scale"], a["ws"], a.get("window", 0))


def _cross(a, fake=False):
    f = ops16.cross_attn_fwd_fake if fake else ops.cross_attn_fwd
    starts = a.get("starts", torch.arange(a["lens"].shape[0] + 1, dtype=I32))
    f(a["out"], a["q"], a["k_cache"], a["v_cache"], a["block_table"], a["lens"], starts,
      a.get("max_q", 1), a["max_len"], a["softmax_scale"], a["ws"])


BOTH = [
    (lambda a: dict(q=a["q"][0]), "q must be 3-D"),
    (lambda a: dict(q=a["q"].float()), "q must be bfloat16 or float16"),
    (lambda a: dict(q=a["q"][..., :32]), "head size D = q.size\\(2\\) must be 64, 128 or 256"),
    (lambda a: dict(q=torch.zeros(2, 64, 4, dtype=BF).transpose(1, 2)), "q must have stride 1"),
    (lambda a: dict(out=a["out"][:1]), "out must have the shape and dtype of q"),
    (lambda a: dict(out=a["out"].half()), "out must have the shape and dtype of q"),
    (lambda a: dict(out=torch.zeros(2, 64, 4, dtype=BF).transpose(1, 2)), "out must have stride 1"),
    (lambda a: dict(k_cache=a["k_cache"][:2]), "k_cache and v_cache must be"),
    (lambda a: dict(k_cache=a["k_cache"].half()), "must have the dtype of q"),
    (lambda a: dict(k_cache=a["k_cache"][:0], v_cache=a["v_cache"][:0]), "must not be empty"),
    (lambda a: dict(k_cache=torch.zeros(5, 16, 64, 2, dtype=BF).transpose(2, 3)),
     "k_cache and v_cache must have stride 1"),
    (lambda a: dict(q=torch.zeros(2, 3, 64, dtype=BF), out=torch.zeros(2, 3, 64, dtype=BF)),
     "Hq = 3 must be a positive multiple of Hkv = 2"),
    (lambda a: dict(q=torch.zeros(2, 130, 64, dtype=BF), out=torch.zeros(2, 130, 64, dtype=BF)),
     "G = Hq/Hkv = 65 exceeds the supported maximum 64"),
    (lambda a: dict(lens=a["lens"].long()), "lens must be int32"),
    (lambda a: dict(block_table=a["block_table"].long()), "block_table must be int32"),
    (lambda a: dict(block_table=a["block_table"][:1]), "block_table has 1 rows, fewer than"),
    (lambda a: dict(block_table=torch.zeros(3, 2, dtype=I32).t()), "stride 1 in their last"),
    (lambda a: dict(max_len=-1), "lens' bound must be >= 0"),
    (lambda a: dict(softmax_scale=0.0), "softmax_scale must be finite and > 0, got 0"),
    (lambda a: dict(softmax_scale=float("nan")), "softmax_scale must be finite"),
    (lambda a: dict(ws=a["ws"].half()), "ws must be contiguous float32"),
    (lambda a: dict(ws=a["ws"].view(8, 8)), "ws must be contiguous float32"),
]
DECODE = [
    (lambda a: dict(lens=torch.ones(1, dtype=I32)), "one token per request: T = 2, num_reqs = 1"),
    (lambda a: dict(window=-1), "window must be >= 0"),
]
CROSS = [
    (lambda a: dict(max_q=-1), "max_query_len must be >= 0"),
    (lambda a: dict(starts=torch.zeros(2, dtype=I32)), "query_start_loc must be contiguous int32"),
    (lambda a: dict(starts=torch.zeros(3)), "query_start_loc must be contiguous int32"),
    (lambda a: dict(starts=torch.zeros(6, dtype=I32)[::2]), "query_start_loc must be contiguous"),
]


@pytest.mark.parametrize(("call", "change", "message"),
                         [(_decode, *c) for c in BOTH + DECODE] + [(_cross, *c) for c in BOTH + CROSS])
def test_refusals(call, change, message):
    a = _args()
    a.update(change(a))
    with pytest.raises(RuntimeError, match=message):
        call(a)
    with pytest.raises(RuntimeError, match=message):
        call(a, fake=True)


@pytest.mark.parametrize("call", [_decode, _cross])
def test_valid_cpu_call_is_refused_last(call):
    a = _args()
    call(a, fake=True)
    with pytest.raises(RuntimeError, match="computes on CUDA tensors only"):
        call(a)


@pytest.mark.parametrize("call", [_decode, _cross])
def test_overlaps_are_refused(call):
    a = _args()
    a["out"] = a["k_cache"][:2, 0].repeat_interleave(2, 1)[:2]  # a copy: allowed so far
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        call(a)
    flat = a["k_cache"].as_strided((2, 4, 64), (256, 64, 1))
    with pytest.raises(RuntimeError, match="out must not overlap an input"):
        call({**a, "out": flat})
    with pytest.raises(RuntimeError, match="ws must not overlap an input"):
        call({**a, "ws": a["lens"].view(torch.float32)})


@pytest.mark.parametrize("call", [_decode, _cross])
def test_out_that_overlaps_itself_is_refused(call):
    a = _args()
    for bad in (a["out"][:1].expand_as(a["q"]), a["out"][:, :1].expand_as(a["q"]),
                torch.zeros(512, dtype=BF).as_strided(a["out"].shape, (128, 64, 1))):
        for fake in (False, True):
            with pytest.raises(RuntimeError, match="out must not overlap itself"):
                call({**a, "out": bad}, fake=fake)
    turned = torch.zeros(4, 2, 64, dtype=BF).transpose(0, 1)  # heads outside, as good
    call({**a, "out": turned}, fake=True)


def test_views_of_a_cache():
    kv = torch.arange(2 * 2 * 16 * 3 * 64, dtype=torch.float32).to(BF).view(2, 2, 3, 16, 64)
    k, v = paged16_views(kv, layout="HND")
    assert k.shape == v.shape == (2, 16, 3, 64) and k.data_ptr() == kv.data_ptr()
    assert torch.equal(v[1, 5, 2], kv[1, 1, 2, 5])
    for bad in (kv[0], kv.float(), kv[:, :1], kv.transpose(3, 4)):
        with pytest.raises(ValueError):
            paged16_views(bad)
    with pytest.raises(ValueError, match="layout must be one of"):
        paged16_views(kv, layout="NDH")
