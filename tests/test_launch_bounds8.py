"""Calls of more tokens than a launch has threads for (2^32) are refused by the C
entries, not left to the launch."""

from __future__ import annotations

import pytest
import torch

from pth_flash_attn import capi
from pth_flash_attn.cache import fp8_cache

needs_lib = pytest.mark.skipif(not capi.LIBRARY_PATH.is_file(), reason="libpth_attn.so not built")


def refused(what, args, tokens):
    args.num_tokens = tokens
    lib = capi.AttnLib()
    assert getattr(lib, what)(args) == capi.PTH_ATTN_EINVAL
    assert "more than 2^32 threads" in lib.last_error()


@needs_lib
@pytest.mark.parametrize(("D", "tokens"), [(64, (1 << 31) - 1), (64, 1 << 27), (1024, 1 << 25)])
def test_rotary(D, tokens):
    """Up to 4 tokens to a work-group of 256 threads, as many as have 1,024 pairs."""
    x = torch.zeros(4, 1, D, dtype=torch.bfloat16)
    longs = torch.zeros(D // 2, dtype=torch.int64)
    refused("rotary", capi.rotary_args(q_out=x, k_out=x, q=x, k=x, positions=longs[:4], turns=longs),
            tokens)


def _cache(device):
    k, v, ks, vs = fp8_cache(3, 32, 2, 64, device=device)
    return dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)


@pytest.mark.gpu
def test_write():
    """128 tokens to a work-group of 1,024."""
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.full((4,), -1, dtype=torch.int64, device="cuda")
    cache = _cache("cuda")
    refused("write_f8", capi.write_f8_args(key=x, value=x, slot_mapping=slots, **cache), (1 << 30) - 1)


@pytest.mark.gpu
def test_gather():
    """16 rows to a work-group of 256."""
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = _cache("cuda")
    refused("gather_f8", capi.gather_f8_args(key=x, value=x, block_table=table, row_start_loc=starts,
                                             **cache), (1 << 31) - 1)
