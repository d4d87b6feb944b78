"""A dimension of one element has no second row to align: its stride, which a
view may leave at any value, refuses no call of the 16-bit cache's ops."""

from __future__ import annotations

import pytest
import torch

from pth_flash_attn import capi, ops

BF = torch.bfloat16
needs_lib = pytest.mark.skipif(not capi.LIBRARY_PATH.is_file(), reason="libpth_attn.so not built")


def of_one(shape, device):
    """Zeros whose strides of one-element dimensions are odd."""
    t = torch.zeros(shape, dtype=BF, device=device)
    return t.as_strided(shape, [s if n > 1 or i == t.dim() - 1 else 24 * s + 7
                                for i, (n, s) in enumerate(zip(t.shape, t.stride()))])


def tensors(T, Hq, cache, device):
    D = cache[3]
    return dict(q=of_one((T, Hq, D), device), out=of_one((T, Hq, D), device),
                k_cache=of_one(cache, device), v_cache=of_one(cache, device))


# One token; one head; one page of one slot and one head.
SHAPES = [(1, 4, (3, 16, 2, 64)), (2, 1, (3, 16, 1, 64)), (1, 1, (1, 1, 1, 64)),
          (1, 2, (1, 16, 2, 128))]


@needs_lib
@pytest.mark.parametrize(("T", "Hq", "cache"), SHAPES)
def test_c_entry_without_a_device(T, Hq, cache):
    if torch.cuda.is_available():
        pytest.skip("needs a machine without a device")
    lib, t = capi.AttnLib(), tensors(T, Hq, cache, "cpu")
    a = capi.paged16_args(**t, block_table=torch.zeros(T, 2, dtype=torch.int32),
                          kv_lens=torch.ones(T, dtype=torch.int32), max_kv_len=1,
                          softmax_scale=0.1, ws=torch.zeros(64))
    assert lib.paged16(a) == capi.PTH_ATTN_EINVAL
    assert "cannot query the compute-unit count" in lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize(("T", "Hq", "cache"), SHAPES)
def test_write_and_attend(T, Hq, cache):
    from paged16_cases import assert_close, queries, reference, starts_of, workspace

    t, (_, block, Hkv, D) = tensors(T, Hq, cache, "cuda"), cache
    t["q"].copy_(queries(T, Hq, D, BF, 1))
    key, value = of_one((T, Hkv, D), "cuda"), of_one((T, Hkv, D), "cuda")
    key.copy_(queries(T, Hkv, D, BF, 2))
    value.copy_(queries(T, Hkv, D, BF, 3))
    slots = torch.arange(T, device="cuda") * block
    ops.reshape_and_cache_16bit(key, value, t["k_cache"], t["v_cache"], slots)
    table = torch.arange(T, dtype=torch.int32, device="cuda").view(T, 1)
    lens = torch.ones(T, dtype=torch.int32, device="cuda")
    keys = [(key[r : r + 1], value[r : r + 1]) for r in range(T)]
    want, tol = reference(t["q"], keys, [1] * T, 0.1, pair=True)
    ops.paged_decode_fwd(t["out"], t["q"], t["k_cache"], t["v_cache"], table, lens, 1, 0.1,
                         workspace(D))
    assert_close(t["out"], want, tol)
    for most in (1, 64):  # either kernel
        t["out"].zero_()
        ops.cross_attn_fwd(t["out"], t["q"], t["k_cache"], t["v_cache"], table, lens,
                           starts_of([1] * T), most, 1, 0.1, workspace(D))
        want, tol = reference(t["q"], keys, [1] * T, 0.1, pair=False)
        assert_close(t["out"], want, tol)
