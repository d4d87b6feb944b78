"""The C ABI of the 16-bit cache's entry points on the CPU: the ctypes mirrors
are the header's structs, and bad arguments are refused before a device is
touched."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from pth_flash_attn import capi, planner

REPO = Path(__file__).resolve().parent.parent
needs_lib = pytest.mark.skipif(not capi.LIBRARY_PATH.is_file(), reason="libpth_attn.so not built")


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
@pytest.mark.parametrize("struct", [capi.PthAttnP16Args, capi.PthAttnWrite16Args,
                                    capi.PthAttnTablesArgs])
def test_ctypes_mirror_matches_the_header(struct, tmp_path):
    name, fields = struct.__name__, [f[0] for f in struct._fields_]
    src, exe = tmp_path / "off.c", tmp_path / "off"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"pth_attn.h\"\n"
                   "int main(void) {\n" + "".join(
                       f'  printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + f'  printf("%zu\\n", sizeof({name}));\n  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c11", f"-I{REPO / 'include'}", str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


@needs_lib
def test_sizes():
    lib = capi.AttnLib().lib
    assert lib.pth_attn_paged16_args_bytes() == ctypes.sizeof(capi.PthAttnP16Args)
    assert lib.pth_attn_write16_args_bytes() == ctypes.sizeof(capi.PthAttnWrite16Args)
    assert lib.pth_attn_tables_args_bytes() == ctypes.sizeof(capi.PthAttnTablesArgs)


def test_workspace_size():
    assert planner.paged16_workspace_floats(D=128, num_sms=256) == 256 * (512 * 130 + 32)
    with pytest.raises(ValueError, match="D must be one of"):
        planner.paged16_workspace_floats(D=96, num_sms=256)
    with pytest.raises(TypeError, match="num_sms must be a host int"):
        planner.paged16_workspace_floats(D=64, num_sms=2.0)


def _attention(D=128):
    kv = torch.zeros(3, 2, 16, 2, D, dtype=torch.bfloat16)
    keep = [kv, torch.zeros(2, 8, D, dtype=torch.bfloat16), torch.zeros(2, 8, D, dtype=torch.bfloat16),
            torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.zeros(64)]
    a = capi.paged16_args(q=keep[1], out=keep[2], k_cache=kv[:, 0], v_cache=kv[:, 1],
                          block_table=keep[3], kv_lens=keep[4], max_kv_len=48, softmax_scale=0.1,
                          ws=keep[5])
    return a, keep


@needs_lib
@pytest.mark.parametrize(("field", "value", "message"), [
    ("abi_version", 1, "abi_version 1 != library ABI 2"),
    ("struct_bytes", 8, "struct_bytes 8 != sizeof(PthAttnP16Args)"),
    ("head_size", 96, "head_size must be 64, 128 or 256"),
    ("dtype", capi.PTH_ATTN_F32, "dtype must be"),
    ("block_size", 0, "block_size >= 1"),
    ("num_q_heads", 7, "positive multiple of num_kv_heads"),
    ("num_q_heads", 130, "at most 64 query heads"),
    ("num_tokens", 3, "num_tokens must equal num_reqs"),
    ("num_reqs", -1, "num_reqs, num_tokens >= 0"),
    ("window", -1, "window must be >= 0"),
    ("max_kv_len", -1, "max_kv_len and block_table_width"),
    ("softmax_scale", float("inf"), "softmax_scale must be finite"),
    ("q", None, "must be non-NULL"),
    ("block_table", None, "block_table must be non-NULL"),
    ("q_stride_token", 24, "16-byte aligned rows"),
])
def test_attention_refusals(field, value, message):
    lib = capi.AttnLib()
    a, _keep = _attention()
    setattr(a, field, value)
    assert lib.paged16(a) == capi.PTH_ATTN_EINVAL
    assert message in lib.last_error()


@needs_lib
def test_window_of_cross_attention_is_refused():
    lib = capi.AttnLib()
    a, keep = _attention()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32)
    a.query_start_loc, a.window = starts.data_ptr(), 4
    assert lib.paged16(a) == capi.PTH_ATTN_EINVAL
    assert "a window needs one query token per request" in lib.last_error()
    a.k_cache.stride_slot = 1 << 24
    a.window = 0
    assert lib.paged16(a) == capi.PTH_ATTN_EINVAL and "2^24" in lib.last_error()


@needs_lib
def test_nothing_to_do_is_ok_without_a_device():
    lib = capi.AttnLib()
    a, _keep = _attention()
    a.num_reqs = a.num_tokens = 0
    assert lib.paged16(a) == capi.PTH_ATTN_OK


def _tables():
    i32 = dict(dtype=torch.int32)
    t = dict(block_table=torch.zeros(2, 4, **i32), slot_mapping=torch.zeros(8, dtype=torch.int64),
             seq_lens=torch.zeros(2, **i32), query_start_loc=torch.zeros(3, **i32),
             pool_out=torch.zeros(2, **i32), context_lens=torch.zeros(2, **i32),
             query_lens=torch.zeros(2, **i32), free_pages=torch.zeros(5, **i32),
             pool_in=torch.zeros(2, **i32))
    return capi.tables_args(block_size=16, **t), t


@needs_lib
@pytest.mark.parametrize(("field", "value", "message"), [
    ("abi_version", 3, "abi_version 3 != library ABI 2"),
    ("struct_bytes", 8, "struct_bytes 8 != sizeof(PthAttnTablesArgs)"),
    ("num_reqs", -1, "num_reqs, num_slots, num_free"),
    ("num_slots", 1 << 30, "must be less than 2^30"),
    ("block_size", 1 << 30, "block_table_width x block_size must be less than 2^31"),
    ("pool_in", None, "must be non-NULL"),
    ("query_lens", None, "must be non-NULL"),
    ("slot_mapping", None, "slot_mapping must be non-NULL"),
    ("free_pages", None, "free_pages must be non-NULL"),
])
def test_tables_refusals(field, value, message):
    lib = capi.AttnLib()
    a, _keep = _tables()
    setattr(a, field, value)
    assert lib.step_tables(a) == capi.PTH_ATTN_EINVAL
    assert message in lib.last_error()


@needs_lib
@pytest.mark.parametrize(("field", "value", "message"), [
    ("abi_version", 3, "abi_version 3 != library ABI 2"),
    ("struct_bytes", 8, "struct_bytes 8 != sizeof(PthAttnWrite16Args)"),
    ("head_size", 32, "head_size must be"),
    ("cache_dtype", capi.PTH_ATTN_F32, "cache_dtype must be"),
    ("kv_dtype", capi.PTH_ATTN_F16, "kv_dtype must be cache_dtype or"),
    ("key", None, "must be non-NULL"),
    ("key_stride_token", 129, "aligned to their element"),
])
def test_writer_refusals(field, value, message):
    lib = capi.AttnLib()
    kv = torch.zeros(2, 2, 16, 2, 64, dtype=torch.bfloat16)
    x, slots = torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    a = capi.write16_args(key=x, value=x, k_cache=kv[:, 0], v_cache=kv[:, 1], slot_mapping=slots)
    setattr(a, field, value)
    assert lib.write_kv16(a) == capi.PTH_ATTN_EINVAL
    assert message in lib.last_error()


@needs_lib
def test_tables_rows_that_overlap_are_refused():
    lib = capi.AttnLib()
    a, _keep = _tables()
    a.block_table_row_stride = 3
    assert lib.step_tables(a) == capi.PTH_ATTN_EINVAL
    assert "rows of block_table must not overlap" in lib.last_error()


@needs_lib
@pytest.mark.parametrize(("head_size", "heads"), [(64, 128), (128, 64), (256, 32)])
def test_writer_launch_bound(head_size, heads):
    """2^22 tokens of 2^13 values: as many threads as a launch does not have."""
    lib = capi.AttnLib()
    kv = torch.zeros(1, 2, 1, heads, head_size, dtype=torch.bfloat16)
    x, slots = torch.zeros(1, heads, head_size, dtype=torch.bfloat16), torch.zeros(1).long()
    a = capi.write16_args(key=x, value=x, k_cache=kv[:, 0], v_cache=kv[:, 1], slot_mapping=slots)
    a.num_tokens = 1 << 22
    assert a.num_tokens * heads * head_size == 1 << 35
    assert lib.write_kv16(a) == capi.PTH_ATTN_EINVAL and "2^35" in lib.last_error()
