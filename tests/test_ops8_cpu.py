"""paged_attn_fp8_fwd's refusals, and the C ABI of rotary positions and the 8-bit
cache on the CPU: the ctypes mirrors are the header's structs, and bad
arguments are refused before a device is touched."""

from __future__ import annotations

import ctypes
import math
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from pth_flash_attn import capi, ops, planner
from pth_flash_attn.cache import fp8_cache

REPO = Path(__file__).resolve().parent.parent
needs_op = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
needs_lib = pytest.mark.skipif(not capi.LIBRARY_PATH.is_file(), reason="libpth_attn.so not built")
BF = torch.bfloat16


def _attention():
    k, v, ks, vs = fp8_cache(3, 32, 2, 64, device="cpu")
    q = torch.zeros(5, 8, 64, dtype=BF)
    return dict(out=q.clone(), q=q, k_cache=k, v_cache=v, k_scale=ks, v_scale=vs,
                block_table=torch.zeros(2, 3, dtype=torch.int32),
                seq_lens=torch.ones(2, dtype=torch.int32),
                query_start_loc=torch.zeros(3, dtype=torch.int32), max_query_len=3, max_seq_len=96,
                softmax_scale=0.1, ws=torch.zeros(64), window=0, causal=True)


@needs_op
@pytest.mark.parametrize(("change", "message"), [
    (lambda a: {}, "computes on CUDA tensors only"),
    (lambda a: dict(q=a["q"][0]), "q must be 3-D"),
    (lambda a: dict(q=a["q"].float()), "q must be bfloat16 or float16"),
    (lambda a: dict(out=a["out"].half()), "out must have the shape and dtype"),
    (lambda a: dict(out=a["out"][:4]), "out must have the shape and dtype"),
    (lambda a: dict(q=torch.zeros(5, 64, 8, dtype=BF).transpose(1, 2)), "q must have stride 1"),
    (lambda a: dict(k_cache=a["k_cache"][:, :, :1]), "k_cache and v_cache must be"),
    (lambda a: dict(v_cache=a["v_cache"].view(torch.uint8)), "must be float8_e4m3fn"),
    (lambda a: dict(k_cache=a["k_cache"][:, :8], v_cache=a["v_cache"][:, :8]), "multiple of 16"),
    (lambda a: dict(v_scale=a["v_scale"].int()), "k_scale and v_scale must be"),
    (lambda a: dict(k_scale=a["k_scale"][:2]), "k_scale and v_scale must be"),
    (lambda a: dict(q=a["q"][:, :7], out=a["out"][:, :7]), "positive multiple of Hkv"),
    (lambda a: dict(q=torch.zeros(5, 130, 64, dtype=BF), out=torch.zeros(5, 130, 64, dtype=BF)),
     "exceeds the supported maximum 64"),
    (lambda a: dict(seq_lens=a["seq_lens"].long()), "seq_lens must be int32"),
    (lambda a: dict(block_table=a["block_table"][:1]), "fewer than num_reqs"),
    (lambda a: dict(block_table=a["block_table"].long()), "block_table must be int32"),
    (lambda a: dict(query_start_loc=a["query_start_loc"][:2]), "query_start_loc must be"),
    (lambda a: dict(query_start_loc=None), "one token per request"),
    (lambda a: dict(max_query_len=-1), "max_query_len must be >= 0"),
    (lambda a: dict(max_seq_len=-1), "max_seq_len must be >= 0"),
    (lambda a: dict(softmax_scale=0.0), "softmax_scale must be finite"),
    (lambda a: dict(softmax_scale=math.inf), "softmax_scale must be finite"),
    (lambda a: dict(window=-1), "window must be >= 0"),
    (lambda a: dict(window=4, causal=False), "a window needs causal"),
    (lambda a: dict(ws=a["ws"].double()), "ws must be contiguous float32"),
    (lambda a: dict(out=a["out"][:1].expand_as(a["out"])), "out must not overlap itself"),
])
def test_refusals(change, message):
    args = _attention()
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.paged_attn_fp8_fwd(**args)
    if "CUDA" not in message:
        with pytest.raises(RuntimeError, match=message):
            ops.ops8.paged_attn_fp8_fwd_fake(**args)


@needs_op
def test_shared_memory_refused():
    a = _attention()
    buf = torch.zeros(5, 10, 64, dtype=BF)
    for bad, message in (
            (dict(q=buf[:, :8], out=buf[:, 2:]), "q itself or share no memory"),
            (dict(ws=a["out"].view(-1).view(torch.float32)), "out and ws must not overlap"),
            (dict(ws=a["q"].view(-1).view(torch.float32)), "ws must not overlap an input"),
            (dict(seq_lens=a["out"].view(-1).view(torch.int32)[:2]), "out must not overlap an input"),
            (dict(k_scale=a["out"].view(-1).view(torch.uint8)[:12].view(3, 2, 2)),
             "out must not overlap an input")):
        with pytest.raises(RuntimeError, match=message):
            ops.paged_attn_fp8_fwd(**{**a, **bad})


STRUCTS = {"rotary": capi.PthAttnRotaryArgs, "write_f8": capi.PthAttnWriteF8Args,
           "gather_f8": capi.PthAttnGatherF8Args, "paged_f8": capi.PthAttnPagedF8Args}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
@pytest.mark.parametrize("struct", [*STRUCTS.values(), capi.PthAttnCacheF8])
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
    for name, struct in STRUCTS.items():
        assert getattr(lib, f"pth_attn_{name}_args_bytes")() == ctypes.sizeof(struct)
    assert planner.fp8_workspace_floats(D=128, num_sms=256) == planner.paged16_workspace_floats(
        D=128, num_sms=256)
    with pytest.raises(ValueError, match="D must be one of"):
        planner.fp8_workspace_floats(D=96, num_sms=256)
    with pytest.raises(ValueError, match="multiple of 16"):
        fp8_cache(2, 24, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="layout must be"):
        fp8_cache(2, 16, 1, 64, layout="HDN", device="cpu")


def _c_args(what):
    k, v, ks, vs = fp8_cache(3, 32, 2, 64, device="cpu")
    cache = dict(k_cache=k, v_cache=v, k_scale=ks, v_scale=vs)
    x = torch.zeros(4, 2, 64, dtype=BF)
    ints = torch.zeros(8, dtype=torch.int32)
    longs = torch.zeros(32, dtype=torch.int64)
    table, ws = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(64)
    keep = [k, v, ks, vs, x, ints, longs, table, ws]
    if what == "rotary":
        return capi.rotary_args(q_out=x, k_out=x, q=x, k=x, positions=longs[:4], turns=longs), keep
    if what == "write_f8":
        return capi.write_f8_args(key=x, value=x, slot_mapping=longs[:4], **cache), keep
    if what == "gather_f8":
        return capi.gather_f8_args(key=x, value=x, block_table=table, row_start_loc=ints[:5],
                                   **cache), keep
    return capi.paged_f8_args(q=x, out=x, block_table=table, kv_lens=ints[:4], max_kv_len=96,
                              softmax_scale=0.1, ws=ws, **cache), keep


@needs_lib
@pytest.mark.parametrize(("what", "field", "value", "message"), [
    *((w, "abi_version", 1, "abi_version 1 != library ABI 2") for w in STRUCTS),
    *((w, "struct_bytes", 8, "struct_bytes 8 != sizeof") for w in STRUCTS),
    *((w, "cache.head_size", 96, "head_size must be 64, 128 or 256") for w in list(STRUCTS)[1:]),
    *((w, "cache.block_size", 24, "positive multiple of 16") for w in list(STRUCTS)[1:]),
    *((w, "cache.block_size", 0, "positive multiple of 16") for w in list(STRUCTS)[1:]),
    *((w, "cache.num_blocks", 0, "num_blocks >= 1") for w in list(STRUCTS)[1:]),
    *((w, "cache.num_kv_heads", 70000, "num_kv_heads 1 .. 65535") for w in list(STRUCTS)[1:]),
    *((w, "cache.k_scale", None, "codes and scales must be non-NULL") for w in list(STRUCTS)[1:]),
    *((w, "cache.k_cache.stride_slot", 72, "16-byte aligned rows") for w in list(STRUCTS)[1:]),
    *((w, "cache.v_cache.stride_slot", 1 << 24, "less than 2\\^24") for w in list(STRUCTS)[1:]),
    *((w, "num_tokens", -1, "num_tokens") for w in STRUCTS),
    ("rotary", "dtype", 7, "dtype must be"),
    ("rotary", "head_size", 2000, "head_size must be 2 .. 1024"),
    ("rotary", "rot_dim", 63, "rot_dim must be even"),
    ("rotary", "rot_dim", 66, "rot_dim must be even, 2 .. head_size"),
    ("rotary", "num_q_heads", 1 << 17, "0 .. 65536"),
    ("rotary", "scale", math.nan, "scale must be finite"),
    ("rotary", "positions", None, "must be non-NULL"),
    ("rotary", "q_stride_token", 3, "aligned to their element"),
    ("write_f8", "kv_dtype", 7, "kv_dtype must be"),
    ("write_f8", "key", None, "must be non-NULL"),
    ("write_f8", "value_stride_token", 3, "aligned to their element"),
    ("write_f8", "num_tokens", 1 << 30, "0 .. 2\\^30 - 1"),
    ("gather_f8", "kv_dtype", 7, "kv_dtype must be"),
    ("gather_f8", "row_start_loc", None, "must be non-NULL"),
    ("gather_f8", "block_table", None, "block_table must be non-NULL"),
    ("gather_f8", "key_stride_token", 8, "16-byte aligned rows"),
    ("paged_f8", "dtype", capi.PTH_ATTN_F32, "dtype must be"),
    ("paged_f8", "num_q_heads", 3, "positive multiple of num_kv_heads"),
    ("paged_f8", "num_q_heads", 130, "at most 64 query heads"),
    ("paged_f8", "num_tokens", 3, "num_tokens must equal num_reqs"),
    ("paged_f8", "window", -1, "window must be >= 0"),
    ("paged_f8", "max_kv_len", -1, "max_kv_len and block_table_width"),
    ("paged_f8", "softmax_scale", 0.0, "softmax_scale must be finite"),
    ("paged_f8", "q", None, "must be non-NULL"),
    ("paged_f8", "block_table", None, "block_table must be non-NULL"),
    ("paged_f8", "out_stride_token", 24, "16-byte aligned rows"),
])
def test_bad_arguments(what, field, value, message):
    a, keep = _c_args(what)
    at = a
    *path, last = field.split(".")
    for name in path:
        at = getattr(at, name)
    setattr(at, last, value)
    lib = capi.AttnLib()
    assert getattr(lib, what)(a) == capi.PTH_ATTN_EINVAL
    with pytest.raises(RuntimeError, match=message):
        lib.check(capi.PTH_ATTN_EINVAL)


@needs_lib
def test_nothing_to_do():
    lib = capi.AttnLib()
    for what in STRUCTS:
        a, keep = _c_args(what)
        a.num_tokens = 0
        if what == "paged_f8":
            a.num_reqs = 0
        assert getattr(lib, what)(a) == capi.PTH_ATTN_OK
        assert getattr(lib.lib, f"pth_attn_{what}")(None, None) == capi.PTH_ATTN_EINVAL
