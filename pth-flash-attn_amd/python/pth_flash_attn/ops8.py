"""Rotary positions, and the ops around a paged cache in 8-bit floating point
with a scale for each block of 16 tokens and KV head.

* ``rotary_embedding``: queries and keys turned by their positions.
* ``reshape_and_cache_fp8``: a step's keys and values into the cache.
* ``gather_cache_fp8``: cached tokens back into rows.
* ``paged_attn_fp8_fwd``: causal attention over the cache, of one new token per
  request, drafts, prompts, or a mix.

``pth_flash_attn.ops`` loads the library that holds them, registers the fakes
of this module and re-exports its wrappers. ``cache.fp8_cache`` makes a cache:
codes, a pair of strided views ``[num_blocks, block_size, Hkv, D]`` of
``float8_e4m3fn`` (``block_size`` a multiple of 16, rows 16-byte aligned), and
scales ``uint8 [num_blocks, block_size / 16, Hkv]``, contiguous: the exponent e
of a block's scale 2^(e - 127). A value is its code times the scale; e = 0 stands
for the scale 0, and above 246, which the writer never leaves, e counts as 246.
No op of this module has a counterpart in the reference, whose cache is int8
with a scale for each token.
"""

from __future__ import annotations

import math

import torch

from pth_flash_attn.ops16 import (
    _HALVES,
    _HEAD_SIZES,
    _INNER,
    _MAX_GROUP,
    _Checks,
    _int32_vector,
    _op,
    _overlaps_itself,
)

NAMES = ("rotary_embedding", "reshape_and_cache_fp8", "gather_cache_fp8", "paged_attn_fp8_fwd")
FP8 = torch.float8_e4m3fn
SPAN = 16  # tokens of a scale
_VALUES = (torch.float32, *_HALVES)


def _int64_vector(t: torch.Tensor, n: int) -> bool:
    return (t.dim() == 1 and t.shape[0] == n and t.dtype == torch.int64 and t.is_contiguous())


def rotary_embedding_fake(q_out, k_out, q, k, positions, turns, interleaved=False, scale=1.0,
                          inverse=False) -> None:
    """Fake of ``rotary_embedding``: its metadata checks (an out-variant)."""
    check = _Checks("rotary_embedding")
    check(q.dim() == 3 and k.dim() == 3, "q and k must be 3-D [T, heads, D]")
    T, _, D = q.shape
    check(k.shape[0] == T and k.shape[2] == D, "q and k must have the same T and D")
    check(2 <= D <= 1024, "head size must be 2 to 1024, got ", D)
    check(q.dtype in _VALUES and k.dtype == q.dtype,
          "q and k must both be float32, bfloat16 or float16")
    check(q_out.shape == q.shape and q_out.dtype == q.dtype and k_out.shape == k.shape
          and k_out.dtype == k.dtype, "q_out and k_out must have the shapes and dtype of q and k")
    check(all(t.stride(2) == 1 for t in (q, k, q_out, k_out)),
          "q, k, q_out and k_out must have stride 1 in their last dimension")
    check(_int64_vector(positions, T), "positions must be contiguous int64 [T]")
    check(turns.dim() == 1 and turns.dtype == torch.int64 and turns.is_contiguous()
          and 1 <= turns.shape[0] and 2 * turns.shape[0] <= D,
          "turns must be contiguous int64 [rot_dim / 2], rot_dim 2 to D")
    check(math.isfinite(scale), "scale must be finite, got ", f"{scale:g}")
    check(all(t.device == q.device for t in (k, q_out, k_out, positions, turns)),
          "all tensors must be on the device of q")
    check(not _overlaps_itself(q_out) and not _overlaps_itself(k_out),
          "q_out and k_out must not overlap themselves")


def _check_cache(check: _Checks, k_cache, v_cache, k_scale, v_scale, D: int) -> None:
    check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == D,
          "k_cache and v_cache must be [num_blocks, block_size, Hkv, ", D, "]")
    check(D in _HEAD_SIZES, "head size must be 64, 128 or 256, got ", D)
    check(k_cache.dtype == FP8 and v_cache.dtype == FP8,
          "k_cache and v_cache must be float8_e4m3fn")
    check(min(k_cache.shape[:3]) >= 1, "k_cache and v_cache must not be empty")
    check(k_cache.shape[1] % SPAN == 0, "block_size must be a multiple of 16, got ",
          k_cache.shape[1])
    check(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "k_cache and v_cache ", _INNER)
    want = (k_cache.shape[0], k_cache.shape[1] // SPAN, k_cache.shape[2])
    check(all(t.dim() == 3 and t.dtype == torch.uint8 and t.is_contiguous()
              and tuple(t.shape) == want for t in (k_scale, v_scale)),
          "k_scale and v_scale must be contiguous uint8 [num_blocks, block_size / 16, Hkv]")


def _check_rows(check: _Checks, key, value, k_cache, v_cache, k_scale, v_scale) -> None:
    check(key.dim() == 3 and value.dim() == 3, "key and value must be 3-D [T, Hkv, D]")
    check(key.shape == value.shape, "key and value must have the same shape")
    _check_cache(check, k_cache, v_cache, k_scale, v_scale, key.shape[2])
    check(k_cache.shape[2] == key.shape[1], "key and value must have the cache's heads")
    check(key.dtype in _VALUES and key.dtype == value.dtype,
          "key and value must both be float32, bfloat16 or float16")
    check(key.stride(2) == 1 and value.stride(2) == 1, "key and value ", _INNER)


def reshape_and_cache_fp8_fake(key, value, k_cache, v_cache, k_scale, v_scale,
                               slot_mapping) -> None:
    """Fake of the writer: its metadata checks (an in-place op)."""
    check = _Checks("reshape_and_cache_fp8")
    _check_rows(check, key, value, k_cache, v_cache, k_scale, v_scale)
    check(_int64_vector(slot_mapping, key.shape[0]), "slot_mapping must be contiguous int64 [T]")
    check(all(t.device == key.device
              for t in (value, k_cache, v_cache, k_scale, v_scale, slot_mapping)),
          "all tensors must be on the device of key")
    check(not _overlaps_itself(k_cache) and not _overlaps_itself(v_cache),
          "k_cache and v_cache must not overlap themselves")


def gather_cache_fp8_fake(key, value, k_cache, v_cache, k_scale, v_scale, block_table,
                          row_start_loc, first=None) -> None:
    """Fake of the reader: its metadata checks (an out-variant)."""
    check = _Checks("gather_cache_fp8")
    _check_rows(check, key, value, k_cache, v_cache, k_scale, v_scale)
    check(_int32_vector(row_start_loc) and row_start_loc.shape[0] >= 1,
          "row_start_loc must be contiguous int32 [num_reqs + 1]")
    R = row_start_loc.shape[0] - 1
    check(block_table.dim() == 2 and block_table.dtype == torch.int32
          and block_table.stride(1) == 1 and block_table.shape[0] >= R,
          "block_table must be int32 [>= num_reqs, max_blocks] with stride 1 in its last "
          "dimension")
    check(first is None or _int32_vector(first, R), "first must be contiguous int32 [num_reqs]")
    others = [value, k_cache, v_cache, k_scale, v_scale, block_table, row_start_loc]
    others += [] if first is None else [first]
    check(all(t.device == key.device for t in others), "all tensors must be on the device of key")
    check(not _overlaps_itself(key) and not _overlaps_itself(value),
          "key and value must not overlap themselves")


def paged_attn_fp8_fwd_fake(out, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                            query_start_loc, max_query_len, max_seq_len, softmax_scale, ws,
                            window=0, causal=True) -> None:
    """Fake of ``paged_attn_fp8_fwd``: its metadata checks (an out-variant)."""
    check = _Checks("paged_attn_fp8_fwd")
    check(q.dim() == 3, "q must be 3-D [T, Hq, D], got ", q.dim(), "-D")
    check(q.dtype in _HALVES, "q must be bfloat16 or float16")
    T, Hq, D = q.shape
    check(q.stride(2) == 1, "q must have stride 1 in its last dimension")
    check(out.dim() == 3 and out.shape == q.shape and out.dtype == q.dtype,
          "out must have the shape and dtype of q")
    check(out.stride(2) == 1, "out must have stride 1 in its last dimension")
    _check_cache(check, k_cache, v_cache, k_scale, v_scale, D)
    Hkv = k_cache.shape[2]
    check(Hq >= 1 and Hq % Hkv == 0, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv)
    check(Hq // Hkv <= _MAX_GROUP, "G = Hq/Hkv = ", Hq // Hkv,
          " exceeds the supported maximum ", _MAX_GROUP)
    check(seq_lens.dim() == 1 and seq_lens.dtype == torch.int32,
          "seq_lens must be int32 [num_reqs]")
    R = seq_lens.shape[0]
    check(block_table.dim() == 2 and block_table.dtype == torch.int32,
          "block_table must be int32 [num_reqs, max_blocks]")
    check(block_table.shape[0] >= R, "block_table has ", block_table.shape[0],
          " rows, fewer than num_reqs = ", R)
    check(seq_lens.stride(0) == 1 and block_table.stride(1) == 1, "seq_lens and block_table ",
          _INNER)
    if query_start_loc is not None:
        check(_int32_vector(query_start_loc, R + 1),
              "query_start_loc must be contiguous int32 [num_reqs + 1]")
    else:
        check(T == R, "q must have one token per request: T = ", T, ", num_reqs = ", R)
    check(max_query_len >= 0, "max_query_len must be >= 0, got ", max_query_len)
    check(max_seq_len >= 0, "max_seq_len must be >= 0, got ", max_seq_len)
    check(math.isfinite(softmax_scale) and softmax_scale > 0.0,
          "softmax_scale must be finite and > 0, got ", f"{softmax_scale:g}")
    check(window >= 0, "window must be >= 0, got ", window)
    check(window == 0 or causal, "a window needs causal")
    check(ws.dtype == torch.float32 and ws.dim() == 1 and ws.is_contiguous(),
          "ws must be contiguous float32 [n]")
    others = [out, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, ws]
    others += [] if query_start_loc is None else [query_start_loc]
    check(all(t.device == q.device for t in others), "all tensors must be on the device of q")
    check(not _overlaps_itself(out), "out must not overlap itself")


FAKES = {name: globals()[f"{name}_fake"] for name in NAMES}


def rotary_embedding(
    q_out: torch.Tensor, k_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor,
    positions: torch.Tensor, turns: torch.Tensor, interleaved: bool = False, scale: float = 1.0,
    inverse: bool = False,
) -> None:
    """``q`` [T, Hq, D] and ``k`` [T, Hkv, D] turned by their ``positions`` (int64 [T]).

    ``turns`` (int64 [rot_dim / 2]) and ``scale`` come from ``rotary.rotary_turns``.
    The pairs are columns (j, j + rot_dim / 2) of each head, or (2 j, 2 j + 1) if
    ``interleaved``; pair (a, b) becomes scale (a cos - b sin, b cos + a sin), and
    the columns from rot_dim on are copied. ``inverse`` turns back: with the same
    scale that is the transpose, which takes the gradients of the outputs to those
    of the inputs (with 1 / scale the inverse). Angles are exact for every
    position, negative ones too; sums are in 32 bits and rounded once.

    float32, bfloat16 or float16; any strides of tokens and heads (rows on
    16-byte addresses, and a rot_dim that divides into 16-byte runs, are fastest).
    ``k`` may have no heads. ``q_out`` may be ``q`` itself and ``k_out`` ``k`` (all
    may be columns of one buffer); other than that outputs share memory with
    nothing. One launch; allocates nothing, reads nothing back.
    """
    _op("rotary_embedding")(q_out, k_out, q, k, positions, turns, interleaved, scale, inverse)


def reshape_and_cache_fp8(
    key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor,
) -> None:
    """``key`` / ``value`` [T, Hkv, D] (float32, bfloat16 or float16) into the 8-bit cache.

    Token t goes to slot ``slot_mapping[t]`` (page ``slot // block_size``, in-page
    slot ``slot % block_size``); a slot outside the cache, as -1, skips it. Tokens
    come in any order; of those that share a slot the last one counts.

    A block of 16 slots that gets tokens takes, for each head, the smallest scale
    that keeps its largest finite value within 448, 2^-126 at least (0 if all are
    0), and no smaller one than it had, unless its first slot is written: that
    begins the block, whose other slots then hold nothing until they are written.
    (So a request's tokens are written in order, or a block's first one before
    the others or with them.) Where a scale grows, the codes that the block held
    are rounded to it again, which is exact but for the smallest. Codes are rounded
    to nearest even; a NaN or an infinity becomes NaN and leaves the scale alone;
    values beyond 448 x 2^119 are cut off there.

    One launch; allocates nothing, reads nothing back; the result does not
    depend on the order in which blocks are worked on. The caches share memory
    with nothing, nor do the scales.
    """
    _op("reshape_and_cache_fp8")(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)


def gather_cache_fp8(
    key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
    row_start_loc: torch.Tensor, first: torch.Tensor | None = None,
) -> None:
    """Cached tokens as rows: ``key`` / ``value`` [T, Hkv, D] (float32, bfloat16 or float16).

    Rows ``row_start_loc[r]`` to ``row_start_loc[r + 1]`` (int32 [R + 1], ascending)
    are request r's tokens from position ``first[r]`` (int32 [R]; 0 if None) on, each
    value rounded once to the type. A token for which the request's row of
    ``block_table`` holds no page of the cache gives zeros; rows of no request are
    left as they were. Rows of key and value are 16-byte aligned. One launch;
    allocates nothing, reads nothing back.
    """
    _op("gather_cache_fp8")(key, value, k_cache, v_cache, k_scale, v_scale, block_table,
                            row_start_loc, first)


def paged_attn_fp8_fwd(
    out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
    seq_lens: torch.Tensor, query_start_loc: torch.Tensor | None, max_query_len: int,
    max_seq_len: int, softmax_scale: float, ws: torch.Tensor, window: int = 0,
    causal: bool = True,
) -> None:
    """Attention over a paged 8-bit cache, into ``out``.

    ``q`` / ``out`` [T, Hq, D], bfloat16 or float16: request r's tokens are rows
    ``query_start_loc[r]`` to ``query_start_loc[r + 1]`` (None: row r is request r's
    one token); query head h reads KV head h // (Hq / Hkv). Causal: a request's n
    tokens are the last n of its ``seq_lens[r]`` keys, and each sees the keys up to
    its own, the last ``window`` of them (all, if 0). Not causal: every token sees
    all of the request's keys. A row that sees no key, or whose weights are all 0,
    is 0; rows of no request are left as they were. What a page holds outside
    of the keys that a row sees does not reach it; a NaN that it sees makes it NaN
    (in V, its column).

    ``max_query_len`` chooses kernel and split (any value is correct);
    ``max_seq_len`` bounds the lengths (longer ones are cut there, at the block
    table's reach and at 2^31 - 8,193 keys); a page number outside the cache reads page 0. ``ws`` is
    workspace of ``planner.fp8_workspace_floats`` floats; it holds nothing between
    calls, and calls that can run at the same time need one each. ``out`` may be
    ``q`` itself; other than that they share no memory.

    At most four launches (two where the batch is not one of prompts and decodes),
    whose sizes depend on host integers only, so a captured graph replays as the
    lengths change. Allocates nothing, reads nothing back,
    is deterministic. Rows of q, out and the cache are 16-byte aligned.
    """
    _op("paged_attn_fp8_fwd")(out, q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                              query_start_loc, max_query_len, max_seq_len, softmax_scale, ws,
                              window, causal)
