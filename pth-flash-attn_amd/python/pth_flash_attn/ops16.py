"""The ops around a paged cache in the model's own 16-bit type (bf16 or fp16).

* ``build_step_tables``: a step's block tables, slot map, lengths and starts on
  the GPU, from its request lengths and a list of free pages.
* ``reshape_and_cache_16bit``: the step's keys and values into the cache.
* ``paged_decode_fwd``: attention of one new token per request.
* ``cross_attn_fwd``: attention of a decoder's tokens to an encoder's states,
  whose keys and values lie in a cache of their own length.

``pth_flash_attn.ops`` loads the library that holds them, registers the fakes
of this module and re-exports its wrappers. A cache is a pair of strided views
``[num_blocks, block_size, Hkv, D]`` (``cache.paged16_views``). No op of this
module has a counterpart in the reference, which reads int8 caches only.
"""

from __future__ import annotations

import math

import torch

NAMES = ("build_step_tables", "reshape_and_cache_16bit", "paged_decode_fwd", "cross_attn_fwd")
_HEAD_SIZES = (64, 128, 256)
_MAX_GROUP = 64
_HALVES = (torch.bfloat16, torch.float16)
_INNER = "must have stride 1 in their last dimension"


class _Checks:
    """``check(ok, message parts)`` raising with the op's name, as the C++ op does."""

    def __init__(self, op: str) -> None:
        self.op = op

    def __call__(self, ok: bool, *parts: object) -> None:
        if not ok:
            raise RuntimeError(f"{self.op}: " + "".join(str(p) for p in parts))


def _int32_vector(t: torch.Tensor, n: int | None = None) -> bool:
    return (t.dim() == 1 and t.dtype == torch.int32 and t.is_contiguous()
            and (n is None or t.shape[0] == n))


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements may share memory: a dimension steps within the
    reach of those of smaller strides."""
    reach = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size > 1:
            if stride < reach:
                return True
            reach += stride * (size - 1)
    return False


def _check_attention(op: str, lens_name: str, out: torch.Tensor, q: torch.Tensor,
                     k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                     lens: torch.Tensor, query_start_loc: torch.Tensor | None, max_len: int,
                     softmax_scale: float, ws: torch.Tensor, window: int) -> None:
    """The attention ops' metadata checks, in the C++ order with the C++ messages."""
    check = _Checks(op)
    check(q.dim() == 3, "q must be 3-D [T, Hq, D], got ", q.dim(), "-D")
    check(q.dtype in _HALVES, "q must be bfloat16 or float16")
    T, Hq, D = q.shape
    check(D in _HEAD_SIZES, "head size D = q.size(2) must be 64, 128 or 256, got ", D)
    check(q.stride(2) == 1, "q must have stride 1 in its last dimension")
    check(out.dim() == 3 and out.shape == q.shape and out.dtype == q.dtype,
          "out must have the shape and dtype of q")
    check(out.stride(2) == 1, "out must have stride 1 in its last dimension")
    check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[3] == D,
          "k_cache and v_cache must be [num_blocks, block_size, Hkv, ", D, "]")
    check(k_cache.dtype == q.dtype and v_cache.dtype == q.dtype,
          "k_cache and v_cache must have the dtype of q")
    check(min(k_cache.shape[:3]) >= 1, "k_cache and v_cache must not be empty")
    check(k_cache.stride(3) == 1 and v_cache.stride(3) == 1, "k_cache and v_cache ", _INNER)
    Hkv = k_cache.shape[2]
    check(Hq >= 1 and Hq % Hkv == 0, "Hq = ", Hq, " must be a positive multiple of Hkv = ", Hkv)
    check(Hq // Hkv <= _MAX_GROUP, "G = Hq/Hkv = ", Hq // Hkv,
          " exceeds the supported maximum ", _MAX_GROUP)
    check(lens.dim() == 1 and lens.dtype == torch.int32, lens_name, " must be int32 [num_reqs]")
    R = lens.shape[0]
    check(block_table.dim() == 2 and block_table.dtype == torch.int32,
          "block_table must be int32 [num_reqs, max_blocks]")
    check(block_table.shape[0] >= R, "block_table has ", block_table.shape[0],
          " rows, fewer than num_reqs = ", R)
    check(lens.stride(0) == 1 and block_table.stride(1) == 1, lens_name, " and block_table ",
          _INNER)
    if query_start_loc is not None:
        check(_int32_vector(query_start_loc, R + 1),
              "query_start_loc must be contiguous int32 [num_reqs + 1]")
    else:
        check(T == R, "q must have one token per request: T = ", T, ", num_reqs = ", R)
    check(max_len >= 0, lens_name, "' bound must be >= 0, got ", max_len)
    check(math.isfinite(softmax_scale) and softmax_scale > 0.0,
          "softmax_scale must be finite and > 0, got ", f"{softmax_scale:g}")
    check(window >= 0, "window must be >= 0, got ", window)
    check(ws.dtype == torch.float32 and ws.dim() == 1 and ws.is_contiguous(),
          "ws must be contiguous float32 [n]")
    others = [out, k_cache, v_cache, block_table, lens, ws]
    if query_start_loc is not None:
        others.append(query_start_loc)
    check(all(t.device == q.device for t in others), "all tensors must be on the device of q")
    check(not _overlaps_itself(out), "out must not overlap itself")


def paged_decode_fwd_fake(out, q, k_cache, v_cache, block_table, seq_lens, max_seq_len,
                          softmax_scale, ws, window=0) -> None:
    """Fake of ``paged_decode_fwd``: its metadata checks (an out-variant)."""
    _check_attention("paged_decode_fwd", "seq_lens", out, q, k_cache, v_cache, block_table,
                     seq_lens, None, max_seq_len, softmax_scale, ws, window)


def cross_attn_fwd_fake(out, q, k_cache, v_cache, block_table, encoder_lens, query_start_loc,
                        max_query_len, max_encoder_len, softmax_scale, ws) -> None:
    """Fake of ``cross_attn_fwd``: its metadata checks (an out-variant)."""
    _Checks("cross_attn_fwd")(max_query_len >= 0, "max_query_len must be >= 0, got ",
                              max_query_len)
    _check_attention("cross_attn_fwd", "encoder_lens", out, q, k_cache, v_cache, block_table,
                     encoder_lens, query_start_loc, max_encoder_len, softmax_scale, ws, 0)


def reshape_and_cache_16bit_fake(key, value, k_cache, v_cache, slot_mapping) -> None:
    """Fake of the writer: its metadata checks (an in-place op)."""
    check = _Checks("reshape_and_cache_16bit")
    check(key.dim() == 3 and value.dim() == 3, "key and value must be 3-D [T, Hkv, D]")
    check(key.shape == value.shape, "key and value must have the same shape")
    T, Hkv, D = key.shape
    check(D in _HEAD_SIZES, "head size must be 64, 128 or 256, got ", D)
    check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape
          and tuple(k_cache.shape[2:]) == (Hkv, D),
          "k_cache and v_cache must be [num_blocks, block_size, ", Hkv, ", ", D, "]")
    check(k_cache.dtype in _HALVES and k_cache.dtype == v_cache.dtype,
          "k_cache and v_cache must both be bfloat16 or float16")
    check(min(k_cache.shape[:3]) >= 1, "k_cache and v_cache must not be empty")
    check(key.dtype == value.dtype and key.dtype in (torch.float32, k_cache.dtype),
          "key and value must both be float32 or have the dtype of the cache")
    check(all(t.stride(-1) == 1 for t in (key, value, k_cache, v_cache)),
          "key, value, k_cache and v_cache ", _INNER)
    check(slot_mapping.dim() == 1 and slot_mapping.shape[0] == T
          and slot_mapping.dtype == torch.int64 and slot_mapping.is_contiguous(),
          "slot_mapping must be contiguous int64 [T]")
    check(all(t.device == key.device for t in (value, k_cache, v_cache, slot_mapping)),
          "all tensors must be on the device of key")
    check(not _overlaps_itself(k_cache) and not _overlaps_itself(v_cache),
          "k_cache and v_cache must not overlap themselves")


def build_step_tables_fake(block_table, slot_mapping, seq_lens, query_start_loc, pool_out,
                           context_lens, query_lens, free_pages, pool_in, block_size) -> None:
    """Fake of ``build_step_tables``: its metadata checks (an out-variant)."""
    check = _Checks("build_step_tables")
    check(_int32_vector(context_lens), "context_lens must be contiguous int32 [n]")
    R = context_lens.shape[0]
    for t, n, name in ((query_lens, R, "query_lens"), (seq_lens, R, "seq_lens"),
                       (query_start_loc, R + 1, "query_start_loc"),
                       (free_pages, None, "free_pages"), (pool_in, 2, "pool_in"),
                       (pool_out, 2, "pool_out")):
        check(_int32_vector(t, n), name, " must be contiguous int32 [", "n" if n is None else n,
              "]")
    check(block_table.dim() == 2 and block_table.dtype == torch.int32
          and block_table.stride(1) == 1 and block_table.shape[0] >= R,
          "block_table must be int32 [>= num_reqs, max_blocks] with stride 1 in its last "
          "dimension")
    check(not _overlaps_itself(block_table), "the rows of block_table must not overlap")
    check(slot_mapping.dim() == 1 and slot_mapping.dtype == torch.int64
          and slot_mapping.is_contiguous(), "slot_mapping must be contiguous int64 [T]")
    check(block_size >= 1, "block_size must be >= 1, got ", block_size)
    check(all(t.device == context_lens.device
              for t in (block_table, slot_mapping, seq_lens, query_start_loc, pool_out, query_lens,
                        free_pages, pool_in)),
          "all tensors must be on the device of context_lens")


FAKES = {name: globals()[f"{name}_fake"] for name in NAMES}


_OVERLOADS: dict = {}  # the loaded library's ops, looked up once


def _op(name: str):
    op = _OVERLOADS.get(name)
    if op is None:
        if not hasattr(torch.ops.pth_flash_attn, name):
            raise RuntimeError(
                f"{name}: the op library is not loaded; run python pth-flash-attn_amd/build.py "
                "and import pth_flash_attn.ops"
            )
        op = _OVERLOADS[name] = getattr(torch.ops.pth_flash_attn, name).default
    return op


def build_step_tables(
    block_table: torch.Tensor, slot_mapping: torch.Tensor, seq_lens: torch.Tensor,
    query_start_loc: torch.Tensor, pool_out: torch.Tensor, context_lens: torch.Tensor,
    query_lens: torch.Tensor, free_pages: torch.Tensor, pool_in: torch.Tensor, block_size: int,
) -> None:
    """A step's tables on the GPU, from its request lengths.

    Request r has ``context_lens[r]`` tokens in the cache, in the pages of its
    row of ``block_table``, and brings ``query_lens[r]`` new ones (negative
    lengths count as 0). The pages that the new tokens need and the row lacks
    come from ``free_pages``, request by request, from entry ``pool_in[0]`` on,
    and are appended to the row; nothing else of ``block_table`` is written.

    A request is refused if it needs more pages than the row has entries, or
    pages behind the end of ``free_pages``: it takes none. Pages are given in
    request order, so once they are short every later request that needs one
    is refused too.

    Outputs:
        seq_lens [R]: the lengths with the new tokens (without, if refused).
        query_start_loc [R + 1]: where each request's new tokens begin, at most T.
        slot_mapping [T]: the slot of each new token; -1 for a refused
            request's, where the row holds a negative page number, and behind
            the last request's (a padded batch).
        pool_out [2]: the entries of ``free_pages`` used so far, and the number
            of requests refused in this step. It can be the next step's
            ``pool_in``.

    One launch; allocates nothing, reads nothing back. Outputs overlap neither
    each other nor an input.
    """
    _op("build_step_tables")(block_table, slot_mapping, seq_lens, query_start_loc, pool_out,
                             context_lens, query_lens, free_pages, pool_in, block_size)


def reshape_and_cache_16bit(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                            v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """``key`` / ``value`` [T, Hkv, D] into the paged cache.

    Token t goes to slot ``slot_mapping[t]`` (page ``slot // block_size``,
    in-page slot ``slot % block_size``); a slot outside the cache, as -1, skips
    it. Slots are distinct. The values have the cache's dtype, or are float32
    and rounded once, to nearest even. Cache rows are 16-byte aligned. The two
    caches share no memory, unless both are one view, written by one tensor.
    """
    _op("reshape_and_cache_16bit")(key, value, k_cache, v_cache, slot_mapping)


def paged_decode_fwd(
    out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    block_table: torch.Tensor, seq_lens: torch.Tensor, max_seq_len: int, softmax_scale: float,
    ws: torch.Tensor, window: int = 0,
) -> None:
    """Attention of one new token per request over a paged 16-bit cache, into ``out``.

    ``q`` / ``out`` [R, Hq, D], row r request r's; query head h reads KV head
    h // (Hq / Hkv). (Where ``build_step_tables`` has packed the tokens of a step
    in which some requests bring none, ``cross_attn_fwd`` with that step's
    ``seq_lens`` and ``query_start_loc`` takes the packed rows.) The token sees the
    last ``window`` (all, if 0) of the request's ``seq_lens[r]`` keys, its own among
    them; a request without keys gives zeros. What a page holds outside of these
    keys reaches no output. A NaN or a score of +inf makes its row NaN, and an
    infinite value its column infinite or NaN. ``out`` may be ``q`` itself; other than that they share no memory (both may be
    views of one buffer, as parts of its columns; where telling that apart takes
    more than 2^16 steps, they are refused).
    ``max_seq_len`` bounds the lengths (longer ones are cut there, and at the
    block table's reach). ``ws`` is workspace of
    ``planner.paged16_workspace_floats`` floats; it holds nothing between calls,
    and calls that can run at the same time need one each.

    At most two launches, whose sizes depend on host integers only, so a
    captured graph replays as the lengths change. Allocates nothing, reads
    nothing back, is deterministic. Rows of q, out and the cache are 16-byte
    aligned.
    """
    _op("paged_decode_fwd")(out, q, k_cache, v_cache, block_table, seq_lens, max_seq_len,
                            softmax_scale, ws, window)


def cross_attn_fwd(
    out: torch.Tensor, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    block_table: torch.Tensor, encoder_lens: torch.Tensor, query_start_loc: torch.Tensor,
    max_query_len: int, max_encoder_len: int, softmax_scale: float, ws: torch.Tensor,
) -> None:
    """Cross attention over a paged 16-bit cache of encoder states, into ``out``.

    ``q`` / ``out`` [T, Hq, D]: request r's tokens are ``query_start_loc[r]`` to
    ``query_start_loc[r + 1]``, and each sees all ``encoder_lens[r]`` keys
    (zeros where there are none); there is no causal mask. Rows that belong to no
    request are left as they were. ``max_query_len`` chooses kernel and split (any
    value is correct); ``max_encoder_len``, ``ws`` and the rest are as in ``paged_decode_fwd``.
    """
    _op("cross_attn_fwd")(out, q, k_cache, v_cache, block_table, encoder_lens, query_start_loc,
                          max_query_len, max_encoder_len, softmax_scale, ws)
