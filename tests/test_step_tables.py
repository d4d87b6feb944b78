"""build_step_tables against the formulas, request by request in Python."""

from __future__ import annotations

import pytest
import torch

from pth_flash_attn import ops

needs_op = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
MARK = -77


def expected(table, ctx, new, free, cursor, block, T):
    """The outputs as lists, and the table as written."""
    table = [list(r) for r in table]
    seq, starts, slots, refused = [], [], [-1] * T, 0
    cursor0 = asked = max(cursor, 0)
    taken, tok = cursor0, 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        have, need = -(-c // block), -(-(c + n) // block)
        wide = need <= len(table[r])
        want = need - have if wide else 0
        first = asked
        asked += want
        fits = wide and (want == 0 or first + want <= len(free))
        starts.append(min(tok, T))
        seq.append(c + n if fits else c)
        refused += not fits
        if fits:
            table[r][have:need] = free[first : first + want] if want else table[r][have:need]
            taken = first + want if want else taken
            for i in range(n):
                page = table[r][(c + i) // block]
                if tok + i < T and page >= 0:
                    slots[tok + i] = page * block + (c + i) % block
        tok += n
    starts.append(min(tok, T))
    return table, slots, seq, starts, [taken, refused]


def build(table, ctx, new, free, cursor, block, T, device="cuda"):
    as32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    R = len(ctx)
    outs = (as32(table).view(R, -1), torch.full((T,), MARK, dtype=torch.int64, device=device),
            as32([MARK] * R), as32([MARK] * (R + 1)), as32([MARK, MARK]))
    ops.build_step_tables(*outs, as32(ctx), as32(new), as32(free), as32([cursor, 99]), block)
    return [t.tolist() for t in outs]


def check(table, ctx, new, free, cursor, block, T):
    got = build(table, ctx, new, free, cursor, block, T)
    want = expected(table, ctx, new, free, cursor, block, T)
    for name, g, w in zip(("block_table", "slot_mapping", "seq_lens", "query_start_loc",
                           "pool_out"), got, want):
        assert g == list(w), name


def batch(R, block, seed, most=60, width=None):
    gen = torch.Generator().manual_seed(seed)
    ctx = torch.randint(0, 5 * block, (R,), generator=gen).tolist()
    new = torch.randint(0, most, (R,), generator=gen).tolist()
    need = max(-(-(c + n) // block) for c, n in zip(ctx, new))
    width = need + 1 if width is None else width
    ids = torch.randperm(R * width, generator=gen).tolist()
    table = [[ids[r * width + j] if j < -(-ctx[r] // block) else MARK for j in range(width)]
             for r in range(R)]
    free = [100_000 + i for i in torch.randperm(R * (need + 1), generator=gen).tolist()]
    return table, ctx, new, free


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1, 2, 63, 64, 65, 256, 257, 1024, 1025, 2500])
@pytest.mark.parametrize("block", [1, 16, 48, 816])
def test_batches(R, block):
    table, ctx, new, free = batch(R, block, R + block)
    check(table, ctx, new, free, 5, block, sum(new) + 9)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [40, 700])
def test_short_pool_refuses_in_order(R):
    table, ctx, new, free = batch(R, 16, 3)
    total = sum(-(-(c + n) // 16) - -(-c // 16) for c, n in zip(ctx, new))
    for left in (0, 1, total // 2, total - 1, total, total + 1):
        check(table, ctx, new, free[:left], 0, 16, sum(new))
    check(table, ctx, new, free[:20], 25, 16, sum(new))  # a cursor past the end


@pytest.mark.gpu
def test_rows_too_narrow_and_negative_pages():
    table, ctx, new, free = batch(300, 16, 4, width=4)
    table[7][0] = -1
    check(table, ctx, new, free, 0, 16, sum(new) + 3)


@pytest.mark.gpu
def test_lengths_out_of_range():
    """Negative lengths count as 0; enormous ones are refused without a sum
    wrapping; more tokens than slots are cut."""
    big = 2**31 - 1
    ctx = [-4, 10, big, 20, 0, big, 16]
    new = [3, -2, big, 5, big, 0, 40]
    table = [[r * 10 + j for j in range(6)] for r in range(7)]
    for T in (1, 12, 64):  # Python's integers do not wrap
        check(table, ctx, new, list(range(500, 520)), -9, 16, T)


@pytest.mark.gpu
def test_large_chunk_and_one_slot():
    """One request of many pages spread over all work-groups; no slots."""
    n, block = 70_000, 16
    width = -(-n // block) + 1
    check([[MARK] * width], [0], [n], list(range(10, 10 + width + 5)), 3, block, n + 100)
    check([[MARK] * width, [MARK] * width], [0, 5], [n, 0], list(range(width)), 0, block, 0)


@pytest.mark.gpu
def test_no_requests():
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    slots = torch.zeros(5, dtype=torch.int64, device="cuda")
    qsl, out = torch.full((1,), 9, dtype=torch.int32, device="cuda"), torch.zeros(
        2, dtype=torch.int32, device="cuda")
    ops.build_step_tables(e.view(0, 4), slots, e, qsl, out, e, e, e,
                          torch.tensor([4, 0], dtype=torch.int32, device="cuda"), 16)
    assert slots.tolist() == [-1] * 5 and qsl.tolist() == [0] and out.tolist() == [4, 0]


@pytest.mark.gpu
def test_graph_of_two_steps_advances():
    """Two captured steps that hand lengths and cursor to each other, replayed."""
    R, block, width = 5, 16, 40
    i32 = dict(dtype=torch.int32, device="cuda")
    ctx = [torch.tensor([3, 16, 0, 40, 31], **i32), torch.zeros(R, **i32)]
    pool = [torch.zeros(2, **i32), torch.zeros(2, **i32)]
    table = torch.full((R, width), MARK, **i32)
    have = [1, 1, 0, 3, 2]
    for r, h in enumerate(have):
        table[r, :h] = torch.arange(1000 + 10 * r, 1000 + 10 * r + h)
    one = torch.tensor([1, 7, 0, 1, 20], **i32)
    free = torch.arange(500, **i32)
    slots = torch.zeros(32, dtype=torch.int64, device="cuda")
    qsl = torch.zeros(R + 1, **i32)

    def two():
        for i in (0, 1):
            ops.build_step_tables(table, slots, ctx[1 - i], qsl, pool[1 - i], ctx[i], one, free,
                                  pool[i], block)

    state = [t.clone() for t in (ctx[0], pool[0], table)]
    two()
    torch.cuda.synchronize()
    for t, s in zip((ctx[0], pool[0], table), state):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        two()
    py_table, py_ctx, cursor = table.tolist(), ctx[0].tolist(), 0
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for _ in range(2):
            py_table, py_slots, py_ctx, _, (cursor, _) = expected(
                py_table, py_ctx, one.tolist(), free.tolist(), cursor, block, 32)
        assert table.tolist() == py_table and ctx[0].tolist() == py_ctx
        assert slots.tolist() == py_slots and pool[0].tolist() == [cursor, 0]
        torch.ones(8, device="cuda").sum().item()


def _cpu_args(R=3, T=8):
    i32 = dict(dtype=torch.int32)
    return dict(block_table=torch.zeros(R, 4, **i32), slot_mapping=torch.zeros(T, dtype=torch.int64),
                seq_lens=torch.zeros(R, **i32), query_start_loc=torch.zeros(R + 1, **i32),
                pool_out=torch.zeros(2, **i32), context_lens=torch.zeros(R, **i32),
                query_lens=torch.zeros(R, **i32), free_pages=torch.zeros(9, **i32),
                pool_in=torch.zeros(2, **i32), block_size=16)


@needs_op
@pytest.mark.parametrize(("change", "message"), [
    (dict(), "computes on CUDA tensors only"),
    (dict(context_lens=torch.zeros(3)), "context_lens must be contiguous int32"),
    (dict(query_lens=torch.zeros(2, dtype=torch.int32)), r"query_lens must be contiguous int32 \[3\]"),
    (dict(query_start_loc=torch.zeros(3, dtype=torch.int32)), r"query_start_loc .* \[4\]"),
    (dict(pool_in=torch.zeros(1, dtype=torch.int32)), "pool_in must be"),
    (dict(block_table=torch.zeros(2, 4, dtype=torch.int32)), "block_table must be int32"),
    (dict(block_table=torch.zeros(4, 3, dtype=torch.int32).t()), "block_table must be int32"),
    (dict(slot_mapping=torch.zeros(8, dtype=torch.int32)), "slot_mapping must be contiguous int64"),
    (dict(block_size=0), "block_size must be >= 1"),
    (dict(block_size=-16), "block_size must be >= 1"),
])
def test_refusals(change, message):
    args = {**_cpu_args(), **change}
    with pytest.raises(RuntimeError, match=message):
        ops.build_step_tables(**args)
    if change:  # the fake refuses alike
        with pytest.raises(RuntimeError, match=message):
            ops.ops16.build_step_tables_fake(**args)


@needs_op
def test_overlaps_are_refused():
    args = _cpu_args()
    args["seq_lens"] = args["context_lens"]
    with pytest.raises(RuntimeError, match="an output must not overlap an input"):
        ops.build_step_tables(**args)
    args = _cpu_args()
    both = torch.zeros(10, dtype=torch.int32)
    args["seq_lens"], args["query_start_loc"] = both[:3], both[2:6]
    with pytest.raises(RuntimeError, match="the outputs must not overlap each other"):
        ops.build_step_tables(**args)


@needs_op
def test_rows_that_overlap_are_refused():
    args = _cpu_args()
    args["block_table"] = torch.zeros(1, 4, dtype=torch.int32).expand(3, 4)
    for f in (ops.build_step_tables, ops.ops16.build_step_tables_fake):
        with pytest.raises(RuntimeError, match="the rows of block_table must not overlap"):
            f(**args)
