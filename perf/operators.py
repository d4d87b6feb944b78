"""Workloads of the operators around a paged cache in the model's own 16-bit
type: the step's block tables and slot map, the cache writer, attention of one
new token per request, and cross attention to an encoder's states.

``listed()`` names the workloads, ``draw(rng)`` gives another one of the same
ranges, ``prepare`` makes a workload's inputs on the GPU, ``run`` makes one
pass: through the framework's entry points where ``own`` is set, in elementary
torch operations in 32 bits otherwise. ``exact`` gives the same outputs in 64
bits, ``work`` the bytes and operations of a pass.

Lengths are drawn from ``len_seed``, so that a workload's work is a property of
the workload; page numbers and values come from the seed. A cache is
``[pages, 2, slots, heads, D]`` (NHD) or ``[pages, 2, heads, slots, D]`` (HND);
page 0 is the null page that the unused tail of every block-table row points
at, and it holds NaN.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False
if str(Path(__file__).resolve().parents[1] / "pth-flash-attn_amd" / "python") not in sys.path:
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "pth-flash-attn_amd" / "python"))

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _tables(name=None, **kw):
    """A step's metadata: ``decodes`` requests of one new token and ``chunks``
    requests of ``chunk_lo``..``chunk_hi`` new tokens, all behind
    ``ctx_lo``..``ctx_hi`` cached ones. ``pad``: the slot map is padded to a
    multiple of it. ``short``: the free pages end before the last requests."""
    case = {"kind": "tables", "decodes": 0, "chunks": 0, "chunk_lo": 1, "chunk_hi": 1,
            "ctx_lo": 0, "ctx_hi": 0, "block": 16, "pad": 8, "short": False, "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _write(name=None, **kw):
    """Keys and values of ``tokens`` tokens, cut from the fused projection's
    output, into the cache; every ``skip``-th token is padding (0: none)."""
    case = {"kind": "write", "tokens": 1, "Hq": 32, "Hkv": 8, "D": 128, "block": 16,
            "layout": "NHD", "dtype": "bf16", "source": "same", "skip": 0}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _decode(name=None, **kw):
    """One new token of ``reqs`` requests with ``len_lo``..``len_hi`` cached
    tokens; ``empty`` of them are padding requests of length 0."""
    case = {"kind": "decode", "reqs": 1, "len_lo": 1, "len_hi": 1, "empty": 0, "window": 0,
            "Hq": 32, "Hkv": 8, "D": 128, "block": 16, "layout": "NHD", "dtype": "bf16",
            "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _cross(name=None, **kw):
    """``reqs`` requests of ``q_lo``..``q_hi`` query tokens against
    ``len_lo``..``len_hi`` encoder states; ``empty`` requests have none."""
    case = {"kind": "cross", "reqs": 1, "q_lo": 1, "q_hi": 1, "len_lo": 1, "len_hi": 1,
            "empty": 0, "Hq": 32, "Hkv": 8, "D": 128, "block": 16, "layout": "NHD",
            "dtype": "bf16", "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The tables of a small decode step: launch latency alone.
        _tables("tables_decode_8", decodes=8, ctx_lo=1000, ctx_hi=4000),
        # A full server's step: 960 decodes beside 64 prompt chunks.
        _tables("tables_mixed_1024", decodes=960, chunks=64, chunk_lo=100, chunk_hi=900,
                ctx_lo=0, ctx_hi=32768, pad=512, len_seed=11),
        # The cache write of a decode step, and of a large prefill step whose
        # keys and values come from an fp32 rotary embedding.
        _write("write_decode_64", tokens=64, skip=9),
        _write("write_prefill_16k", tokens=16384, source="fp32", block=32),
        # One short chat request on one tensor-parallel shard: latency alone.
        _decode("decode_1x1k", Hq=4, Hkv=1, reqs=1, len_lo=1024, len_hi=1024),
        # A full decode batch of ragged lengths: the largest by bytes.
        _decode("decode_64x32k", reqs=64, len_lo=1024, len_hi=32768, len_seed=2024),
        # One very long request.
        _decode("decode_1x128k", reqs=1, len_lo=131072, len_hi=131072),
        # Many requests of small heads without grouping, head-major pages, fp16.
        _decode("decode_d64_mha_48x4k", Hq=16, Hkv=16, D=64, dtype="fp16", layout="HND", reqs=48,
                len_lo=300, len_hi=4096, empty=3, len_seed=48),
        # Head size 256, 6 query heads per KV head, a sliding window, large pages.
        _decode("decode_d256_window_16x64k", Hq=12, Hkv=2, D=256, block=816, reqs=16,
                len_lo=4000, len_hi=65536, window=4096, len_seed=256),
        # Decoding against an encoder's 1,500 states, one request without any.
        _cross("cross_decode_32x1500", Hq=16, Hkv=16, D=64, dtype="fp16", reqs=32, len_lo=1500,
               len_hi=1500, empty=1, len_seed=15),
        # Short prompts of a decoder against as many states as their inputs had.
        _cross("cross_prompt_16x448", Hq=16, Hkv=16, D=64, dtype="fp16", block=32, reqs=16,
               q_lo=4, q_hi=448, len_lo=301, len_hi=1500, len_seed=16),
        # Long prompts against image states, grouped heads: the largest by operations.
        _cross("cross_prefill_4x2k", reqs=4, q_lo=1500, q_hi=2048, len_lo=1601, len_hi=6404,
               len_seed=4),
    ]


# (Hq, Hkv) by head size: whole models and their tensor-parallel shards.
HEADS = {
    64: [(16, 4), (16, 16), (32, 8), (64, 8)],
    128: [(4, 1), (8, 1), (8, 8), (16, 2), (16, 4), (32, 4), (32, 8), (64, 8)],
    256: [(6, 1), (12, 2), (16, 4), (16, 8), (24, 4)],
}
MOST_PADDED = 8.6e9  # bytes of keys and values if all requests were as long as the longest
MOST_BYTES = 4.2e9
MOST_FLOPS = 5.0e11
MOST_SCORES = 1.6e9


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["tables", "write", "decode", "decode", "decode", "cross", "cross", "cross"])
    seed = rng.randrange(1, 1 << 30)
    if what == "tables":
        return _tables(decodes=_log(rng, 1, 1024), chunks=rng.choice([0, _log(rng, 1, 64)]),
                       chunk_lo=rng.randint(1, 100), chunk_hi=_log(rng, 100, 900),
                       ctx_lo=rng.choice([0, 1, 100]), ctx_hi=_log(rng, 100, 65536),
                       block=rng.choice([16, 16, 32, 64, 528, 816]), pad=rng.choice([1, 8, 256]),
                       short=rng.random() < 0.2, len_seed=seed)
    D = rng.choice([64, 128, 128, 256])
    Hq, Hkv = rng.choice(HEADS[D])
    base = {"Hq": Hq, "Hkv": Hkv, "D": D, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "layout": rng.choice(["NHD", "NHD", "HND"]),
            "block": rng.choice([16, 16, 32, 64, 528, 816])}
    if what == "write":
        return _write(tokens=_log(rng, 1, 16384), source=rng.choice(["same", "same", "fp32"]),
                      skip=rng.choice([0, 0, rng.randint(2, 50)]), **base)
    while True:
        kw = dict(base, reqs=_log(rng, 1, 128), len_seed=seed)
        kw["empty"] = rng.choice([0, 0, kw["reqs"] // 8])
        if what == "decode":
            kw["len_hi"] = _log(rng, 8, 131072)
            kw["window"] = rng.choice([0, 0, 0, 500, 1024, 4096])
        else:
            kw["len_hi"] = _log(rng, 8, 8192)
            kw["q_hi"] = rng.choice([1, rng.randint(2, 8), _log(rng, 8, 2048)])
            kw["q_lo"] = rng.randint(1, kw["q_hi"])
        kw["len_lo"] = _log(rng, 1, kw["len_hi"])
        case = _decode(**kw) if what == "decode" else _cross(**kw)
        padded = case["reqs"] * case["len_hi"] * Hkv * D * 4
        scores = case["reqs"] * case["len_hi"] * Hq * case.get("q_hi", 1)
        w = work(case)
        if padded <= MOST_PADDED and scores <= MOST_SCORES and w["bytes"] <= MOST_BYTES \
                and w["flops"] <= MOST_FLOPS:
            return case


def lengths(case):
    """Per request: (query tokens, keys) of an attention workload, (new tokens,
    cached tokens) of a step's tables."""
    rng = np.random.default_rng(case["len_seed"])
    if case["kind"] == "tables":
        R = case["decodes"] + case["chunks"]
        ctx = rng.integers(case["ctx_lo"], max(case["ctx_lo"], case["ctx_hi"]) + 1, R)
        new = np.ones(R, np.int64)
        new[case["decodes"]:] = rng.integers(case["chunk_lo"], max(case["chunk_lo"], case["chunk_hi"]) + 1, case["chunks"])
        return new, ctx
    keys = rng.integers(case["len_lo"], case["len_hi"] + 1, case["reqs"])
    q = rng.integers(case["q_lo"], case["q_hi"] + 1, case["reqs"]) if case["kind"] == "cross" \
        else np.ones(case["reqs"], np.int64)
    keys[rng.permutation(case["reqs"])[: case["empty"]]] = 0
    return q, keys


def work(case):
    if case["kind"] == "tables":
        new, ctx = lengths(case)
        R, T, B = len(new), int(new.sum()), case["block"]
        pages = int((-(-(ctx + new) // B) + (-ctx // B)).sum())
        # Both lengths and the partly filled last page of each request, the
        # free pages taken; the new table entries, lengths, starts and slots.
        return {"bytes": 12 * R + 8 * pages + 8 * R + 8 * T, "flops": 0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "write":
        kept = case["tokens"] - (case["tokens"] // case["skip"] if case["skip"] else 0)
        source = 4 if case["source"] == "fp32" else 2
        return {"bytes": 2 * kept * Hkv * D * (source + 2) + 8 * case["tokens"], "flops": 0}
    q, keys = lengths(case)
    if case.get("window"):
        keys = np.minimum(keys, case["window"])
    T = int(q.sum())
    return {"bytes": int(keys.sum()) * Hkv * D * 4 + 2 * T * Hq * D * 2
            + 4 * int((-(-keys // case["block"])).sum()),
            "flops": 4 * D * Hq * int((q * keys).sum())}


def _cache(case, pages, gen):
    """(storage, K view, V view) of a cache of ``pages`` pages."""
    BS, Hkv, D = case["block"], case["Hkv"], case["D"]
    shape = (pages, 2, BS, Hkv, D) if case["layout"] == "NHD" else (pages, 2, Hkv, BS, D)
    if gen is None:
        kv = torch.zeros(shape, dtype=DTYPES[case["dtype"]], device=DEVICE)
    else:
        kv = torch.randn(shape, dtype=DTYPES[case["dtype"]], device=DEVICE, generator=gen)
        kv[0] = math.nan
    nhd = kv if case["layout"] == "NHD" else kv.transpose(2, 3)
    return kv, nhd[:, 0], nhd[:, 1]


def _table(pages_of, width, first, ids):
    """Block tables of requests of so many pages each, from shuffled page ids;
    the rest of each row points at page 0."""
    n = torch.from_numpy(np.asarray(pages_of)).to(DEVICE)
    start = torch.cumsum(n, 0) - n + first
    j = torch.arange(width, device=DEVICE)
    at = (start[:, None] + j).clamp_max(ids.numel() - 1)
    return torch.where(j < n[:, None], ids[at], 0).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "tables":
        return _prepare_tables(case, gen)
    Hq, Hkv, D, BS = case["Hq"], case["Hkv"], case["D"], case["block"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "write":
        T = case["tokens"]
        source = torch.float32 if case["source"] == "fp32" else dtype
        # Keys and values as the fused projection leaves them, behind the queries.
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=DEVICE).to(source)
        pages = -(-T // BS) + 3
        kv, k, v = _cache(case, pages, None)
        ids = torch.randperm(pages, generator=gen, device=DEVICE)
        pos = torch.arange(T, device=DEVICE)
        slots = ids[pos // BS] * BS + pos % BS
        if case["skip"]:
            slots[case["skip"] - 1 :: case["skip"]] = -1
        return {"case": case, "kv": kv, "k": k, "v": v, "slots": slots,
                "key": qkv[:, Hq * D : (Hq + Hkv) * D].view(T, Hkv, D),
                "value": qkv[:, (Hq + Hkv) * D :].view(T, Hkv, D)}
    q_lens, keys = lengths(case)
    need = -(-keys // BS)
    pages = int(need.sum()) + 4
    kv, k, v = _cache(case, pages, gen)
    ids = 1 + torch.randperm(pages - 1, generator=gen, device=DEVICE)
    table = _table(need, max(1, int(need.max())), 0, ids)
    T = int(q_lens.sum())
    q = torch.randn(T, Hq, D, generator=gen, device=DEVICE).to(dtype)
    s = {"case": case, "kv": kv, "k": k, "v": v, "table": table, "q": q,
         "out": torch.empty_like(q), "scale": 1.0 / math.sqrt(D),
         "lens": torch.from_numpy(keys.astype(np.int32)).to(DEVICE),
         "max_len": max(1, int(keys.max()))}
    if case["kind"] == "cross":
        starts = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        s.update(starts=torch.from_numpy(starts).to(DEVICE), max_q=int(q_lens.max()))
    if own:  # the workspace that a program allocates once at load
        from pth_flash_attn import planner

        cus = torch.cuda.get_device_properties(DEVICE).multi_processor_count
        s["ws"] = torch.empty(planner.paged16_workspace_floats(D=D, num_sms=cus), device=DEVICE)
    return s


def _prepare_tables(case, gen):
    new, ctx = lengths(case)
    R, T, BS = len(new), int(new.sum()), case["block"]
    have, need = -(-ctx // BS), -(-(ctx + new) // BS)
    taken = int((need - have).sum())
    ids = 1 + torch.randperm(int(need.sum()) + 8, generator=gen, device=DEVICE)
    width = int(need.max()) + 2
    free = ids[int(have.sum()) :].to(torch.int32)
    if case["short"]:
        free = free[: 3 + taken - taken // 3]
    as32 = lambda a: torch.from_numpy(np.asarray(a).astype(np.int32)).to(DEVICE)  # noqa: E731
    return {"case": case, "table": _table(have, width, 0, ids), "free": free,
            "ctx": as32(ctx), "new": as32(new),
            "slots": torch.zeros(-(-T // case["pad"]) * case["pad"], dtype=torch.int64, device=DEVICE),
            "seq": torch.zeros(R, dtype=torch.int32, device=DEVICE),
            "starts": torch.zeros(R + 1, dtype=torch.int32, device=DEVICE),
            # Three pages of the list were taken by the step before.
            "pool_in": torch.tensor([3, 0], dtype=torch.int32, device=DEVICE),
            "pool_out": torch.zeros(2, dtype=torch.int32, device=DEVICE)}


def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)[case["kind"]](s, case)


# The framework's calls.


def _own_tables(s, case):
    from pth_flash_attn import ops

    ops.build_step_tables(s["table"], s["slots"], s["seq"], s["starts"], s["pool_out"], s["ctx"],
                          s["new"], s["free"], s["pool_in"], case["block"])
    return s["table"], s["slots"], s["seq"], s["starts"], s["pool_out"]


def _own_write(s, case):
    from pth_flash_attn import ops

    ops.reshape_and_cache_16bit(s["key"], s["value"], s["k"], s["v"], s["slots"])
    return s["kv"]


def _own_decode(s, case):
    from pth_flash_attn import ops

    ops.paged_decode_fwd(s["out"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["max_len"],
                         s["scale"], s["ws"], case["window"])
    return s["out"]


def _own_cross(s, case):
    from pth_flash_attn import ops

    ops.cross_attn_fwd(s["out"], s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"],
                       s["max_q"], s["max_len"], s["scale"], s["ws"])
    return s["out"]


_run_own = {"tables": _own_tables, "write": _own_write, "decode": _own_decode,
            "cross": _own_cross}


# The plain forms.


def _plain_tables(s, case):
    BS, table, free = case["block"], s["table"], s["free"].long()
    ctx, new = s["ctx"].long().clamp_min(0), s["new"].long().clamp_min(0)
    have, need = (ctx + BS - 1) // BS, (ctx + new + BS - 1) // BS
    wide = need <= table.shape[1]
    want = torch.where(wide, need - have, 0)
    first = s["pool_in"][0].long().clamp_min(0) + torch.cumsum(want, 0) - want
    fits = wide & ((want == 0) | (first + want <= free.numel()))
    j = torch.arange(table.shape[1], device=table.device)
    at = (first[:, None] + j - have[:, None]).clamp(0, free.numel() - 1)
    fresh = fits[:, None] & (j >= have[:, None]) & (j < need[:, None])
    table.copy_(torch.where(fresh, free[at], table.long()))
    s["seq"].copy_(torch.where(fits, ctx + new, ctx))
    ends = torch.cumsum(new, 0)
    T = s["slots"].numel()
    s["starts"][:1] = 0
    s["starts"][1:] = ends.clamp_max(T)
    t = torch.arange(T, device=table.device)
    r = torch.searchsorted(ends, t, right=True)
    live = r < ends.numel()
    r = r.clamp_max(ends.numel() - 1)
    p = ctx[r] + t - (ends[r] - new[r])
    page = table[r, (p // BS).clamp(0, table.shape[1] - 1)].long()
    s["slots"].copy_(torch.where(live & fits[r] & (page >= 0), page * BS + p % BS, -1))
    s["pool_out"][0] = s["pool_in"][0].clamp_min(0) + torch.where(fits, want, 0).sum()
    s["pool_out"][1] = (~fits).sum()
    return table, s["slots"], s["seq"], s["starts"], s["pool_out"]


def _plain_write(s, case):
    BS, slots = case["block"], s["slots"]
    # A padding token writes back what the first kept token's slot gets.
    kept = slots >= 0
    first = torch.argmax(kept.to(torch.int32))
    src = torch.where(kept, torch.arange(slots.numel(), device=slots.device), first)
    at = slots[src]
    s["k"].index_put_((at // BS, at % BS), s["key"][src].to(s["k"].dtype))
    s["v"].index_put_((at // BS, at % BS), s["value"][src].to(s["v"].dtype))
    return s["kv"]


def _plain_attend(q, s, lo, most):
    """Attention in 32 bits of q [R, n, Hq, D] over keys [lo, lens) of each
    request, at most ``most`` of them; rows that see no key are 0."""
    R, n, Hq, D = q.shape
    BS, Hkv = s["k"].shape[1], s["k"].shape[2]
    pos = lo[:, None].long() + torch.arange(most, device=q.device)
    seen = (pos < s["lens"][:, None])[:, None, None, :]
    page = torch.gather(s["table"], 1, (pos // BS).clamp_max(s["table"].shape[1] - 1)).long()
    at = pos % BS
    k = s["k"][page, at].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][page, at].float().permute(0, 2, 1, 3).contiguous()
    v = torch.where(seen[:, :, 0, :, None], v, 0.0)
    rows = q.float().view(R, n, Hkv, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, -1, D)
    x = (rows * s["scale"]) @ k
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0.0)
    return o.view(R, Hkv, n, Hq // Hkv, D).permute(0, 2, 1, 3, 4).reshape(R, n, Hq, D)


def _plain_decode(s, case):
    W = case["window"]
    lo = (s["lens"] - W).clamp_min(0) if W else torch.zeros_like(s["lens"])
    most = min(s["max_len"], W or s["max_len"])
    s["out"].copy_(_plain_attend(s["q"][:, None], s, lo, most)[:, 0])
    return s["out"]


def _plain_cross(s, case):
    starts, T = s["starts"].long(), s["q"].shape[0]
    i = torch.arange(s["max_q"], device=starts.device)
    padded = s["q"][(starts[:-1, None] + i).clamp_max(T - 1)]
    o = _plain_attend(padded, s, torch.zeros_like(s["lens"]), s["max_len"])
    t = torch.arange(T, device=starts.device)
    r = torch.searchsorted(starts[1:], t, right=True)
    s["out"].copy_(o[r, t - starts[r]])
    return s["out"]


_run_plain = {"tables": _plain_tables, "write": _plain_write, "decode": _plain_decode,
              "cross": _plain_cross}


def exact(case, seed):
    """The outputs in 64 bits, request by request; none for the tables, which
    are whole numbers."""
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    BS, Hkv, D = case["block"], case["Hkv"], case["D"]
    if case["kind"] == "write":
        kv = s["kv"].double()
        nhd = kv if case["layout"] == "NHD" else kv.transpose(2, 3)
        kept = torch.nonzero(s["slots"] >= 0)[:, 0]
        page, at = s["slots"][kept] // BS, s["slots"][kept] % BS
        nhd[page, 0, at] = s["key"][kept].double()
        nhd[page, 1, at] = s["value"][kept].double()
        return kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    G, t0 = case["Hq"] // Hkv, 0
    for r, (n, L) in enumerate(zip(*lengths(case))):
        n, L = int(n), int(L)
        first = max(0, L - case["window"]) if case.get("window") else 0
        if L:
            ids = s["table"][r, : -(-L // BS)].long()
            k = s["k"][ids].double().reshape(-1, Hkv, D)[first:L]
            v = s["v"][ids].double().reshape(-1, Hkv, D)[first:L]
            for h in range(Hkv):
                kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
                rows = s["q"][t0 : t0 + n, h * G : (h + 1) * G].double().reshape(n * G, D)
                p = torch.softmax(rows @ kt * s["scale"], -1)
                out[t0 : t0 + n, h * G : (h + 1) * G] = (p @ vh).view(n, G, D)
        t0 += n
    return out
