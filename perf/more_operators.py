"""Workloads of the operators around a paged cache in 8-bit floating point with
a scale for each block of 16 tokens and KV head: rotary positions, the cache
writer, its reading back, and attention over it.

``listed()`` names the workloads, ``draw(rng)`` gives another one of the same
ranges, ``prepare`` makes a workload's inputs on the GPU, ``run`` makes one
pass: through the framework's entry points where ``own`` is set, in elementary
torch operations in 32 bits (angles in 64) otherwise. ``exact`` gives the same
outputs in 64 bits, ``work`` the bytes and operations of a pass.

The cache: codes ``float8_e4m3fn`` [pages, 2, slots, heads, D] (NHD) or
[pages, 2, heads, slots, D] (HND); scales ``uint8`` [2, pages, slots / 16, heads],
the biased exponent e of the block's scale 2^(e - 127), 0 for the scale 0. A
block's scale is the smallest that keeps its largest value within 448; it grows
as tokens come, and starts anew with the block's first slot. Codes are returned
as they are, in the floating type whose values are those in units of the scale,
beside the exponents.

Lengths are drawn from ``len_seed``, so that a workload's work is a property of
the workload; page numbers and values come from the seed. Page 0 is the null
page that the unused tail of every block-table row points at; it holds NaN.
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
FP8 = torch.float8_e4m3fn
SPAN = 16  # tokens of a scale


def _rope(name=None, **kw):
    """Queries and keys of ``tokens`` tokens, cut from the fused projection's
    output, rotated in their first ``rot`` columns. ``chunk``: tokens of a
    request (1: a decode step); positions begin anywhere up to ``far``.
    ``scaling``: "none", "linear" (all frequencies by ``factor``) or "ramp" (those
    of few turns within ``original`` positions by ``factor``, those of many
    not, a ramp between)."""
    case = {"kind": "rope", "tokens": 1, "chunk": 1, "far": 4096, "Hq": 32, "Hkv": 8, "D": 128,
            "rot": 128, "interleaved": False, "base": 10000.0, "scaling": "none", "factor": 1.0,
            "original": 4096, "dtype": "bf16", "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _write(name=None, **kw):
    """Keys and values of ``reqs`` requests' ``n_lo``..``n_hi`` new tokens behind
    ``ctx_lo``..``ctx_hi`` cached ones into the cache; every ``skip``-th token
    is padding (0: none)."""
    case = {"kind": "write", "reqs": 1, "n_lo": 1, "n_hi": 1, "ctx_lo": 0, "ctx_hi": 0, "Hq": 32,
            "Hkv": 8, "D": 128, "block": 16, "layout": "NHD", "dtype": "bf16", "skip": 0,
            "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _gather(name=None, **kw):
    """``n_lo``..``n_hi`` cached tokens of each of ``reqs`` requests, from
    position ``ctx_lo``..``ctx_hi`` on, into packed rows."""
    case = {"kind": "gather", "reqs": 1, "n_lo": 1, "n_hi": 1, "ctx_lo": 0, "ctx_hi": 0, "Hkv": 8,
            "D": 128, "block": 16, "layout": "NHD", "dtype": "bf16", "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def _attend(name=None, **kw):
    """``decodes`` requests of ``q`` new tokens behind ``ctx_lo``..``ctx_hi``
    cached ones and ``chunks`` of ``chunk_lo``..``chunk_hi`` behind
    ``pre_lo``..``pre_hi``, causal, all new tokens in the cache; ``empty`` padding
    requests bring none."""
    case = {"kind": "attend", "decodes": 0, "q": 1, "ctx_lo": 0, "ctx_hi": 0, "chunks": 0,
            "chunk_lo": 1, "chunk_hi": 1, "pre_lo": 0, "pre_hi": 0, "empty": 0, "window": 0,
            "Hq": 32, "Hkv": 8, "D": 128, "block": 16, "layout": "NHD", "dtype": "bf16",
            "len_seed": 1}
    case.update(kw)
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # A decode step's queries and keys: launch latency alone.
        _rope("rope_decode_64", tokens=64, far=32768, base=500000.0, len_seed=3),
        # A large prefill step under a long-context scaling.
        _rope("rope_prefill_16k", tokens=16384, chunk=2048, far=131072, base=500000.0,
              scaling="ramp", factor=8.0, original=8192, len_seed=5),
        # Interleaved pairs in a quarter of a wide head, fp16, an odd number of
        # tokens at very far positions.
        _rope("rope_partial_far", tokens=2001, chunk=667, far=1 << 20, Hq=16, Hkv=4, D=256, rot=64,
              interleaved=True, scaling="linear", factor=4.0, dtype="fp16", len_seed=7),
        # The write of a decode step: most tokens fall inside a block.
        _write("write8_decode_64", reqs=64, ctx_lo=100, ctx_hi=9000, skip=9, len_seed=64),
        # The write of a large prefill step: chunks that begin and end inside blocks.
        _write("write8_prefill_16k", reqs=9, n_lo=1500, n_hi=2100, ctx_lo=0, ctx_hi=2000,
               block=32, len_seed=16),
        # Cached prefixes of a few requests back into rows, from inside a block on.
        _gather("gather8_short", reqs=5, n_lo=1, n_hi=90, ctx_lo=0, ctx_hi=37, D=64, Hkv=4,
                dtype="fp16", layout="HND", len_seed=2),
        # Long prefixes into rows, as they leave the card or another kernel takes them.
        _gather("gather8_8x4k", reqs=8, n_lo=1000, n_hi=4096, len_seed=8),
        # One short chat request on one tensor-parallel shard: latency alone.
        _attend("attend8_1x1k", decodes=1, ctx_lo=1023, ctx_hi=1023, Hq=4, Hkv=1),
        # A full decode batch of ragged lengths: the largest by bytes.
        _attend("attend8_64x32k", decodes=64, ctx_lo=1024, ctx_hi=32768, len_seed=2024),
        # Drafts of four tokens in a window, small heads, head-major pages, fp16.
        _attend("attend8_verify_24x8k", decodes=24, q=4, ctx_lo=100, ctx_hi=8192, window=2048,
                empty=2, Hq=16, Hkv=4, D=64, dtype="fp16", layout="HND", len_seed=24),
        # A mixed step of a wide-headed model: two prompt chunks far into their
        # requests beside decodes, large pages.
        _attend("attend8_mixed_d256", decodes=30, ctx_lo=500, ctx_hi=9000, chunks=2, chunk_lo=400,
                chunk_hi=512, pre_lo=4000, pre_hi=16000, Hq=16, Hkv=4, D=256, block=816,
                len_seed=256),
        # Long prompts, some behind a cached prefix: the largest by operations.
        _attend("attend8_prefill_4x2k", chunks=4, chunk_lo=1500, chunk_hi=2048, pre_lo=0,
                pre_hi=6000, len_seed=4),
    ]


# (Hq, Hkv) by head size: whole models and their tensor-parallel shards.
HEADS = {
    64: [(16, 4), (16, 16), (32, 8), (64, 8)],
    128: [(4, 1), (8, 1), (8, 8), (16, 2), (16, 4), (32, 4), (32, 8), (40, 8), (64, 8)],
    256: [(6, 1), (16, 4), (16, 8), (8, 4)],
}
MOST_PADDED = 4.3e9  # bytes of keys and values if all requests were as long as the longest
MOST_BYTES = 2.1e9
MOST_FLOPS = 2.5e11
MOST_SCORES = 1.0e9


def _log(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    what = rng.choice(["rope", "rope", "write", "write", "gather", "attend", "attend", "attend",
                       "attend"])
    seed = rng.randrange(1, 1 << 30)
    D = rng.choice([64, 128, 128, 256])
    Hq, Hkv = rng.choice(HEADS[D])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if what == "rope":
        n = _log(rng, 1, 16384)
        return _rope(tokens=n, chunk=rng.choice([1, _log(rng, 1, n)]), far=_log(rng, 1, 1 << 20),
                     Hq=Hq, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2, D // 4, 2 * rng.randint(1, D // 2)]),
                     interleaved=rng.random() < 0.4, base=rng.choice([10000.0, 500000.0, 1000000.0]),
                     scaling=rng.choice(["none", "linear", "ramp"]), factor=rng.choice([2.0, 4.0, 8.0, 40.0]),
                     original=rng.choice([4096, 8192]),
                     dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), len_seed=seed)
    base = {"Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "layout": rng.choice(["NHD", "NHD", "HND"]),
            "block": rng.choice([16, 16, 32, 64, 528, 816]), "len_seed": seed}
    while True:
        kw = dict(base)
        if what in ("write", "gather"):
            kw["reqs"] = _log(rng, 1, 256)
            kw["n_hi"] = rng.choice([1, rng.randint(2, 40), _log(rng, 16, 16384)])
            kw["n_lo"] = rng.randint(1, kw["n_hi"])
            kw["ctx_hi"] = rng.choice([0, rng.randint(1, 40), _log(rng, 1, 8192)])
            if what == "write":
                kw["dtype"] = rng.choice(["bf16", "bf16", "fp16", "fp32"])
                kw["skip"] = rng.choice([0, 0, rng.randint(2, 50)])
                case = _write(**kw)
            else:
                del kw["Hq"]
                case = _gather(**kw)
            n, ctx = lengths(case)
            if int(n.sum()) <= 17000 and int((n + ctx).sum()) * Hkv * D <= 1 << 28:
                return case
            continue
        kw["decodes"] = _log(rng, 1, 128)
        kw["ctx_hi"] = _log(rng, 8, 131072)
        kw["ctx_lo"] = rng.randint(0, kw["ctx_hi"])
        kw["q"] = rng.choice([1, 1, 1, rng.randint(2, 16)])
        kw["empty"] = rng.choice([0, 0, kw["decodes"] // 8])
        kw["window"] = rng.choice([0, 0, 0, rng.randint(1, 300), 1024, 4096])
        if rng.random() < 0.5:
            kw["chunks"] = _log(rng, 1, 16)
            kw["chunk_hi"] = _log(rng, 8, 2048)
            kw["chunk_lo"] = rng.randint(1, kw["chunk_hi"])
            kw["pre_hi"] = rng.choice([0, rng.randint(1, 100), _log(rng, 8, 8192)])
            if rng.random() < 0.5:
                kw["decodes"], kw["empty"], kw["ctx_lo"], kw["ctx_hi"] = 0, 0, 0, 0
        case = _attend(**kw)
        n, keys = lengths(case)
        padded = len(n) * int(keys.max()) * Hkv * D * 2
        scores = len(n) * int(keys.max()) * Hq * int(n.max())
        w = work(case)
        if padded <= MOST_PADDED and scores <= MOST_SCORES and w["bytes"] <= MOST_BYTES \
                and w["flops"] <= MOST_FLOPS and int(n.sum()):
            return case


def lengths(case):
    """Per request (new tokens, keys with them) of an attention workload, (new
    tokens, cached tokens) of a write, (tokens, first position) of a gather."""
    rng = np.random.default_rng(case["len_seed"])
    if case["kind"] in ("write", "gather"):
        n = rng.integers(case["n_lo"], case["n_hi"] + 1, case["reqs"])
        return n, rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, case["reqs"])
    q = np.full(case["decodes"], case["q"], np.int64)
    ctx = rng.integers(case["ctx_lo"], case["ctx_hi"] + 1, case["decodes"])
    gone = rng.permutation(case["decodes"])[: case["empty"]]
    q[gone], ctx[gone] = 0, 0
    n = np.concatenate([q, rng.integers(case["chunk_lo"], case["chunk_hi"] + 1, case["chunks"])])
    pre = rng.integers(case["pre_lo"], case["pre_hi"] + 1, case["chunks"])
    return n, np.concatenate([ctx, pre]) + n


def work(case):
    elt = 4 if case["dtype"] == "fp32" else 2
    D, Hkv = case["D"], case["Hkv"]
    if case["kind"] == "rope":
        return {"bytes": 2 * case["tokens"] * (case["Hq"] + Hkv) * D * elt + 8 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["Hq"] + Hkv) * case["rot"]}
    n, keys = lengths(case)
    T = int(n.sum())
    if case["kind"] == "write":
        kept = T - (T // case["skip"] if case["skip"] else 0)
        return {"bytes": 2 * kept * Hkv * D * (elt + 1) + 8 * T, "flops": 0}
    if case["kind"] == "gather":
        return {"bytes": 2 * T * Hkv * D * (elt + 1), "flops": 0}
    Hq, W = case["Hq"], case["window"]
    # Query token t of n sees the keys before keys - n + t + 1, the last W of them.
    last = keys - n
    pairs = n * last + n * (n + 1) // 2
    if W:
        cut = np.maximum(keys - W, 0)  # keys that the last token no longer sees
        few = np.minimum(cut, n)
        pairs = pairs - (few * cut - few * (few - 1) // 2)
    read = np.where(n > 0, np.minimum(keys, W + n - 1) if W else keys, 0)
    return {"bytes": int(read.sum()) * Hkv * D * 2 + 2 * T * Hq * D * elt
            + 2 * Hkv * int((-(-read // SPAN)).sum()) + 4 * int((-(-read // case["block"])).sum()),
            "flops": 4 * D * Hq * int(pairs.sum())}


def _cache(case, pages, gen):
    """Codes, scales [2, pages, blocks, heads], and the codes' K and V views, of
    a cache of ``pages`` pages: values of about unit size, block scales within a
    factor of eight of each other."""
    BS, Hkv, D = case["block"], case["Hkv"], case["D"]
    shape = (pages, 2, BS, Hkv, D) if case["layout"] == "NHD" else (pages, 2, Hkv, BS, D)
    kv = torch.empty(shape, dtype=FP8, device=DEVICE)
    step = max(1, (1 << 27) // (2 * BS * Hkv * D))
    for i in range(0, pages, step):
        x = torch.randn(kv[i : i + step].shape, device=DEVICE, generator=gen)
        kv[i : i + step] = (x * 60.0).clamp(-448.0, 448.0).to(FP8)
    scale = torch.randint(120, 123, (2, pages, BS // SPAN, Hkv), device=DEVICE, generator=gen,
                          dtype=torch.uint8)
    kv[0] = torch.full(kv[0].shape, math.nan, device=DEVICE).to(FP8)
    scale[:, 0] = 254
    nhd = kv if case["layout"] == "NHD" else kv.transpose(2, 3)
    return kv, scale, nhd[:, 0], nhd[:, 1]


def _table(pages_of, width, ids):
    """Block tables of requests of so many pages each, from shuffled page ids;
    the rest of each row points at page 0."""
    n = torch.from_numpy(np.asarray(pages_of)).to(DEVICE)
    start = torch.cumsum(n, 0) - n
    j = torch.arange(width, device=DEVICE)
    at = (start[:, None] + j).clamp_max(ids.numel() - 1)
    return torch.where(j < n[:, None], ids[at], 0).to(torch.int32)


def _starts(n):
    return torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).to(DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    Hkv, D, dtype = case["Hkv"], case["D"], DTYPES[case["dtype"]]
    if case["kind"] == "rope":
        Hq, T = case["Hq"], case["tokens"]
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=DEVICE).to(dtype)
        rng = np.random.default_rng(case["len_seed"])
        first = rng.integers(0, case["far"] + 1, -(-T // case["chunk"]))
        pos = (first[:, None] + np.arange(case["chunk"])).reshape(-1)[:T]
        s = {"case": case, "q": qkv[:, : Hq * D].view(T, Hq, D),
             "k": qkv[:, Hq * D : (Hq + Hkv) * D].view(T, Hkv, D),
             "pos": torch.from_numpy(pos).to(DEVICE),
             "freq": torch.from_numpy(_frequencies(case)).to(DEVICE),
             "mscale": _attention_scale(case),
             "q_out": torch.empty(T, Hq, D, dtype=dtype, device=DEVICE),
             "k_out": torch.empty(T, Hkv, D, dtype=dtype, device=DEVICE)}
        if own:  # the frequencies that a program lays out once at load
            from pth_flash_attn import rotary

            s["turns"], s["mscale"] = rotary.rotary_turns(
                case["rot"], base=case["base"], scaling=case["scaling"], factor=case["factor"],
                original_max_position=case["original"], device=DEVICE)
        return s
    n, ctx = lengths(case)
    BS, T = case["block"], int(n.sum())
    need = -(-(n + ctx if case["kind"] != "attend" else ctx) // BS)
    pages = int(need.sum()) + 4
    kv, scale, k, v = _cache(case, pages, gen)
    ids = 1 + torch.randperm(pages - 1, generator=gen, device=DEVICE)
    table = _table(need, max(1, int(need.max())), ids)
    s = {"case": case, "kv": kv, "scale": scale, "k": k, "v": v, "table": table, "starts": _starts(n)}
    if case["kind"] == "gather":
        s.update(first=torch.from_numpy(ctx.astype(np.int32)).to(DEVICE), tokens=T,
                 key=torch.empty(T, Hkv, D, dtype=dtype, device=DEVICE),
                 value=torch.empty(T, Hkv, D, dtype=dtype, device=DEVICE))
        return s
    Hq = case["Hq"]
    if case["kind"] == "write":
        # As the fused projection leaves them, behind the queries: some channels
        # far larger than the others, some tokens larger than those before.
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device=DEVICE)
        loud = torch.rand(qkv.shape[1], generator=gen, device=DEVICE) < 0.02
        late = torch.rand(T, generator=gen, device=DEVICE) < 0.1
        qkv = (qkv * torch.where(loud, 8.0, 1.0) * torch.where(late, 5.0, 1.0)[:, None]).to(dtype)
        r = torch.from_numpy(np.repeat(np.arange(len(n)), n)).to(DEVICE)
        p = torch.from_numpy(np.concatenate([c + np.arange(m) for m, c in zip(n, ctx)])).to(DEVICE)
        slots = table[r, p // BS].long() * BS + p % BS
        if case["skip"]:
            slots[case["skip"] - 1 :: case["skip"]] = -1
        s.update(key=qkv[:, Hq * D : (Hq + Hkv) * D].view(T, Hkv, D),
                 value=qkv[:, (Hq + Hkv) * D :].view(T, Hkv, D), slots=slots)
        return s
    q = torch.randn(T, Hq, D, generator=gen, device=DEVICE).to(dtype)
    s.update(q=q, out=torch.empty_like(q), sm=1.0 / math.sqrt(D), max_q=int(n.max()),
             lens=torch.from_numpy(ctx.astype(np.int32)).to(DEVICE), max_len=int(ctx.max()))
    if own:  # the workspace that a program allocates once at load
        from pth_flash_attn import planner

        cus = torch.cuda.get_device_properties(DEVICE).multi_processor_count
        s["ws"] = torch.empty(planner.fp8_workspace_floats(D=D, num_sms=cus), device=DEVICE)
    return s


def run(s):
    case = s["case"]
    return (_run_own if own else _run_plain)[case["kind"]](s, case)


# The framework's calls.


def _own_rope(s, case):
    from pth_flash_attn import ops

    ops.rotary_embedding(s["q_out"], s["k_out"], s["q"], s["k"], s["pos"], s["turns"],
                         case["interleaved"], s["mscale"])
    return s["q_out"], s["k_out"]


def _own_write(s, case):
    from pth_flash_attn import ops

    ops.reshape_and_cache_fp8(s["key"], s["value"], s["k"], s["v"], s["scale"][0], s["scale"][1],
                              s["slots"])
    return s["kv"], s["scale"]


def _own_gather(s, case):
    from pth_flash_attn import ops

    ops.gather_cache_fp8(s["key"], s["value"], s["k"], s["v"], s["scale"][0], s["scale"][1],
                         s["table"], s["starts"], s["first"])
    return s["key"], s["value"]


def _own_attend(s, case):
    from pth_flash_attn import ops

    ops.paged_attn_fp8_fwd(s["out"], s["q"], s["k"], s["v"], s["scale"][0], s["scale"][1],
                           s["table"], s["lens"], s["starts"], s["max_q"], s["max_len"], s["sm"],
                           s["ws"], case["window"])
    return s["out"]


_run_own = {"rope": _own_rope, "write": _own_write, "gather": _own_gather, "attend": _own_attend}


# The plain forms.


def _frequencies(case):
    """Radians per position of each pair, in 64 bits."""
    rot = case["rot"]
    f = case["base"] ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)
    if case["scaling"] == "linear":
        return f / case["factor"]
    if case["scaling"] == "ramp":
        # Pairs of 32 turns or more within the original positions keep their
        # frequency, those of one or less are scaled; a ramp over the pairs between.
        at = lambda turns: rot * math.log(case["original"] / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))  # noqa: E731
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        keep = 1.0 - np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return f * keep + f / case["factor"] * (1.0 - keep)
    return f


def _attention_scale(case):
    return 0.1 * math.log(case["factor"]) + 1.0 if case["scaling"] == "ramp" else 1.0


def _plain_rope(s, case):
    rot = case["rot"]
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["mscale"]).float()[:, None, :] for f in (torch.cos, torch.sin))

    def rotated(out, x):
        x32 = x[..., :rot].float()
        if case["interleaved"]:
            a, b = x32[..., 0::2], x32[..., 1::2]
        else:
            a, b = x32[..., : rot // 2], x32[..., rot // 2 :]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1 if case["interleaved"] else -2)
        out[..., :rot] = y.reshape(x32.shape).to(out.dtype)
        out[..., rot:] = x[..., rot:]
        return out

    return rotated(s["q_out"], s["q"]), rotated(s["k_out"], s["k"])


def _power(e):
    """2^(e - 127) of whole numbers e up to 254, 0 where e is not positive."""
    return (e.clamp_min(0).to(torch.int32) << 23).view(torch.float32)


def _plain_write(s, case):
    BS, slots = case["block"], s["slots"]
    kept = torch.nonzero(slots >= 0)[:, 0]
    slots = slots[kept]
    ids, of = torch.unique(slots // SPAN, return_inverse=True)  # blocks that get tokens
    page, sub, row = ids // (BS // SPAN), ids % (BS // SPAN), slots % SPAN
    begun = torch.zeros(ids.numel(), dtype=torch.int32, device=DEVICE)
    begun = begun.index_add_(0, of, (row == 0).int()) > 0
    at = sub[:, None] * SPAN + torch.arange(SPAN, device=DEVICE)
    for cache, scale, new in ((s["k"], s["scale"][0], s["key"]), (s["v"], s["scale"][1], s["value"])):
        x = new[kept].float()
        fine = torch.isfinite(x)
        top = torch.where(fine, x.abs(), 0.0).amax(-1).view(torch.int32)
        # The smallest exponent that leaves the largest value at most 448 = 1.75 x 2^8.
        need = (top >> 23) - 8 + ((top & 0x7FFFFF) > 0x600000).int()
        need = torch.where(top == 0, 0, need.clamp_min(1))
        had = scale[page, sub].int()
        old = torch.where(begun[:, None], 0, had)
        e = old.scatter_reduce(0, of[:, None].expand(need.shape), need, "amax")
        # The rows that the block keeps, in units of its scale as it is now.
        codes = cache[page[:, None], at].float()
        moved = torch.where((old > 0) & (e > old), _power(old - e + 127), torch.where((old == 0) & (e > 0), 0.0, 1.0))
        moved = torch.where(begun[:, None], 1.0, moved)
        codes = codes * moved[:, None, :, None]
        unit = x * _power(254 - e[of])[:, :, None]
        codes[of, row] = torch.where(fine, unit, math.nan)
        cache[page[:, None], at] = codes.to(FP8)
        scale[page, sub] = e.to(torch.uint8)
    return s["kv"], s["scale"]


def _plain_values(cache, scale, page, at):
    """Cached rows (page, slot) in 32 bits."""
    return cache[page, at].float() * _power(scale[page, at // SPAN].int())[..., None]


def _plain_gather(s, case):
    BS = case["block"]
    t = torch.arange(s["tokens"], device=DEVICE)
    r = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    p = s["first"][r].long() + t - s["starts"][r].long()
    page, at = s["table"][r, p // BS].long(), p % BS
    s["key"].copy_(_plain_values(s["k"], s["scale"][0], page, at))
    s["value"].copy_(_plain_values(s["v"], s["scale"][1], page, at))
    return s["key"], s["value"]


def _plain_attend(s, case):
    BS, Hkv, D, W = case["block"], case["Hkv"], case["D"], case["window"]
    Hq, G = case["Hq"], case["Hq"] // case["Hkv"]
    starts, T = s["starts"].long(), s["q"].shape[0]
    n, lens = starts[1:] - starts[:-1], s["lens"].long()
    R, N = n.numel(), s["max_q"]
    # A window leaves the last W + N - 1 keys of a request at most.
    most = min(s["max_len"], W + N - 1) if W else s["max_len"]
    lo = (lens - most).clamp_min(0) if W else torch.zeros_like(lens)
    pos = lo[:, None] + torch.arange(most, device=DEVICE)
    page = torch.gather(s["table"], 1, (pos // BS).clamp_max(s["table"].shape[1] - 1)).long()
    here = (pos < lens[:, None])[:, :, None, None]
    k = torch.where(here, _plain_values(s["k"], s["scale"][0], page, pos % BS), 0.0)
    v = torch.where(here, _plain_values(s["v"], s["scale"][1], page, pos % BS), 0.0)
    k = k.permute(0, 2, 3, 1).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()
    i = torch.arange(N, device=DEVICE)
    q = s["q"][(starts[:-1, None] + i).clamp_max(T - 1)].float()
    q = q.view(R, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(R, Hkv, N * G, D)
    x = (q * s["sm"]) @ k
    end = (lens - n)[:, None] + i + 1  # one past the last key of a token
    seen = (pos[:, None, :] < end[:, :, None]) & (pos < lens[:, None])[:, None, :]
    if W:
        seen &= pos[:, None, :] >= end[:, :, None] - W
    x = torch.where(seen[:, None, :, None, :], x.view(R, Hkv, N, G, -1), -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = p.view(R, Hkv, N * G, -1) @ v
    o = torch.where(total > 0, o.view(R, Hkv, N, G, D) / total, 0.0)
    o = o.permute(0, 2, 1, 3, 4).reshape(R, N, Hq, D)
    t = torch.arange(T, device=DEVICE)
    r = torch.searchsorted(starts[1:], t, right=True)
    s["out"].copy_(o[r, t - starts[r]])
    return s["out"]


_run_plain = {"rope": _plain_rope, "write": _plain_write, "gather": _plain_gather,
              "attend": _plain_attend}


# The definitions in 64 bits.


def _exact_rope(s, case):
    """Each pair as a complex number, turned."""
    rot, half = case["rot"], case["rot"] // 2
    angle = s["pos"].double()[:, None, None] * torch.from_numpy(_frequencies(case)).to(DEVICE)
    turn = torch.polar(torch.full_like(angle, _attention_scale(case)), angle)
    outs = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        first = slice(0, rot, 2) if case["interleaved"] else slice(0, half)
        second = slice(1, rot, 2) if case["interleaved"] else slice(half, rot)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_write(s, case):
    """Block by block on the host, the codes as values in units of their scale."""
    BS, Hkv = case["block"], case["Hkv"]
    kv, scale = s["kv"].double().cpu().numpy(), s["scale"].cpu().numpy().astype(np.int64)
    nhd = kv if case["layout"] == "NHD" else kv.swapaxes(2, 3)
    new = (s["key"].double().cpu().numpy(), s["value"].double().cpu().numpy())
    tokens = {}
    for t, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            tokens.setdefault(slot // SPAN, []).append((slot % SPAN, t))
    for block, rows in tokens.items():
        page, sub = divmod(block, BS // SPAN)
        at = [sub * SPAN + row for row, _ in rows]
        rest = [sub * SPAN + i for i in range(SPAN) if sub * SPAN + i not in at]
        begun = any(row == 0 for row, _ in rows)
        for j in (0, 1):
            x = new[j][[t for _, t in rows]]  # [rows, heads, D]
            top = np.abs(x).max((0, 2))
            old = np.zeros(Hkv, np.int64) if begun else scale[j, page, sub]
            with np.errstate(divide="ignore"):
                need = np.where(top > 0, np.ceil(np.log2(top / 448.0)) + 127, 0).astype(np.int64)
            e = np.maximum(old, need)
            if not begun:
                nhd[page, j, rest] *= np.where(old > 0, np.exp2((old - e).astype(np.float64)), (e == 0) * 1.0)[:, None]
            nhd[page, j, at] = x * np.where(e > 0, np.exp2(127.0 - e), 0.0)[:, None]
    return torch.from_numpy(kv).to(DEVICE), None


def _exact_gather(s, case):
    Hkv, D, BS = case["Hkv"], case["D"], case["block"]
    rows = ([], [])
    for r, (n, c) in enumerate(zip(*lengths(case))):
        ids = s["table"][r, c // BS : -(-(c + n) // BS)].long()
        off = int(c % BS)
        for j, cache in enumerate((s["k"], s["v"])):
            e = s["scale"][j][ids].double().repeat_interleave(SPAN, 1)
            x = cache[ids].double() * torch.exp2(e - 127.0)[..., None]
            rows[j].append(x.reshape(-1, Hkv, D)[off : off + int(n)])
    return torch.cat(rows[0]), torch.cat(rows[1])


def _exact_attend(s, case):
    Hkv, D, BS, W = case["Hkv"], case["D"], case["block"], case["window"]
    G, t0 = case["Hq"] // Hkv, 0
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for r, (n, L) in enumerate(zip(*lengths(case))):
        n, L = int(n), int(L)
        if n == 0:
            continue
        ids = s["table"][r, : -(-L // BS)].long()
        k, v = ((cache[ids].double() * torch.exp2(scale[ids].double().repeat_interleave(SPAN, 1) - 127.0)[..., None])
                .reshape(-1, Hkv, D)[:L] for cache, scale in ((s["k"], s["scale"][0]), (s["v"], s["scale"][1])))
        q_at = torch.arange(L - n, L, device=DEVICE)[:, None]
        k_at = torch.arange(L, device=DEVICE)[None, :]
        hidden = k_at > q_at
        if W:
            hidden |= k_at <= q_at - W
        hidden = hidden[:, None, :].expand(n, G, L).reshape(n * G, L)
        for h in range(Hkv):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            rows = s["q"][t0 : t0 + n, h * G : (h + 1) * G].double().reshape(n * G, D)
            p = torch.softmax((rows @ kt * s["sm"]).masked_fill(hidden, -math.inf), -1)
            out[t0 : t0 + n, h * G : (h + 1) * G] = (p @ vh).view(n, G, D)
        t0 += n
    return out


def exact(case, seed):
    """The outputs in 64 bits; none for the scales' exponents, which are whole numbers."""
    s = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "gather": _exact_gather,
            "attend": _exact_attend}[case["kind"]](s, case)
