"""Inputs, references and tolerances of the ops around a paged 8-bit cache
(test infrastructure).

Tolerance of an attention output, element by element, from the roundings made
(h = finfo.eps / 2 of the 16-bit type, u = 2^-24; A = sum p |v| / sum p, the
weighted mean of |v|; S = the largest sum |q k| scale of the row):

* the output's own rounding: h |out| (half a spacing of the type's subnormals
  near 0);
* P: rounded once to bf16 (8 significant bits: half a step is 2^-8 of the value)
  where many rows of bf16 queries are computed, 2^-8 A; a bf16 pair otherwise,
  whose second rounds the first's remainder, 2^-16 A;
* scores in 32 bits: D products, D additions, the block's scale, the softmax's
  and its conversion to powers of two, each u of a partial sum that is at most S:
  weights off by a factor 1 +- (D + 5) u S, for numerator and denominator:
  2 (D + 5) u S A;
* exp2 (2 u), and sums over L keys in 32 bits, numerator and denominator:
  2 (L + 8) u A.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from pth_flash_attn import ops, planner

DEV = "cuda"
FP8 = torch.float8_e4m3fn
SPAN = 16
NAN_CODE = 0x7F


@dataclass
class Cache8:
    codes: torch.Tensor  # storage, uint8
    k: torch.Tensor
    v: torch.Tensor
    ks: torch.Tensor
    vs: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor
    keys: list  # per request: (K, V) [L, Hkv, D] as 64-bit values

    @property
    def views(self):
        return self.k, self.v, self.ks, self.vs


def workspace(D, device=DEV):
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    # NaN: a slot that is read without having been written shows.
    return torch.full((planner.fp8_workspace_floats(D=D, num_sms=cus),), math.nan, device=device)


def storage(pages, block, Hkv, D, layout="NHD", fill=NAN_CODE, device=DEV, pad=0):
    """(codes as uint8, K view, V view, K scales, V scales); ``pad`` bytes between pages."""
    inner = (2, block, Hkv, D) if layout == "NHD" else (2, Hkv, block, D)
    flat = torch.full((pages, math.prod(inner) + pad), fill, dtype=torch.uint8, device=device)
    codes = flat[:, : math.prod(inner)].view(pages, *inner)
    nhd = codes if layout == "NHD" else codes.transpose(2, 3)
    scale = torch.full((2, pages, block // SPAN, Hkv), 254, dtype=torch.uint8, device=device)
    return codes, nhd[:, 0].view(FP8), nhd[:, 1].view(FP8), scale[0], scale[1]


def power(e):
    """2^(e - 127) in 64 bits, 0 for e = 0, above 246 as 246."""
    e = e.clamp_max(246).double()
    return torch.where(e > 0, torch.exp2(e - 127.0), 0.0)


def make_cache(lens, *, Hkv, D, block, seed, layout="NHD", spare=2, width=None, pad=0, spread=3):
    """A cache of shuffled pages: NaN codes and the largest exponent wherever no
    request's token lies, page 0 (the null page of the tables' unused entries)
    among it. Exponents of blocks differ by up to ``spread``."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-max(n, 0) // block) for n in lens]
    pages = sum(need) + spare + 1
    codes, k, v, ks, vs = storage(pages, block, Hkv, D, layout, pad=pad)
    ids = 1 + torch.randperm(pages - 1, generator=gen, device=DEV)
    table = torch.zeros(len(lens), max(need + [width or 1]), dtype=torch.int32, device=DEV)
    keys, at = [], 0
    for r, L in enumerate(lens):
        mine = ids[at : at + need[r]]
        at += need[r]
        table[r, : need[r]] = mine.to(torch.int32)
        pos = torch.arange(max(L, 0), device=DEV)
        row = []
        for cache, scale in ((k, ks), (v, vs)):
            x = (torch.randn(len(pos), Hkv, D, generator=gen, device=DEV) * 60).clamp(-448, 448)
            x = x.to(FP8)
            e = torch.randint(121 - spread // 2, 122 + spread // 2, (-(-len(pos) // SPAN), Hkv),
                              generator=gen, device=DEV).to(torch.uint8)
            if len(pos):
                page = mine[pos // block]
                cache.view(torch.uint8)[page, pos % block] = x.view(torch.uint8)
                first = pos[::SPAN]
                scale[mine[first // block], first % block // SPAN] = e
                row.append(x.double() * power(e)[pos // SPAN][..., None])
            else:
                row.append(x.double())
        keys.append(tuple(row))
    return Cache8(codes, k, v, ks, vs, table, torch.tensor(lens, dtype=torch.int32, device=DEV),
                  keys)


def starts_of(q_lens):
    s = torch.zeros(len(q_lens) + 1, dtype=torch.int32)
    s[1:] = torch.tensor(list(q_lens)).cumsum(0).to(torch.int32)
    return s.to(DEV)


def reference(q, keys, q_lens, scale, *, window=0, causal=True, single=False):
    """(out, tolerance) in 64 bits; rows of no request NaN with tolerance 0.
    ``single``: P rounded once to bf16."""
    T, Hq, D = q.shape
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    info = torch.finfo(q.dtype)
    h, u = info.eps / 2, 2.0**-24
    t0 = 0
    for n, (k, v) in zip(q_lens, keys):
        L, Hkv = k.shape[:2]
        G = Hq // Hkv
        own = torch.arange(L - n, L, device=q.device)[:, None]
        at = torch.arange(L, device=q.device)[None, :]
        seen = (at <= own) if causal else torch.ones(n, L, dtype=torch.bool, device=q.device)
        if window:
            seen = seen & (at > own - window)
        seen = seen[:, None, :].expand(n, G, L).reshape(n * G, L)
        for hd in range(Hkv if n else 0):
            rows = q[t0 : t0 + n, hd * G : (hd + 1) * G].double().reshape(n * G, D)
            kt, vh = k[:, hd].t().contiguous(), v[:, hd].contiguous()
            bad = vh.isnan()
            vh = vh.nan_to_num(0.0)
            # A NaN in K reaches the rows that see it alone.
            x = torch.where(seen, rows @ kt * scale, -math.inf)
            top = x.amax(-1, keepdim=True) if L else torch.zeros(n * G, 1, device=q.device)
            p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total != 0, p / total, 0.0)
            S = torch.where(seen, rows.abs() @ kt.abs() * scale, 0.0)
            S = S.nan_to_num(0.0).amax(-1, keepdim=True) if L else top
            o, A = p @ vh, p @ vh.abs()
            o = torch.where(seen.double() @ bad.double() > 0, math.nan, o)
            t = h * o.abs() + info.smallest_normal * h + A * (
                (2.0**-8 if single else 2.0**-16) + 2 * (D + 5) * u * S + 2 * (L + 8) * u)
            out[t0 : t0 + n, hd * G : (hd + 1) * G] = o.view(n, G, D)
            tol[t0 : t0 + n, hd * G : (hd + 1) * G] = t.view(n, G, D)
        t0 += n
    return out, tol


def assert_close(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    if not got.numel():
        return
    excess = ((got.double() - want).abs() - tol).nan_to_num(0.0)
    assert excess.max().item() <= 0.0, f"{excess.max().item():.3g} beyond the tolerance"


def attend(c, q, q_lens, scale, *, window=0, causal=True, max_len=None, max_q=None, ws=None,
           out=None, starts=None, table=None, lens=None, decode=False):
    out = torch.full_like(q, math.nan) if out is None else out
    most = max([len(k) for k, _ in c.keys] + [1]) if max_len is None else max_len
    if starts is None and not decode:
        starts = starts_of(q_lens)
    ops.paged_attn_fp8_fwd(out, q, *c.views, c.table if table is None else table,
                           c.lens if lens is None else lens, starts,
                           (max(q_lens) if q_lens else 0) if max_q is None else max_q, most, scale,
                           workspace(q.shape[2]) if ws is None else ws, window, causal)
    return out


def queries(T, Hq, D, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(T, Hq, D, generator=gen, device=DEV).to(dtype)


def exponent_for(top):
    """The smallest e, 1 to 246, with top <= 448 x 2^(e - 127), of finite values
    top >= 0 in 64 bits; 0 for 0."""
    e = torch.ceil(torch.log2(top / 448.0)) + 127
    # log2's rounding is far finer than the gap between two 32-bit values.
    return torch.where(top > 0, e.clamp(1, 246), 0.0).to(torch.int64)


def write_reference(key, value, k, v, ks, vs, slots):
    """What the writer leaves in copies of the cache: (k, v as uint8, ks, vs) on
    the CPU, block by block."""
    out = []
    tokens: dict[int, dict[int, int]] = {}
    pages, block = k.shape[:2]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * block:
            tokens.setdefault(s // SPAN, {})[s % SPAN] = t
    for cache, scale, new in ((k, ks, key), (v, vs, value)):
        code, exp = cache.view(torch.uint8).cpu().clone(), scale.cpu().clone()
        x = new.cpu().double()
        for b, rows in tokens.items():
            page, sub = divmod(b, block // SPAN)
            src = x[list(rows.values())]
            fine = torch.isfinite(src)
            need = exponent_for(torch.where(fine, src.abs(), 0.0).amax((0, 2)))
            had = exp[page, sub].long().clamp_max(246)
            old = torch.zeros_like(had) if 0 in rows else had
            e = torch.maximum(old, need)
            at = [sub * SPAN + i for i in rows]
            rest = [sub * SPAN + i for i in range(SPAN) if i not in rows]
            unit = torch.where(e > 0, torch.exp2(127.0 - e.double()), 0.0)
            y = (src * unit[:, None]).clamp(-448.0, 448.0)
            y = torch.where(fine, y, math.nan)
            code[page, at] = y.float().to(FP8).view(torch.uint8)
            if rest and 0 not in rows:
                kept = code[page, rest]
                move = torch.where(old > 0, torch.exp2((old - e).double()), 0.0)
                moved = (kept.view(FP8).double() * move[:, None]).float().to(FP8).view(torch.uint8)
                code[page, rest] = torch.where((e > old)[:, None], moved, kept)
            exp[page, sub] = e.to(torch.uint8)
        out.append((code, exp))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def assert_codes(got, want):
    """Equal codes; a NaN may have either sign."""
    got, want = got.cpu(), want.cpu()
    nan = (want & 0x7F) == NAN_CODE
    assert torch.equal((got & 0x7F) == NAN_CODE, nan)
    assert torch.equal(got.masked_fill(nan, 0), want.masked_fill(nan, 0))
