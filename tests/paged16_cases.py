"""Inputs, 64-bit references and tolerances of the ops around a paged 16-bit
cache (test infrastructure).

Tolerance of an attention output, element by element, from the roundings made
(h = finfo.eps / 2 of the 16-bit type, u = 2^-24; A = sum p |v| / sum p, the
weighted mean of |v|; S = the largest sum |q k| scale of the row):

* the output's own rounding: h |out| (half a spacing of the type's subnormals
  near 0);
* P rounded once to the type: h A (the kernel of many rows; the one of few
  rows keeps the remainder too, h^2 A);
* scores in 32 bits: D products, D additions, the scale and its conversion to
  powers of two, each u of a partial sum that is at most S: weights off by a
  factor 1 +- (D + 4) u S, for numerator and denominator: 2 (D + 4) u S A;
* exp2 (2 u), and sums over L keys in 32 bits, numerator and denominator:
  2 (L + 8) u A.
"""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from pth_flash_attn import ops, planner
from pth_flash_attn.cache import paged16_views

DEV = "cuda"


@dataclass
class Cache16:
    kv: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    table: torch.Tensor
    lens: torch.Tensor
    keys: list  # per request: (K, V) [L, Hkv, D] as stored


def workspace(D, device=DEV):
    cus = torch.cuda.get_device_properties(device).multi_processor_count
    # NaN: a slot that is read without having been written shows.
    return torch.full((planner.paged16_workspace_floats(D=D, num_sms=cus),), math.nan,
                      device=device)


def make_cache(lens, *, Hkv, D, block, dtype, seed, layout="NHD", spare=2, scale=1.0, width=None,
               pad=0):
    """A cache of shuffled pages: NaN wherever no request's token lies, page 0
    (the null page of the tables' unused entries) among it. ``pad``: that many
    values between the pages."""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // block) for n in lens]
    pages = sum(need) + spare + 1
    inner = (2, block, Hkv, D) if layout == "NHD" else (2, Hkv, block, D)
    flat = torch.full((pages, math.prod(inner) + pad), math.nan, dtype=dtype, device=DEV)
    kv = flat[:, : math.prod(inner)].view(pages, *inner)
    k, v = paged16_views(kv, layout=layout)
    ids = 1 + torch.randperm(pages - 1, generator=gen, device=DEV)
    table = torch.zeros(len(lens), max(need + [width or 1]), dtype=torch.int32, device=DEV)
    keys, at = [], 0
    for r, L in enumerate(lens):
        mine = ids[at : at + need[r]]
        at += need[r]
        table[r, : need[r]] = mine.to(torch.int32)
        kk = (scale * torch.randn(L, Hkv, D, generator=gen, device=DEV)).to(dtype)
        vv = torch.randn(L, Hkv, D, generator=gen, device=DEV).to(dtype)
        pos = torch.arange(L, device=DEV)
        if L:
            k[mine[pos // block], pos % block] = kk
            v[mine[pos // block], pos % block] = vv
        keys.append((kk, vv))
    return Cache16(kv, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), keys)


def starts_of(q_lens):
    s = torch.zeros(len(q_lens) + 1, dtype=torch.int32)
    s[1:] = torch.tensor(list(q_lens)).cumsum(0).to(torch.int32)
    return s.to(DEV)


def reference(q, keys, q_lens, scale, window=0, pair=False):
    """(out, tolerance) in 64 bits; rows of no request NaN with tolerance 0."""
    T, Hq, D = q.shape
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    info = torch.finfo(q.dtype)
    h, u = info.eps / 2, 2.0**-24
    t0 = 0
    for n, (k, v) in zip(q_lens, keys):
        L, Hkv = k.shape[:2]
        G = Hq // Hkv
        first = max(0, L - window) if window else 0
        kd, vd = k[first:].double(), v[first:].double()
        for hd in range(Hkv):
            rows = q[t0 : t0 + n, hd * G : (hd + 1) * G].double().reshape(n * G, D)
            if L == 0:
                o = t = torch.zeros(n * G, D, dtype=torch.float64, device=q.device)
            elif n:
                kt = kd[:, hd].t().contiguous()
                p = torch.softmax(rows @ kt * scale, -1)
                S = (rows.abs() @ kt.abs() * scale).amax(-1, keepdim=True)
                o = p @ vd[:, hd].contiguous()
                A = p @ vd[:, hd].abs().contiguous()
                t = h * o.abs() + info.smallest_normal * h + A * (
                    (h * h if pair else h) + 2 * (D + 4) * u * S + 2 * (L + 8) * u)
            else:
                continue
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


def decode(c, q, scale, *, window=0, max_len=None, ws=None, out=None, table=None, lens=None):
    out = torch.full_like(q, math.nan) if out is None else out
    lens = c.lens if lens is None else lens
    most = max([len(k) for k, _ in c.keys] + [1]) if max_len is None else max_len
    ops.paged_decode_fwd(out, q, c.k, c.v, c.table if table is None else table, lens, most, scale,
                         workspace(q.shape[2]) if ws is None else ws, window)
    return out


def cross(c, q, q_lens, scale, *, max_len=None, max_q=None, ws=None, out=None, starts=None):
    out = torch.full_like(q, math.nan) if out is None else out
    most = max([len(k) for k, _ in c.keys] + [1]) if max_len is None else max_len
    ops.cross_attn_fwd(out, q, c.k, c.v, c.table, c.lens,
                       starts_of(q_lens) if starts is None else starts,
                       max(q_lens) if max_q is None else max_q, most, scale,
                       workspace(q.shape[2]) if ws is None else ws)
    return out


def queries(T, Hq, D, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(T, Hq, D, generator=gen, device=DEV).to(dtype)
