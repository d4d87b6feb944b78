"""rotary_embedding against its formula, its inverse and gradient, and its refusals."""

from __future__ import annotations

import math
from fractions import Fraction

import pytest
import torch

from pth_flash_attn import ops, rotary

needs_op = pytest.mark.skipif(not ops.is_available(), reason="op library not built")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0**-24
# Of a cosine or sine: the angle's 32 bits of a turn, its conversion and scaling
# (two roundings of at most pi / 4), the Taylor sums' remainder ((pi/4)^10 / 10!),
# three roundings of terms of at most 1.
TRIG = 2 * math.pi * 2.0**-33 + 2 * U * math.pi / 4 + 2.5e-8 + 3 * U
# Half a step of the type, relative to the value: 8, 11 and 24 significant bits.
ROUNDING = {t: torch.finfo(t).eps / 2 for t in (BF, HF, F32)}


def expected(x, angle, rot, interleaved, scale):
    """(result, tolerance) in 64 bits; ``angle`` [T, rot / 2]."""
    y = x.double().clone()
    half = rot // 2
    first = slice(0, rot, 2) if interleaved else slice(0, half)
    second = slice(1, rot, 2) if interleaved else slice(half, rot)
    a, b = y[..., first].clone(), y[..., second].clone()
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y[..., first], y[..., second] = scale * (a * cos - b * sin), scale * (b * cos + a * sin)
    tol = torch.zeros_like(y)
    # The factor times the scale, and the products: three roundings more.
    t = scale * (a.abs() + b.abs()) * (TRIG + 3 * U)
    tol[..., first] = tol[..., second] = t
    rounded = torch.zeros_like(y)
    rounded[..., :rot] = ROUNDING[x.dtype] * y[..., :rot].abs() + torch.finfo(x.dtype).smallest_normal * ROUNDING[x.dtype]
    return y, tol * (1 + ROUNDING[x.dtype]) + rounded


def angles_of(positions, turns):
    """Exactly, from the 64-bit fractions."""
    rows = [[2 * math.pi * (p * t % (1 << 64)) / 2.0**64 for t in turns.tolist()]
            for p in positions.tolist()]
    return torch.tensor(rows, dtype=torch.float64, device="cuda")


def fused(T, Hq, Hkv, D, dtype, seed, odd=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D + odd, generator=gen, device="cuda").to(dtype)
    return (qkv[:, odd : odd + Hq * D].view(T, Hq, D),
            qkv[:, odd + Hq * D : odd + (Hq + Hkv) * D].view(T, Hkv, D))


def close(got, x, angle, rot, interleaved, scale):
    want, tol = expected(x, angle, rot, interleaved, scale)
    excess = ((got.double() - want).abs() - tol).max().item()
    assert excess <= 0, f"{excess:.3g} beyond the tolerance"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize(("D", "rot", "Hq", "Hkv", "T", "odd"), [
    (128, 128, 8, 2, 5, 0), (64, 64, 3, 1, 1, 0), (256, 64, 4, 4, 33, 0), (128, 6, 2, 1, 7, 0),
    (80, 20, 2, 2, 9, 0), (192, 100, 1, 1, 3, 0), (64, 32, 5, 1, 17, 1), (2, 2, 1, 1, 4, 0),
    (1024, 1024, 1, 1, 2, 0), (63, 62, 2, 1, 5, 0), (128, 64, 4, 0, 3, 0), (128, 128, 0, 2, 3, 0),
    (128, 128, 2, 1, 5000, 0),
])
def test_formula(dtype, interleaved, D, rot, Hq, Hkv, T, odd):
    """Every type, layout and step width; the rest of the head copied bit for bit."""
    q, k = fused(T, Hq, Hkv, D, dtype, D + rot, odd)
    gen = torch.Generator().manual_seed(T)
    pos = torch.randint(0, 1 << 20, (T,), generator=gen)
    pos[0] = 0
    turns, scale = rotary.rotary_turns(rot, scaling="ramp", factor=8.0, base=500000.0)
    q_out, k_out = torch.full(q.shape, math.nan, dtype=dtype, device="cuda"), torch.full(k.shape, math.nan, dtype=dtype, device="cuda")
    ops.rotary_embedding(q_out, k_out, q, k, pos.cuda(), turns, interleaved, scale)
    some = torch.unique(torch.linspace(0, T - 1, 40).long())
    angle = angles_of(pos[some], turns)
    for out, x in ((q_out, q), (k_out, k)):
        if x.shape[1]:
            close(out[some.cuda()], x[some.cuda()], angle, rot, interleaved, scale)
            assert not out.isnan().any()
            assert torch.equal(out[..., rot:], x[..., rot:])


@pytest.mark.gpu
def test_positions_of_64_bits():
    """Angles are the wrapped product, for any position."""
    pos = torch.tensor([0, 1, -1, 1 << 31, (1 << 31) + 1, -(1 << 40) - 3, (1 << 62) + 12345,
                        (1 << 63) - 1, -(1 << 63)])
    turns, _ = rotary.rotary_turns(64)
    q, k = fused(len(pos), 2, 1, 64, F32, 3)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    ops.rotary_embedding(q_out, k_out, q, k, pos.cuda(), turns)
    close(q_out, q, angles_of(pos, turns), 64, False, 1.0)
    close(k_out, k, angles_of(pos, turns), 64, False, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_in_place_in_one_buffer(dtype):
    """Queries and keys of the fused projection where they lie; its values untouched."""
    T, Hq, Hkv, D = 70, 4, 2, 128
    gen = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=gen, device="cuda").to(dtype)
    was = qkv.clone()
    q = qkv[:, : Hq * D].view(T, Hq, D)
    k = qkv[:, Hq * D : (Hq + Hkv) * D].view(T, Hkv, D)
    turns, _ = rotary.rotary_turns(64)
    pos = torch.arange(T, device="cuda") + 1000
    q_out, k_out = torch.empty(T, Hq, D, dtype=dtype, device="cuda"), torch.empty(T, Hkv, D, dtype=dtype, device="cuda")
    ops.rotary_embedding(q_out, k_out, q, k, pos, turns, True)
    ops.rotary_embedding(q, k, q, k, pos, turns, True)
    assert torch.equal(q, q_out) and torch.equal(k, k_out)
    assert torch.equal(qkv[:, (Hq + Hkv) * D :], was[:, (Hq + Hkv) * D :])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    """``inverse`` with the same scale is the transpose: against the formula's
    gradient, and against differences of the op's own outputs (the op is linear, so
    that differences of size 1 have rounding alone)."""
    T, Hq, Hkv, D, rot = 6, 2, 1, 64, 32
    q, k = fused(T, Hq, Hkv, D, F32, 5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    dq, dk = (torch.randn(x.shape, generator=gen, device="cuda") for x in (q, k))
    turns, _ = rotary.rotary_turns(rot)
    pos = torch.randint(0, 100000, (T,), generator=torch.Generator().manual_seed(7))
    scale = 1.25
    gq, gk = torch.empty_like(dq), torch.empty_like(dk)
    ops.rotary_embedding(gq, gk, dq, dk, pos.cuda(), turns, interleaved, scale, inverse=True)
    angle = angles_of(pos, turns)
    close(gq, dq, -angle, rot, interleaved, scale)
    x = q.double().requires_grad_()
    half = rot // 2
    first = slice(0, rot, 2) if interleaved else slice(0, half)
    second = slice(1, rot, 2) if interleaved else slice(half, rot)
    cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., first], x[..., second]
    loss = (scale * (a * cos - b * sin) * dq[..., first].double()).sum() + \
        (scale * (b * cos + a * sin) * dq[..., second].double()).sum() + \
        (x[..., rot:] * dq[..., rot:].double()).sum()
    loss.backward()
    tol = 2 * scale * dq.abs().max().item() * (TRIG + 4 * U)
    assert (gq.double() - x.grad).abs().max().item() <= tol
    for t, h, j in ((0, 0, 0), (3, 1, 17), (5, 0, 40)):
        up = q.clone()
        up[t, h, j] += 1.0
        step = (up[t, h, j] - q[t, h, j]).double().item()
        outs = []
        for z in (up, q):
            o, e = torch.empty_like(z), torch.empty_like(k)
            ops.rotary_embedding(o, e, z, k, pos.cuda(), turns, interleaved, scale)
            outs.append(o.double())
        diff = ((outs[0] - outs[1]) * dq.double()).sum().item() / step
        bound = 4 * U * 2 * scale * (q[t, h].abs().max().item() + 1) * dq[t, h].abs().sum().item() + tol
        assert abs(diff - gq[t, h, j].item()) <= bound


@pytest.mark.gpu
def test_inverse_and_empty():
    q, k = fused(11, 2, 1, 64, F32, 9)
    turns, scale = rotary.rotary_turns(64, scaling="ramp", factor=4.0)
    pos = torch.arange(11, device="cuda") * 977
    a, b = torch.empty_like(q), torch.empty_like(k)
    ops.rotary_embedding(a, b, q, k, pos, turns, False, scale)
    ops.rotary_embedding(a, b, a, b, pos, turns, False, 1 / scale, True)
    bound = 4 * (TRIG + 4 * U) * q.abs().max().item()
    assert (a - q).abs().max().item() <= bound
    ops.rotary_embedding(a[:0], b[:0], q[:0], k[:0], pos[:0], turns)


PI = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")


@pytest.mark.parametrize(("scaling", "kw"), [
    ("none", {}), ("linear", {"factor": 4.0}), ("base", {"factor": 8.0}),
    ("ramp", {"factor": 16.0, "original_max_position": 8192}),
    ("smooth", {"factor": 8.0, "original_max_position": 8192}),
    ("factors", {"factors": [1.0 + j for j in range(32)], "factor": 2.0}),
])
def test_frequencies(scaling, kw):
    """The 64-bit fractions are the frequencies over 2 pi to the double's rounding
    and that of the fraction; the scalings at their two ends."""
    f = rotary.rotary_frequencies(64, scaling=scaling, **kw)
    turns, scale = rotary.rotary_turns(64, scaling=scaling, device="cpu", **kw)
    plain = [10000.0 ** (-2 * j / 64) for j in range(32)]
    for x, t in zip(f, turns.tolist()):
        want = Fraction(x) / (2 * PI)
        got = Fraction(t % (1 << 64), 1 << 64)
        # 2 pi and the quotient as doubles, the fraction's last bit.
        assert abs(got - want) <= want * Fraction(3, 1 << 53) + Fraction(1, 1 << 65)
    ends = {"none": (1, 1), "linear": (4, 4), "base": (1, 8), "ramp": (1, 16), "smooth": (1, 8),
            "factors": (1, 32)}[scaling]
    assert f[0] == pytest.approx(plain[0] / ends[0], rel=1e-12)
    assert f[-1] == pytest.approx(plain[-1] / ends[1], rel=1e-12)
    assert scale == pytest.approx({"ramp": 0.1 * math.log(16) + 1,
                                   "factors": math.sqrt(1 + math.log(2) / math.log(4096))}.get(scaling, 1.0))


@pytest.mark.parametrize(("args", "kw"), [
    ((63,), {}), ((0,), {}), ((64,), {"scaling": "other"}), ((64,), {"base": 0.0}),
    ((64,), {"factor": math.inf}), ((64,), {"scaling": "factors", "factors": [1.0]}),
    ((2,), {"scaling": "base"}), ((64,), {"scaling": "smooth", "low_freq_factor": 5.0}),
    ((64,), {"scaling": "ramp", "slow_turns": 0.0}), ((64,), {"original_max_position": 0}),
])
def test_frequencies_refused(args, kw):
    with pytest.raises(ValueError):
        rotary.rotary_turns(*args, device="cpu", **kw)


def _cpu():
    q, k = torch.zeros(4, 2, 64, dtype=BF), torch.zeros(4, 1, 64, dtype=BF)
    return dict(q_out=q.clone(), k_out=k.clone(), q=q, k=k,
                positions=torch.zeros(4, dtype=torch.int64), turns=torch.zeros(32, dtype=torch.int64))


REFUSALS = [
    (lambda a: {}, "computes on CUDA tensors only"),
    (lambda a: dict(q=a["q"][0]), "must be 3-D"),
    (lambda a: dict(k=a["k"][:3]), "same T and D"),
    (lambda a: dict(q=torch.zeros(4, 2, 1, dtype=BF), k=torch.zeros(4, 1, 1, dtype=BF)), "head size"),
    (lambda a: dict(q=a["q"].double(), k=a["k"].double()), "must both be float32"),
    (lambda a: dict(k=a["k"].half()), "must both be float32"),
    (lambda a: dict(q_out=a["q_out"].float()), "shapes and dtype"),
    (lambda a: dict(k_out=a["k_out"][:, :, :32]), "shapes and dtype"),
    (lambda a: dict(q=torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)), "stride 1"),
    (lambda a: dict(positions=a["positions"].int()), "positions must be"),
    (lambda a: dict(positions=a["positions"][:3]), "positions must be"),
    (lambda a: dict(turns=torch.zeros(33, dtype=torch.int64)), "turns must be"),
    (lambda a: dict(turns=torch.zeros(0, dtype=torch.int64)), "turns must be"),
    (lambda a: dict(turns=torch.zeros(32)), "turns must be"),
    (lambda a: dict(scale=math.nan), "scale must be finite"),
    (lambda a: dict(q_out=a["q_out"][:1].expand_as(a["q_out"])), "overlap themselves"),
]


@needs_op
@pytest.mark.parametrize(("change", "message"), REFUSALS)
def test_refusals(change, message):
    args = _cpu()
    args.update(change(args))
    with pytest.raises(RuntimeError, match=message):
        ops.rotary_embedding(**args)
    if "CUDA" not in message:
        with pytest.raises(RuntimeError, match=message):
            ops.ops8.rotary_embedding_fake(**args)


@needs_op
def test_shared_memory_refused():
    """Outputs that share memory with another tensor than their own input's view."""
    buf = torch.zeros(4, 6 * 64, dtype=BF)
    a = _cpu()
    q, k = buf[:, :128].view(4, 2, 64), buf[:, 128:192].view(4, 1, 64)
    for bad in (dict(q=q, k=k, q_out=buf[:, 64:192].view(4, 2, 64), k_out=buf[:, 192:256].view(4, 1, 64)),
                dict(q=q, k=k, q_out=buf[:, 8:136].view(4, 2, 64)),
                dict(q_out=q, k_out=buf[:, 64:128].view(4, 1, 64))):
        with pytest.raises(RuntimeError, match="share no memory|share memory with one"):
            ops.rotary_embedding(**{**a, **bad})
    ids = torch.zeros(4 * 64, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="must not overlap positions"):
        ops.rotary_embedding(**{**a, "positions": ids[:4], "k_out": ids.view(BF)[:256].view(4, 1, 64)})
