"""Rotary positions with several axes, differential attention and AdamW over many tensors against plain 64-bit forms.

Tolerances are bounds, element by element.  A rounding to a type is off by at most half a step, eps / 2 of the value (fp16 also by 2^-25, half its
smallest step).  What is rounded on the way is the P and dS of the matrix products' operands, the maps' own outputs that D = dO . O_m is made of, and
the result; everything else is fp32: its errors are taken as 2^-22 of the absolute sums, times 1 + the largest score for the exponents."""
import copy
import math

import pytest
import torch

import hsenet_amd as H
from hsenet_amd import _lib as L
from hsenet_amd import _ops as O

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP = 2.0 ** -22


def half(dt):
    return torch.finfo(dt).eps / 2


def floor(dt):
    return 2.0 ** -25 if dt == F16 else 0.0


def within(got, ref, tol, what=""):
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs() / tol.clamp(min=1e-300)).nan_to_num(1e9).max():.3g} of the bound"


def rnd(g, *shape, dtype=F32, scale=1.0, dev="cuda"):
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


# ---- rotary ------------------------------------------------------------------------------------------------------------------
def turned(x, pos, plan, sign=1.0):
    """(value, bound) of the turn in 64 bits; pos [axes, B, N]"""
    y, P = x.double().clone(), plan.pairs
    ang = (pos.double()[plan.axis.long()].movedim(0, -1) * plan.freq)[:, :, None]
    lo, hi = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if plan.interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = y[..., lo].clone(), y[..., hi].clone()
    y[..., lo], y[..., hi] = a * ang.cos() - sign * b * ang.sin(), sign * a * ang.sin() + b * ang.cos()
    tol = half(x.dtype) * y.abs() + floor(x.dtype)
    size = (a.abs() + b.abs()) * 2.0 ** -20               # 3 products and a sum, cos and sin of a fraction of a turn held to 2^-25
    tol[..., lo] += size
    tol[..., hi] += size
    if x.shape[-1] > 2 * P:
        tol[..., 2 * P:] = 0
    return y, tol


@pytest.mark.parametrize("B,N,Hq,Hk,dh,sections,inter,dtype,pos", [
    (1, 1, 1, 0, 2, (1,), False, F32, "i32"), (2, 5, 3, 1, 64, (8, 12, 12), False, BF, "i32"), (2, 65, 12, 12, 64, (10, 11, 11), True, BF, "i64"),
    (3, 33, 4, 2, 80, (8, 13, 15), True, F32, "f32"), (1, 130, 2, 2, 33, (3, 0, 4), False, F16, "i32"), (1, 7, 2, 1, 33, (5, 11), True, F16, "i32"),
    (2, 9, 5, 2, 96, (20, 13), False, F16, "i32"), (1, 4099, 3, 1, 128, (16, 24, 24), False, BF, "i32"), (4, 17, 2, 2, 34, (4, 9, 4), False, BF, "f32"),
    (1, 4100, 12, 12, 64, (7, 11, 11), False, BF, "i32"), (2, 31, 3, 2, 80, (9, 13, 9), False, F32, "f32"), (1, 6, 1, 0, 4096, (100, 203), False, F16, "i64"),
    (1, 4100, 5, 3, 64, (7, 11, 11), True, BF, "i32"), (2, 31, 3, 1, 72, (9, 13, 9), True, F32, "f32"), (1, 9, 2, 1, 2080, (1,), False, F32, "i32"),
    (2, 5, 40, 8, 8, (1, 1, 1), False, BF, "i32"), (2, 5, 40, 8, 8, (1, 1, 1), True, F16, "i32")])
def test_rotary_values_and_gradient(dev, B, N, Hq, Hk, dh, sections, inter, dtype, pos):
    g = torch.Generator("cuda").manual_seed(B * 1000 + N)
    plan = H.RotaryAxes(sections, theta=5000.0, ladder="shared" if N % 2 else "per_axis", interleaved=inter)
    qkv = rnd(g, B, N, Hq + Hk + 1, dh, dtype=dtype)
    q, k = qkv[:, :, :Hq].requires_grad_(), (qkv[:, :, Hq:Hq + Hk].requires_grad_() if Hk else None)
    p = torch.randint(-300, 1_000_000, (len(sections), B, N), generator=g, device="cuda")
    p = p.float() / 8 if pos == "f32" else p.to(torch.int32) if pos == "i32" else p
    out = H.rotary_axes(q, k, p, plan)
    outs, ins = ((out,), (q,)) if k is None else (out, (q, k))
    ups = [rnd(g, *o.shape, dtype=dtype) for o in outs]
    grads = torch.autograd.grad(outs, ins, ups)
    for x, y, u, d in zip(ins, outs, ups, grads):
        within(y.detach(), *turned(x.detach(), p, plan), "turn")
        within(d, *turned(u, p, plan, -1.0), "gradient")
    # in place, and one set of positions for all entries
    same = H.rotary_axes(q.detach(), None, p[:, 0], plan)
    z = qkv.clone()
    with torch.no_grad():
        back = H.rotary_axes(z[:, :, :Hq], z[:, :, Hq:Hq + Hk] if Hk else None, p, plan, inplace=True)
    assert torch.equal(z[:, :, :Hq], outs[0]) and torch.equal(z[:, :, Hq + Hk:], qkv[:, :, Hq + Hk:])
    assert (back if k is None else back[0]).data_ptr() == z.data_ptr()
    within(same, *turned(q.detach(), p[:, :1].expand_as(p), plan), "shared positions")


def test_rotary_unaligned_transposed_and_empty(dev):
    g = torch.Generator("cuda").manual_seed(3)
    plan = H.RotaryAxes((4, 6, 6))
    pos = torch.randint(0, 99, (3, 2, 6), generator=g, device="cuda", dtype=torch.int32)
    flat = rnd(g, 2 * 6 * 3 * 32 + 1, dtype=BF)
    for x in (flat[1:].view(2, 6, 3, 32), rnd(g, 2, 3, 6, 32, dtype=BF).transpose(1, 2), rnd(g, 32, 2, 6, 3, dtype=BF).permute(1, 2, 3, 0),
              rnd(g, 2, 6, 1, 32, dtype=BF).expand(2, 6, 3, 32)):
        within(H.rotary_axes(x, None, pos, plan), *turned(x, pos, plan))
    q = rnd(g, 2, 6, 3, 32, dtype=BF)
    a, b = H.rotary_axes(q, q[:, :, :0], pos, plan)
    assert b.shape == (2, 6, 0, 32) and torch.equal(a, H.rotary_axes(q, None, pos, plan))
    a, b = H.rotary_axes(q[:, :, :0], q, pos, plan)
    assert a.numel() == 0 and torch.equal(b, H.rotary_axes(q, None, pos, plan))
    assert H.rotary_axes(q[:, :0], None, pos[:, :, :0], plan).shape == (2, 0, 3, 32)


def test_rotary_refusals(dev):
    plan, q = H.RotaryAxes((4, 6, 6)), torch.zeros(2, 6, 3, 32, dtype=BF, device="cuda")
    pos = torch.zeros(3, 2, 6, dtype=torch.int32, device="cuda")
    for args in ((q, q.half(), pos, plan), (q, q[:, :5], pos, plan), (q, q[..., :16], pos, plan), (q[..., :16], None, pos, plan),
                 (q.double(), None, pos, plan), (q, None, pos.short(), plan), (q, None, pos[:2], plan), (q, None, pos[:, :1], plan), (q[0], None, pos, plan),
                 (q, None, pos.cpu(), plan), (q, None, pos, H.RotaryAxes((4, 6, 6), device="cpu")), (q, None, pos, None)):
        with pytest.raises(L.HsError):
            H.rotary_axes(*args)
    with pytest.raises(L.HsError, match="not differentiable"):
        H.rotary_axes(q.requires_grad_(), None, pos, plan, inplace=True)
    with pytest.raises(L.HsError, match="twice"), torch.no_grad():
        H.rotary_axes(q, q, pos, plan, inplace=True)
    with pytest.raises(L.HsError, match="broadcast"):
        H.rotary_axes(q.detach()[:, :, :1].expand(2, 6, 3, 32), None, pos, plan, inplace=True)


def test_rotary_in_place_refuses_overlaps(dev):
    plan, pos = H.RotaryAxes((4, 6, 6)), torch.zeros(3, 2, 6, dtype=torch.int32, device="cuda")
    x = torch.zeros(2, 6, 8, 32, dtype=BF, device="cuda")
    own = torch.zeros(999, dtype=BF, device="cuda").as_strided((2, 6, 3, 32), (300, 32, 32, 1))
    with torch.no_grad():
        for q, k in ((x[:, :, :4], x[:, :, 3:]), (x[:, :, 3:], x[:, :, :4]), (own, None)):
            with pytest.raises(L.HsError, match="overlap"):
                H.rotary_axes(q, k, pos, plan, inplace=True)
        H.rotary_axes(x[:, :, 0::2], x[:, :, 1::2], pos, plan, inplace=True)
        H.rotary_axes(x[:, :, 0::2], x[:, :, 0:0], pos, plan, inplace=True)


# ---- differential attention ----------------------------------------------------------------------------------------------------
def diff_reference(q, k, v, lam, go, scale, causal, start, lens):
    """values and bounds {o, q, k, v, lam: (value, bound)} in 64 bits"""
    dt, h = q.dtype, half(q.dtype)
    B, Nq, H2, d = q.shape
    Nk, Hkv, Hq = k.shape[1], v.shape[2], H2 // 2
    G = Hq // Hkv
    Q, K, V, GO = (t.detach().double() for t in (q, k, v, go))
    lamv = lam.detach().double().reshape(-1).expand(Hq) if lam.numel() == 1 else lam.detach().double()
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    r = {"o": z(B, Nq, Hq, 2 * d), "q": z(*q.shape), "k": z(*k.shape), "v": z(*v.shape), "lam": z(Hq)}
    t = {n: torch.zeros_like(x) for n, x in r.items()}
    j = torch.arange(Nk, device=q.device)
    up = 16.0 if dt == F16 else 1.0
    fP, fB = (2.0 ** -24, 2.0 ** -25 / up) if dt == F16 else (0.0, 0.0)       # P to its map's largest, P and dS of the backward pass
    for b in range(B):
        n = Nk if lens is None else int(lens[b])
        seen = (j < n)[None].expand(Nq, Nk)
        if causal:
            seen = seen & (j[None] <= int(start[b]) + torch.arange(Nq, device=q.device)[:, None])
        kb, vb = K[b].clone(), V[b].clone()
        kb[n:], vb[n:] = 0, 0
        for hq in range(Hq):
            g = hq // G
            Vh, Gh, lm = vb[:, g], GO[b, :, hq], lamv[hq]
            dP, dPa = Gh @ Vh.T, Gh.abs() @ Vh.abs().T
            o_tol, pc, pc_tol = 0, 0, 0
            for m, w in ((0, 1.0), (1, -lm)):
                Km, Qm = kb[:, 2 * g + m], Q[b, :, 2 * hq + m]
                S = (Qm @ Km.T) * scale
                noise = FP * (1 + ((Qm.abs() @ Km.abs().T) * scale).masked_fill(~seen, 0).max())
                p = torch.softmax(S.masked_fill(~seen, -math.inf), -1).nan_to_num(0.0)
                pv_tol = (p * (h + noise)) @ Vh.abs() + fP * (seen.double() @ Vh.abs())
                o = p @ Vh
                r["o"][b, :, hq] += w * o
                o_tol = o_tol + abs(w) * pv_tol
                pc, pc_tol = pc + w * p, pc_tol + abs(w) * noise * p
                D = (p * dP).sum(-1, keepdim=True)
                eD = (Gh.abs() * (h * o.abs() * 1.01 + pv_tol + floor(dt))).sum(-1, keepdim=True) + FP * (Gh.abs() * o.abs()).sum(-1, keepdim=True)
                dS = w * p * (dP - D)
                dS_tol = abs(w) * p * (noise * ((dP - D).abs() + dPa) + eD) * (1 + h) + (h + noise) * dS.abs() + fB * seen * max(1.0, float(abs(w)))
                r["q"][b, :, 2 * hq + m] = scale * dS @ Km
                t["q"][b, :, 2 * hq + m] = scale * dS_tol @ Km.abs()
                r["k"][b, :, 2 * g + m] += scale * dS.T @ Qm
                t["k"][b, :, 2 * g + m] += scale * dS_tol.T @ Qm.abs()
                if m:
                    r["lam"][hq] -= D.sum()
                    t["lam"][hq] += (2 * noise * p * dPa).sum() + FP * D.abs().sum()
            t["o"][b, :, hq] = o_tol
            r["v"][b, :, g] += pc.T @ Gh
            t["v"][b, :, g] += (pc_tol + h * pc.abs() + fB).T @ Gh.abs()
    if lam.numel() == 1:
        r["lam"], t["lam"] = r["lam"].sum().view(lam.shape), t["lam"].sum().view(lam.shape)
    for n in r:
        if n == "lam":
            t[n] = t[n] + 2.0 ** -23 * r[n].abs()
        else:
            t[n] = (t[n] + FP * r[n].abs()) * (1 + h) + h * r[n].abs() + floor(dt)
    return {n: (r[n], t[n] * 1.01 + 1e-30) for n in r}


def diff_case(seed, B, Nq, Nk, Hq, Hkv, d, dtype, causal=False, lens=None, start=None, lam="heads", scale=None, size=1.0, grow=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    q, k = rnd(g, B, Nq, 2 * Hq, d, dtype=dtype, scale=size), rnd(g, B, Nk, 2 * Hkv, d, dtype=dtype)
    v, go = rnd(g, B, Nk, Hkv, 2 * d, dtype=dtype), rnd(g, B, Nq, Hq, 2 * d, dtype=dtype)
    lm = torch.rand(Hq, generator=g, device="cuda") * 1.4 - 0.2 if lam == "heads" else torch.full((1,) if lam == "one" else (), 0.4, device="cuda")
    k[:, Nk // 2:] *= grow                                  # scores that leave the first ones far behind
    it = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    starts = start if start is not None else [Nk - Nq] * B
    ref = diff_reference(q, k, v, lm, go, d ** -0.5 if scale is None else scale, causal, starts, lens)
    return q, k, v, lm, go, dict(causal=causal, scale=scale, q_start=it(start), kv_len=it(lens)), ref


def run_diff(q, k, v, lam, go, kw):
    ins = [x.detach().clone().requires_grad_() if x.is_contiguous() else x.detach().requires_grad_() for x in (q, k, v, lam)]
    o = H.diff_attention(*ins, **kw)
    grads = torch.autograd.grad(o, ins, go)
    return dict(zip(("o", "q", "k", "v", "lam"), (o.detach(), *grads)))


@pytest.mark.parametrize("case", [
    dict(B=1, Nq=1, Nk=1, Hq=1, Hkv=1, d=64, dtype=BF), dict(B=2, Nq=3, Nk=33, Hq=2, Hkv=1, d=32, dtype=F16, lam="one"),
    dict(B=1, Nq=64, Nk=64, Hq=2, Hkv=2, d=64, dtype=BF, causal=True), dict(B=2, Nq=65, Nk=63, Hq=2, Hkv=1, d=64, dtype=F16, causal=True),
    dict(B=1, Nq=257, Nk=257, Hq=3, Hkv=3, d=64, dtype=BF, lam="none"), dict(B=1, Nq=130, Nk=300, Hq=2, Hkv=2, d=128, dtype=BF, causal=True),
    dict(B=3, Nq=97, Nk=97, Hq=4, Hkv=1, d=32, dtype=BF, causal=True, lens=[0, 50, 97], start=[0, 0, 0]),
    dict(B=3, Nq=40, Nk=200, Hq=2, Hkv=2, d=128, dtype=F16, lens=[0, 1, 200]), dict(B=2, Nq=300, Nk=129, Hq=2, Hkv=1, d=64, dtype=BF, causal=True, start=[-40, 100]),
    dict(B=1, Nq=129, Nk=577, Hq=1, Hkv=1, d=64, dtype=F16, scale=0.3), dict(B=1, Nq=70, Nk=190, Hq=2, Hkv=1, d=64, dtype=BF, size=12.0),
    dict(B=1, Nq=33, Nk=64, Hq=8, Hkv=2, d=128, dtype=BF), dict(B=2, Nq=1025, Nk=1025, Hq=1, Hkv=1, d=32, dtype=BF, causal=True),
    dict(B=1, Nq=300, Nk=200, Hq=1, Hkv=1, d=64, dtype=BF, grow=36.0), dict(B=1, Nq=70, Nk=333, Hq=2, Hkv=1, d=32, dtype=F16, grow=36.0),
    dict(B=1, Nq=140, Nk=150, Hq=1, Hkv=1, d=128, dtype=F16, grow=20.0, causal=True), dict(B=1, Nq=5, Nk=3000, Hq=1, Hkv=1, d=64, dtype=F16, grow=36.0),
    # few queries: the keys are cut and joined
    dict(B=2, Nq=1, Nk=255, Hq=4, Hkv=2, d=64, dtype=BF, causal=True), dict(B=2, Nq=1, Nk=257, Hq=8, Hkv=1, d=64, dtype=F16, lens=[256, 257]),
    dict(B=3, Nq=1, Nk=5000, Hq=4, Hkv=2, d=64, dtype=BF, lens=[0, 1, 4999], causal=True, start=[5, 0, 4998]),
    dict(B=1, Nq=7, Nk=3001, Hq=8, Hkv=2, d=128, dtype=F16, causal=True), dict(B=2, Nq=13, Nk=1300, Hq=2, Hkv=1, d=32, dtype=BF, causal=True, start=[600, 1]),
    dict(B=1, Nq=2, Nk=20000, Hq=2, Hkv=2, d=128, dtype=BF, size=4.0), dict(B=1, Nq=31, Nk=700, Hq=1, Hkv=1, d=64, dtype=BF, causal=True, start=[-10])],
    ids=lambda c: f"{c['B']}x{c['Nq']}x{c['Nk']}-{c['Hq']}/{c['Hkv']}x{c['d']}")
def test_diff_attention_values_and_gradients(dev, case):
    *ins, kw, ref = diff_case(case["Nq"] * 7 + case["Nk"], **case)
    got = run_diff(*ins, kw)
    for n, (value, bound) in ref.items():
        within(got[n], value, bound, n)
    with torch.no_grad():
        assert torch.equal(H.diff_attention(*ins[:4], **kw), got["o"])       # without a graph: the same bits
    again = run_diff(*ins, kw)
    assert all(torch.equal(got[n], again[n]) for n in got)                    # no atomics


@pytest.mark.parametrize("case", [                             # so many rows that the keys are not cut
    dict(B=4, Nq=65, Nk=63, Hq=32, Hkv=32, d=64, dtype=F16, causal=True), dict(B=1, Nq=257, Nk=257, Hq=32, Hkv=32, d=64, dtype=BF, causal=True),
    dict(B=1, Nq=1025, Nk=1030, Hq=8, Hkv=8, d=32, dtype=BF, causal=True), dict(B=1, Nq=130, Nk=300, Hq=32, Hkv=32, d=128, dtype=BF, causal=True),
    dict(B=3, Nq=40, Nk=200, Hq=32, Hkv=32, d=128, dtype=F16, lens=[0, 1, 200], lam="one"),
    dict(B=3, Nq=97, Nk=97, Hq=32, Hkv=8, d=32, dtype=BF, causal=True, lens=[0, 50, 97], start=[0, -20, 3]),
    dict(B=2, Nq=300, Nk=129, Hq=32, Hkv=16, d=64, dtype=BF, causal=True, start=[-40, 100], lam="none"),
    dict(B=1, Nq=300, Nk=200, Hq=32, Hkv=32, d=64, dtype=BF, grow=36.0), dict(B=4, Nq=70, Nk=333, Hq=32, Hkv=32, d=32, dtype=F16, grow=36.0),
    dict(B=1, Nq=140, Nk=150, Hq=32, Hkv=32, d=128, dtype=F16, grow=20.0, causal=True), dict(B=2, Nq=300, Nk=190, Hq=16, Hkv=16, d=64, dtype=BF, size=12.0),
    dict(B=70, Nq=70, Nk=31, Hq=2, Hkv=2, d=64, dtype=F16, scale=0.3), dict(B=2, Nq=130, Nk=300, Hq=32, Hkv=32, d=128, dtype=BF, causal=True),
    dict(B=6, Nq=40, Nk=200, Hq=32, Hkv=32, d=128, dtype=F16, lens=[0, 1, 200, 31, 32, 33], lam="one"),
    dict(B=2, Nq=140, Nk=150, Hq=32, Hkv=32, d=128, dtype=F16, grow=20.0, causal=True), dict(B=2, Nq=129, Nk=161, Hq=32, Hkv=32, d=128, dtype=BF, grow=36.0),
    dict(B=5, Nq=100, Nk=70, Hq=32, Hkv=16, d=128, dtype=BF, causal=True, lens=[70, 64, 0, 1, 65], start=[-30, -99, 0, 5, -40], lam="none"),
    dict(B=8, Nq=65, Nk=100, Hq=32, Hkv=32, d=64, dtype=F16, causal=True), dict(B=4, Nq=130, Nk=97, Hq=32, Hkv=32, d=64, dtype=BF, causal=True),
    dict(B=12, Nq=97, Nk=97, Hq=32, Hkv=8, d=32, dtype=BF, causal=True, lens=[0, 50, 97] * 4, start=[0, -20, 3] * 4),
    dict(B=4, Nq=130, Nk=300, Hq=32, Hkv=32, d=128, dtype=BF, causal=True), dict(B=4, Nq=129, Nk=161, Hq=32, Hkv=32, d=128, dtype=BF, grow=36.0),
    dict(B=8, Nq=40, Nk=200, Hq=32, Hkv=32, d=128, dtype=F16, lens=[0, 1, 200, 31, 32, 33, 199, 64], lam="one"),
    dict(B=4, Nq=140, Nk=150, Hq=32, Hkv=32, d=128, dtype=F16, grow=20.0, causal=True)],
    ids=lambda c: f"{c['B']}x{c['Nq']}x{c['Nk']}-{c['Hq']}/{c['Hkv']}x{c['d']}")
def test_diff_attention_of_many_rows(dev, case):
    test_diff_attention_values_and_gradients(dev, case)


@pytest.mark.parametrize("case", [                             # many rows of few heads: the whole forward's keys come in parts
    dict(B=1, Nq=600, Nk=2000, Hq=16, Hkv=16, d=64, dtype=BF, causal=True), dict(B=2, Nq=520, Nk=2047, Hq=8, Hkv=4, d=64, dtype=F16, grow=36.0),
    dict(B=2, Nq=600, Nk=1500, Hq=10, Hkv=10, d=32, dtype=BF, lens=[33, 1499], lam="one"), dict(B=1, Nq=1300, Nk=1300, Hq=8, Hkv=8, d=64, dtype=BF, causal=True),
    dict(B=3, Nq=700, Nk=1100, Hq=6, Hkv=6, d=32, dtype=F16, causal=True, lens=[0, 1100, 64], start=[0, -650, 30]),
    dict(B=1, Nq=300, Nk=1500, Hq=4, Hkv=2, d=128, dtype=F16, causal=True), dict(B=2, Nq=70, Nk=1000, Hq=2, Hkv=2, d=128, dtype=BF, lens=[1000, 40])],
    ids=lambda c: f"{c['B']}x{c['Nq']}x{c['Nk']}-{c['Hq']}/{c['Hkv']}x{c['d']}")
def test_diff_attention_of_few_heads(dev, case):
    test_diff_attention_values_and_gradients(dev, case)


@pytest.mark.parametrize("case", [                             # many queries for each key: the gradients of keys and values come in parts
    dict(B=1, Nq=300, Nk=260, Hq=8, Hkv=1, d=64, dtype=BF, causal=True), dict(B=2, Nq=290, Nk=140, Hq=6, Hkv=1, d=128, dtype=F16, lens=[0, 139]),
    dict(B=2, Nq=200, Nk=300, Hq=6, Hkv=2, d=64, dtype=F16, causal=True, start=[-150, 90]), dict(B=1, Nq=900, Nk=1, Hq=2, Hkv=1, d=32, dtype=BF, lam="one"),
    dict(B=3, Nq=500, Nk=33, Hq=4, Hkv=2, d=128, dtype=BF, causal=True, lens=[1, 33, 20], start=[-499, -300, 0])],
    ids=lambda c: f"{c['B']}x{c['Nq']}x{c['Nk']}-{c['Hq']}/{c['Hkv']}x{c['d']}")
def test_diff_attention_of_few_keys(dev, case):
    test_diff_attention_values_and_gradients(dev, case)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("Nq", [1, 200])
@pytest.mark.parametrize("B", [2, 64])
def test_diff_one_visible_key_gives_its_value(dev, d, Nq, B):
    """softmax of one key is 1, and of two equal keys a half, whatever the scores: no rounding of P may show"""
    g = torch.Generator("cuda").manual_seed(d + Nq)
    q, k, v = rnd(g, B, Nq, 4, d, dtype=BF), rnd(g, B, 300, 4, d, dtype=BF), rnd(g, B, 300, 2, 2 * d, dtype=BF)
    k[1::2, 1], v[1::2, 1] = k[1::2, 0], v[1::2, 0]
    o = H.diff_attention(q, k, v, torch.tensor([0.5, 0.0], device="cuda"), kv_len=torch.tensor([1, 2] * (B // 2), dtype=torch.int32, device="cuda"))
    assert torch.equal(o[:, :, 0], (0.5 * v[:, :1, 0]).expand_as(o[:, :, 0])) and torch.equal(o[:, :, 1], v[:, :1, 1].expand_as(o[:, :, 1]))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("Nk", [2, 2000])
@pytest.mark.parametrize("weight,size", [(0.5, 4000.0), (-3.0, 1300.0)])
def test_diff_fp16_gradients_up_to_their_limit(dev, d, Nk, weight, size):
    """|P (dP - D)| max(1, |lam|) just under 4094, where two equal scores of -0.04 powers of two make a row's sum 1.94 times its power of two: dq, dk
    and dlam are as far from their 64-bit values as roundings are, and finite"""
    B, Nq, Hq = 1, 40, 2
    q, k = torch.zeros(B, Nq, 2 * Hq, d, dtype=F16, device="cuda"), torch.full((B, Nk, 2 * Hq, d), math.nan, dtype=F16, device="cuda")
    v, go = torch.full((B, Nk, Hq, 2 * d), math.nan, dtype=F16, device="cuda"), torch.full((B, Nq, Hq, 2 * d), 50.0, dtype=F16, device="cuda")
    q[..., 0], k[:, :2] = 0.125, 0.0                       # (dk, 40 queries' sum of dS q, is 20000 at most: fp16 ends at 65504)
    k[:, :2, :, 0] = -0.2216
    for j, side in enumerate((1.0, -1.0)):
        k[:, j, :, 1], v[:, j] = side / 16, side * size / (50.0 * d)
    lam, lens = torch.full((Hq,), weight, device="cuda"), None if Nk == 2 else [2]
    got = run_diff(q, k, v, lam, go, dict(scale=1.0, kv_len=None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")))
    for n, (value, bound) in diff_reference(q, k[:, :2], v[:, :2], lam, go, 1.0, False, [0], None).items():
        within(got[n][:, :2] if n in "kv" else got[n], value, bound, n)
    assert float(got["q"][..., 0::2, 1].abs().max()) > size / 16


def test_diff_gradient_against_differences(dev):
    """<gradient, u> against the difference of two runs' losses along u.  The loss is taken of 64-bit references, so that only the formula is in question."""
    q, k, v, lam, go, kw, ref = diff_case(5, 1, 19, 23, 2, 1, 32, F16, causal=True)
    got = run_diff(q, k, v, lam, go, kw)
    g = torch.Generator("cuda").manual_seed(6)
    def loss(q, k, v, lam):
        S = [torch.einsum("bihd,bjd->bhij", q[:, :, m::2], k[:, :, m]) * 32 ** -0.5 for m in (0, 1)]
        hide = torch.arange(23, device="cuda")[None] > 4 + torch.arange(19, device="cuda")[:, None]
        p = [torch.softmax(s.masked_fill(hide, -math.inf), -1) for s in S]
        return ((torch.einsum("bhij,bjc->bihc", p[0] - lam[:, None, None] * p[1], v[:, :, 0])) * go.double()).sum()
    x = [t.double() for t in (q, k, v, lam)]
    for i, n in enumerate(("q", "k", "v", "lam")):
        u = torch.randn(x[i].shape, generator=g, device="cuda", dtype=torch.float64)
        e = 1e-5
        up, down = ([t + s * e * u if a == i else t for a, t in enumerate(x)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * e)
        # central differences: e^2 of the third derivative and 2^-52 |loss| / e, both far below the gradient's own bound
        assert abs(float((got[n].double() * u).sum() - slope)) <= float((ref[n][1] * u.abs()).sum()) + 1e-5


def test_diff_caches_views_and_what_lies_behind(dev):
    """strided operands (thirds of a projection, a cache longer than its tokens), an unaligned one, and NaN in every place that does not count"""
    g = torch.Generator("cuda").manual_seed(11)
    B, N, Hq, d, S = 2, 37, 2, 64, 50
    proj = rnd(g, B, N, 3 * 2 * Hq * d, dtype=BF)
    q, k = (t.view(B, N, 2 * Hq, d) for t in proj.chunk(3, -1)[:2])
    v = proj.chunk(3, -1)[2].view(B, N, Hq, 2 * d)
    lam, go = torch.full((Hq,), 0.3, device="cuda"), rnd(g, B, Hq, N, 2 * d, dtype=BF).transpose(1, 2)
    lens = torch.tensor([20, 37], dtype=torch.int32, device="cuda")
    want = run_diff(q.contiguous(), k.contiguous(), v.contiguous(), lam, go.contiguous(), dict(kv_len=lens))
    ck, cv = (torch.full((B, S, h, w), math.nan, dtype=BF, device="cuda") for h, w in ((2 * Hq, d), (Hq, 2 * d)))
    for b, n in enumerate(lens.tolist()):
        ck[b, :n], cv[b, :n] = k[b, :n], v[b, :n]
    odd = torch.empty(q.numel() + 1, dtype=BF, device="cuda")[1:].view(q.shape).copy_(q)
    for a, b, c in ((q, k, v), (odd, k, v), (q, ck, cv), (q.transpose(1, 2).contiguous().transpose(1, 2), k, v)):
        got = run_diff(a, b, c, lam, go, dict(kv_len=lens))
        for n in want:
            x = got[n][:, :N] if n in "kv" else got[n]
            assert torch.equal(x, want[n]), n
            if n in "kv":
                assert all(not got[n][i, m:].any() for i, m in enumerate(lens.tolist()))
    with torch.no_grad():
        one = H.diff_attention(q[:, :1], ck, cv, lam, kv_len=lens)
        assert torch.isfinite(one).all() and torch.equal(one, H.diff_attention(q[:, :1], k, v, lam, kv_len=lens))
        over = H.diff_attention(q, k, v, lam, kv_len=torch.tensor([-5, 1000], dtype=torch.int32, device="cuda"))
        assert not over[0].any() and torch.equal(over[1], H.diff_attention(q, k, v, lam)[1])
        assert H.diff_attention(q[:, :0], k, v, lam).shape == (B, 0, Hq, 2 * d) and not H.diff_attention(q, k[:, :0], v[:, :0], lam).any()


@pytest.mark.parametrize("B,Nq,Hq,Hkv,d", [(2, 1, 4, 2, 64), (2, 5, 8, 2, 128), (3, 40, 2, 2, 32), (8, 70, 16, 16, 64), (4, 100, 16, 16, 128), (8, 100, 16, 16, 128), (16, 100, 16, 16, 128)])
def test_diff_causal_cache_filled_to_its_queries(dev, B, Nq, Hq, Hkv, d):
    """a cache that holds NaN behind the last query's own position: the causal mask alone says that nothing there counts"""
    g = torch.Generator("cuda").manual_seed(Nq)
    S = Nq + 90
    q, k, v = rnd(g, B, Nq, 2 * Hq, d, dtype=BF), rnd(g, B, S, 2 * Hkv, d, dtype=BF), rnd(g, B, S, Hkv, 2 * d, dtype=BF)
    lam, go = torch.full((Hq,), 0.3, device="cuda"), rnd(g, B, Nq, Hq, 2 * d, dtype=BF)
    start = torch.tensor(([0, 61, -3, 40] * 4)[:B], dtype=torch.int32, device="cuda")
    kw = dict(causal=True, q_start=start)
    want = run_diff(q, k, v, lam, go, dict(kw, kv_len=(start + Nq).clamp_(0, S).to(torch.int32)))
    gap = torch.arange(S, device="cuda")[None, :] >= (start + Nq)[:, None]
    got = run_diff(q, k.masked_fill(gap[..., None, None], math.nan), v.masked_fill(gap[..., None, None], math.nan), lam, go, kw)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    assert not got["k"][gap].any() and not got["v"][gap].any()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hkv,d", [(3, 70, 50, 2, 1, 64), (3, 70, 50, 4, 2, 128), (3, 45, 40, 4, 1, 32), (3, 300, 2100, 2, 2, 64), (3, 300, 2100, 2, 2, 32),
                                              (3, 300, 2100, 2, 1, 128), (9, 130, 70, 32, 32, 64), (9, 130, 70, 32, 32, 32), (9, 130, 70, 32, 32, 128), (3, 5, 900, 4, 2, 64)])
def test_diff_what_queries_without_keys_hold(dev, B, Nq, Nk, Hq, Hkv, d, dtype):
    """a batch padded on the left, and entries without keys: NaN and infinities in q and dO of the queries that see nothing show nowhere"""
    g = torch.Generator("cuda").manual_seed(Nq + d)
    q, k, v = rnd(g, B, Nq, 2 * Hq, d, dtype=dtype), rnd(g, B, Nk, 2 * Hkv, d, dtype=dtype), rnd(g, B, Nk, Hkv, 2 * d, dtype=dtype)
    lam, go = torch.full((Hq,), 0.3, device="cuda"), rnd(g, B, Nq, Hq, 2 * d, dtype=dtype)
    start = torch.tensor(([-40, -3, 5] * 3)[:B], dtype=torch.int32, device="cuda")
    lens = torch.tensor(([Nk, Nk - 7, 0] * 3)[:B], dtype=torch.int32, device="cuda")
    for kw in (dict(causal=True, q_start=start), dict(causal=True, q_start=start, kv_len=lens), dict(kv_len=lens)):
        blind = torch.zeros(B, Nq, dtype=torch.bool, device="cuda")
        if kw.get("causal"):
            blind |= torch.arange(Nq, device="cuda")[None] < -start[:, None]
        if "kv_len" in kw:
            blind |= (lens == 0)[:, None]
        at = blind[..., None, None]
        want = run_diff(q.masked_fill(at, 0), k, v, lam, go.masked_fill(at, 0), kw)
        assert all(torch.isfinite(x).all() for x in want.values()) and not want["o"][blind].any() and not want["q"][blind].any()
        for x, y in ((math.nan, math.nan), (math.inf, -math.inf), (math.nan, 1.0), (1.0, math.inf)):
            got = run_diff(q.masked_fill(at, x), k, v, lam, go.masked_fill(at, y), kw)
            for n in want:
                assert torch.equal(got[n], want[n]), (n, x, y)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_diff_saved_tensors_that_come_back_dense(dev, d):
    """operands that are views, saved to host memory for the backward pass: the copies that come back have strides of their own"""
    g = torch.Generator("cuda").manual_seed(d)
    B, N, Hq = 2, 150, 2
    proj = rnd(g, B, N, 3 * 2 * Hq * d, dtype=BF).requires_grad_()
    lam, go = torch.full((Hq,), 0.3, device="cuda", requires_grad=True), rnd(g, B, Hq, N, 2 * d, dtype=BF).transpose(1, 2)
    lens, start = torch.tensor([N, N - 9], dtype=torch.int32, device="cuda"), torch.tensor([0, -5], dtype=torch.int32, device="cuda")
    plan, pos = H.RotaryAxes((4, 6, 6)), torch.randint(0, 99, (3, N), generator=g, device="cuda")
    def grads():
        q, k, v = proj.chunk(3, -1)
        q = H.rotary_axes(q.view(B, N, 2 * Hq, d), None, pos.t().contiguous().t(), plan)
        o = H.diff_attention(q, k.view(B, N, 2 * Hq, d), v.view(B, N, Hq, 2 * d), lam, causal=True, q_start=start, kv_len=lens)
        return lambda: (o, *torch.autograd.grad(o, (proj, lam), go))
    want = grads()()
    with torch.autograd.graph.save_on_cpu():
        later = grads()
    assert all(torch.equal(a, b) for a, b in zip(want, later()))


def test_diff_shared_and_broadcast_weight(dev):
    q, k, v, _, go, kw, _ = diff_case(21, 2, 50, 60, 4, 2, 32, BF)
    lam = torch.tensor(0.7, device="cuda")
    a = run_diff(q, k, v, lam, go, kw)
    per = lam.clone().requires_grad_()
    o = H.diff_attention(q, k, v, per.expand(4), **kw)
    (d,) = torch.autograd.grad(o, per, go)
    heads = run_diff(q, k, v, lam.expand(4).contiguous(), go, kw)
    assert torch.equal(o, a["o"]) and torch.equal(o, heads["o"])
    assert abs(float(d - a["lam"])) <= 2.0 ** -21 * float(heads["lam"].abs().sum())          # the same four numbers, added in another order


def test_diff_captured(dev):
    """forward and backward captured (no eager graph of the leaves lives then: torch's accumulation nodes would tie it to the capture); replays
    with other inputs and eager work between them"""
    B, N, Hq, d = 2, 100, 2, 64
    g = torch.Generator("cuda").manual_seed(31)
    ins = [rnd(g, B, N, 2 * Hq, d, dtype=BF), rnd(g, B, N, 2 * Hq, d, dtype=BF), rnd(g, B, N, Hq, 2 * d, dtype=BF), torch.rand(Hq, generator=g, device="cuda")]
    go = rnd(g, B, N, Hq, 2 * d, dtype=BF)
    one = [rnd(g, B, 1, 2 * Hq, d, dtype=BF), torch.zeros(B, 4000, 2 * Hq, d, dtype=BF, device="cuda"), rnd(g, B, 4000, Hq, 2 * d, dtype=BF)]
    lens = torch.tensor([3000, 7], dtype=torch.int32, device="cuda")
    plan, pos = H.RotaryAxes((8, 12, 12)), torch.randint(0, 999, (3, N), generator=g, device="cuda", dtype=torch.int32)
    def work():
        q, k = H.rotary_axes(ins[0], ins[1], pos, plan)
        o = H.diff_attention(q, k, ins[2], ins[3], causal=True)
        with torch.no_grad():
            t = H.diff_attention(one[0], one[1], one[2], ins[3], kv_len=lens)
        return [o, *torch.autograd.grad(o, ins, go), t]
    for x in ins:
        x.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for i in range(3):
        with torch.no_grad():
            for x in (*ins, *one):
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
            lens.copy_(torch.tensor([1000 * i, 4000 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = work()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        del want


def test_diff_on_two_streams_at_once(dev):
    cases = [diff_case(41 + i, 1, 1 if i % 2 else 200, 3000, 4, 2, 64, BF, causal=True) for i in range(4)]
    want = [run_diff(*c[:5], c[5]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None] * 4
    for i, (s, c) in enumerate(zip(streams, cases)):
        with torch.cuda.stream(s):
            got[i] = run_diff(*c[:5], c[5])
    torch.cuda.synchronize()
    assert all(torch.equal(a[n], b[n]) for a, b in zip(got, want) for n in a)


def test_diff_refusals(dev):
    q, k = torch.zeros(2, 5, 8, 64, dtype=BF, device="cuda"), torch.zeros(2, 7, 4, 64, dtype=BF, device="cuda")
    v, lam = torch.zeros(2, 7, 2, 128, dtype=BF, device="cuda"), torch.zeros(4, device="cuda")
    ok = torch.zeros(2, dtype=torch.int32, device="cuda")
    for args, kw in (((q.float(), k, v, lam), {}), ((q.float(), k.float(), v.float(), lam), {}), ((q[..., :48], k[..., :48], v[..., :96], lam), {}),
                     ((q[:, :, :7], k, v, lam), {}), ((q, k[:, :, :3], v, lam), {}), ((q, torch.cat([k, k[:, :, :2]], 2), v, lam), {}), ((q, k, v[..., :64], lam), {}),
                     ((q, k, v[:, :6], lam), {}), ((q[:1], k, v, lam), {}), ((q, k, v, lam.half()), {}), ((q, k, v, lam[:3]), {}), ((q, k, v, lam.cpu()), {}),
                     ((q, k, v, lam), dict(scale=0.0)), ((q, k, v, lam), dict(scale=-1.0)), ((q, k, v, lam), dict(kv_len=ok.long())), ((q, k, v, lam), dict(kv_len=ok[:1])),
                     ((q, k, v, lam), dict(q_start=[0, 0])), ((q, k, v, lam), dict(q_start=ok.cpu())), ((q[0], k, v, lam), {})):
        with pytest.raises((L.HsError, TypeError)):
            H.diff_attention(*args, **kw)
    o = H.diff_attention(q.requires_grad_(), k, v, lam)
    (dq,) = torch.autograd.grad(o.float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.float().sum().backward()


# ---- AdamW -------------------------------------------------------------------------------------------------------------------
NUM = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def adamw_reference(p, g, m, v, t):
    """(p, m, v) in 64 bits after a step from 64-bit m, v, and the bounds of fp32 arithmetic with p rounded to its type"""
    b1, b2 = NUM["betas"]
    P, G = p.double(), g.double()
    m2, v2 = b1 * m + (1 - b1) * G, b2 * v + (1 - b2) * G * G
    move = NUM["lr"] / (1 - b1 ** t) * m2 / (v2.sqrt() / math.sqrt(1 - b2 ** t) + NUM["eps"])
    new = P * (1 - NUM["lr"] * NUM["weight_decay"]) - move
    tm = 2.0 ** -22 * (b1 * m.abs() + (1 - b1) * G.abs())
    tv = 2.0 ** -22 * v2 + 1e-44
    rel = torch.where(m2 != 0, tm / m2.abs().clamp(min=1e-300), torch.zeros_like(m2))
    tp = half(p.dtype) * new.abs() + floor(p.dtype) + 2.0 ** -22 * (P.abs() + move.abs()) + move.abs() * rel * 1.01 + 1e-30
    return (new, tp), (m2, tm), (v2, tv)


def make(shapes, dtype, seed, unaligned=False):
    g = torch.Generator("cuda").manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        n = math.prod(s)
        flat = rnd(g, n + 1, dtype=dtype, scale=0.5)
        p = flat[1:].view(s) if unaligned else flat[:n].view(s)
        if len(s) == 2 and i % 2:
            p = p.view(s[1], s[0]).t()
        out.append(p.detach().requires_grad_())
    return out, g


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("unaligned", [False, True])
def test_adamw_values(dev, dtype, bits, unaligned):
    shapes = [(1,), (3,), (255,), (256,), (257,), (33, 65), (65, 33), (4096,), (4097,), (0,), (5, 3, 7), (20000,)] + [(i + 1,) for i in range(60)]
    ps, g = make(shapes, dtype, 1, unaligned)
    opt = H.AdamW(ps, state_bits=bits, **NUM)
    for t in (1, 2, 3):
        before = [p.detach().clone() for p in ps]
        if t == 1:
            ms = vs = [torch.zeros_like(p, dtype=torch.float64) for p in ps]
        else:
            ms, vs = zip(*[[x.double() for x in opt.moments(p)] for p in ps])
        for i, p in enumerate(ps):
            p.grad = None if i == 5 and t == 2 else rnd(g, *p.shape, dtype=dtype, scale=10.0 ** (i % 7 - 4)) * (torch.rand(p.shape, generator=g, device="cuda") < 0.9)
        opt.step()
        for i, (p, b, m, v) in enumerate(zip(ps, before, ms, vs)):
            if p.grad is None:
                assert torch.equal(p, b)
                continue
            count = t - (i == 5 and t == 3)
            assert int(opt.state[p]["step"][0]) == count
            (rp, tp), (rm, tm), (rv, tv) = adamw_reference(b, p.grad, m, v, count)
            within(p.detach(), rp, tp, f"p{i} step {t}")
            gm, gv = opt.moments(p)
            if bits == 8 and p.numel():
                # memory order; a code is the nearest step of the square-root scale: off by half a step in the root, and what fp32 adds
                order = sorted(range(p.dim()), key=lambda a: -p.stride(a))
                flat = lambda x: torch.cat([x.permute(order).reshape(-1), x.new_zeros(-x.numel() % 256)]).view(-1, 256)  # noqa: E731
                for got, ref, top in ((gm, rm, 127), (gv.double().sqrt(), rv.sqrt(), 255)):
                    x, y = flat(got.double()), flat(ref)
                    s = y.abs().amax(1, keepdim=True).clamp(min=1e-30)
                    r = lambda z: z.sign() * (z.abs() / s).sqrt() * top  # noqa: E731
                    off = (r(x) - r(y)).abs()
                    lift = (top == 255) & (y > 0) & (r(y) < 1)               # a v > 0 is held as the smallest step at least
                    assert bool((torch.where(lift, off - 1, off - 0.5) <= top * 2.0 ** -18 + 1e-6).all()), (i, t, top, float(off.max()))
                assert bool((gv[rv > 1e-30] > 0).all())
            else:
                within(gm, rm, tm, f"m{i}")
                within(gv, rv, tv, f"v{i}")


def test_adamw_follows_torch(dev):
    """20 steps with fp32 moments beside torch.optim.AdamW on the same gradients: the same formula up to rounding (each step's error, bounded as
    above, adds up to 20 of them)"""
    ps, g = make([(64, 48), (100,), (7, 5, 3)], F32, 2)
    qs = [p.detach().clone().requires_grad_() for p in ps]
    a, b = H.AdamW(ps, **NUM), torch.optim.AdamW(qs, **NUM)
    for _ in range(20):
        for p, q in zip(ps, qs):
            p.grad = rnd(g, *p.shape)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    for p, q in zip(ps, qs):
        within(p.detach(), q.detach().double(), 20 * 2.0 ** -21 * (q.detach().double().abs() + 20 * NUM["lr"]) + 1e-30)


def test_adamw_state_dict_groups_and_reload(dev):
    ps, g = make([(300,), (65, 33), (9,)], BF, 3)
    groups = lambda x: [{"params": x[:2]}, {"params": x[2:], "state_bits": 32, "lr": 1e-2, "weight_decay": 0.0}]  # noqa: E731
    opt = H.AdamW(groups(ps), state_bits=8, **NUM)
    grads = [[rnd(g, *p.shape, dtype=BF) for p in ps] for _ in range(4)]
    def step(o, params, gs):
        for p, x in zip(params, gs):
            p.grad = x
        o.step()
    for gs in grads[:2]:
        step(opt, ps, gs)
    import io
    f = io.BytesIO()
    torch.save(opt.state_dict(), f)
    f.seek(0)
    qs = [p.detach().clone(memory_format=torch.preserve_format).requires_grad_() for p in ps]
    new = H.AdamW(groups(qs), state_bits=8, **NUM)
    new.load_state_dict(torch.load(f, weights_only=True))
    assert new.state[qs[0]]["exp_avg"].dtype == torch.int8 and new.state[qs[0]]["exp_avg_sq"].dtype == torch.uint8
    assert new.state[qs[1]]["exp_avg"].stride() == qs[1].stride() and new.state[qs[2]]["exp_avg"].dtype == F32
    for gs in grads[2:]:
        step(opt, ps, gs)
        step(new, qs, gs)
    assert all(torch.equal(a, b) for a, b in zip(ps, qs))
    out = [torch.empty_like(p, dtype=BF, requires_grad=False) for p in ps], [torch.empty_like(p, dtype=BF, requires_grad=False) for p in ps]
    new.read_moments(*out)
    for i, p in enumerate(qs):
        m, v = new.moments(p)
        assert torch.equal(out[0][i], m.bfloat16()) and torch.equal(out[1][i], v.bfloat16())


def test_adamw_gradients_of_another_order_and_not_finite(dev):
    g = torch.Generator("cuda").manual_seed(4)
    p = rnd(g, 70, 40).requires_grad_()
    q = p.detach().clone().requires_grad_()
    a, b = H.AdamW([p], state_bits=8, **NUM), H.AdamW([q], state_bits=8, **NUM)
    x = rnd(g, 40, 70).t()
    p.grad, q.grad = x, x.contiguous()
    a.step()
    b.step()
    assert torch.equal(p, q)
    for worst in (math.nan, math.inf):
        q.grad = torch.zeros_like(q)
        q.grad.view(-1)[300] = worst
        b.step()
        m, v = (t.view(-1) for t in b.moments(q))
        assert torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all() and torch.isfinite(m[:256]).all() and torch.isfinite(v[512:]).all()
        assert not torch.isfinite(q.view(-1)[300]) and torch.isfinite(q.view(-1)[512:]).all()


def test_adamw_captured(dev):
    g = torch.Generator("cuda").manual_seed(5)
    ps = [rnd(g, 500).requires_grad_(), rnd(g, 30, 30).requires_grad_()]
    qs = [p.detach().clone().requires_grad_() for p in ps]
    a, b = H.AdamW(ps, state_bits=8, **NUM), H.AdamW(qs, state_bits=8, **NUM)
    for p, q in zip(ps, qs):
        p.grad = torch.zeros_like(p)
        q.grad = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(L.HsError, match="before a graph is captured"):
        with torch.cuda.graph(graph):
            a.step()
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for i in range(4):
        for p, q in zip(ps, qs):
            x = rnd(g, *p.shape)
            p.grad.copy_(x)
            q.grad.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and int(a.state[ps[0]]["step"][0]) == i + 2


def test_adamw_refusals(dev):
    p = torch.zeros(8, 8, device="cuda", requires_grad=True)
    opt = H.AdamW([p], state_bits=8)
    p.grad = torch.zeros(8, 8, device="cuda").to_sparse()
    with pytest.raises(L.HsError, match="dense"):
        opt.step()
    gap = torch.zeros(8, 16, device="cuda")[:, :8].requires_grad_()
    gap.grad = torch.zeros(8, 8, device="cuda")
    with pytest.raises(L.HsError):
        H.AdamW([gap]).step()
    c, s = torch.zeros(8, 8, dtype=torch.int8, device="cuda"), torch.zeros(1, device="cuda")
    for kw in (dict(exp_avg=c.float(), exp_avg_sq=c.byte()), dict(exp_avg=c.t()[:4], exp_avg_sq=c.byte()), dict(exp_avg=c, exp_avg_sq=c),
               dict(exp_avg=c, exp_avg_sq=c.byte(), exp_avg_scale=s.double()), dict(exp_avg=c.cpu(), exp_avg_sq=c.byte())):
        with pytest.raises(L.HsError):
            opt.set_state(p, step=0, **{"exp_avg_scale": s, "exp_avg_sq_scale": s, **kw})
    q = torch.zeros(6, 4, device="cuda", requires_grad=True)
    other = H.AdamW([q], state_bits=8)
    q.grad = torch.ones_like(q)
    other.step()
    held = other.state[q]["exp_avg"]
    other.state[q]["exp_avg"] = held.cpu()                    # a state that was moved, a parameter that was given other data
    with pytest.raises(L.HsError, match="device"):
        other.step()
    other.state[q]["exp_avg"], q.grad = held, None
    q.data = torch.zeros(60, 40, device="cuda")
    q.grad = torch.ones_like(q)
    with pytest.raises(L.HsError, match="shape"):
        other.step()
    m = torch.zeros(8, 8, device="cuda")
    for bad in (([m], []), ([m.half()], [m.half()]), ([m[:4]], [m[:4]]), ([m.t()[:, :4]], [m]), ([m], [m.bfloat16()])):
        with pytest.raises(L.HsError):
            opt.read_moments(*bad)


def test_adamw_steps_a_tower(dev):
    """the framework's own encoder under this optimizer: the steps of torch's AdamW, and a forward pass that uses the new weights"""
    torch.manual_seed(4)
    a = H.ViT_stage1(1, (8, 32, 32), (4, 16, 16), num_layers=1, pos_embed="perceptron", classification=True).to("cuda").eval()
    b = copy.deepcopy(a)
    x = torch.rand(2, 1, 8, 32, 32, device="cuda")
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    mine, other = H.AdamW(a.parameters(), **kw), torch.optim.AdamW(b.parameters(), **kw)
    old = a(x)[0].detach().clone()
    for _ in range(2):
        mine.zero_grad(), other.zero_grad()
        a(x)[0].square().sum().backward()
        for p, q in zip(a.parameters(), b.parameters()):
            q.grad = None if p.grad is None else p.grad.clone()
            q.data.copy_(p)
        mine.step(), other.step()
        for (n, p), q in zip(a.named_parameters(), b.parameters()):
            # a step is at most lr (1 / (1 - beta1)) long; a dozen roundings of 2^-24 on it, two on the weight
            assert ((p - q).abs() <= 12 * 2.0 ** -24 * 10 * kw["lr"] + 2.0 ** -23 * q.abs()).all(), n
    b.load_state_dict(a.state_dict())
    new = a(x)[0]
    assert torch.equal(new, b(x)[0]) and not torch.equal(new, old)


# ---- offsets beyond 32 bits --------------------------------------------------------------------------------------------------------
def test_tokens_that_lie_far_apart(dev):
    """tokens 2^20 and 2^21 elements apart, over more than 2^32 elements: the bits of the same tensors side by side"""
    g = torch.Generator("cuda").manual_seed(21)
    Nk, d, far = 4200, 64, 1 << 20
    room = torch.empty(Nk * far, dtype=BF, device="cuda")
    for Nq, Hq, Hkv in ((1, 4, 2), (40, 16, 16), (300, 16, 8)):
        q, k, v = rnd(g, 1, Nq, 2 * Hq, d, dtype=BF), rnd(g, 1, Nk, 2 * Hkv, d, dtype=BF), rnd(g, 1, Nk, Hkv, 2 * d, dtype=BF)
        K = room.as_strided((1, Nk, 2 * Hkv, d), (Nk * far, far, d, 1))
        V = room.as_strided((1, Nk, Hkv, 2 * d), (Nk * far, far, 2 * d, 1), 4096)
        K.copy_(k), V.copy_(v)
        lam, go = torch.full((Hq,), 0.3, device="cuda"), rnd(g, 1, Nq, Hq, 2 * d, dtype=BF)
        want, got = run_diff(q, k, v, lam, go, dict(causal=True)), run_diff(q, K, V, lam, go, dict(causal=True))
        assert all(torch.equal(want[n], got[n]) for n in want)
    plan, N = H.RotaryAxes((9, 10, 12)), 1000
    x, pos = rnd(g, 2, N, 2, d, dtype=BF), torch.randint(0, 500, (3, 2, N), generator=g, device="cuda")
    X = room.as_strided((2, N, 2, d), (N * 2 * far, 2 * far, d, 1))
    X.copy_(x)
    want = H.rotary_axes(x, None, pos, plan)
    assert torch.equal(H.rotary_axes(X, None, pos, plan), want)
    with torch.no_grad():
        H.rotary_axes(X, None, pos, plan, inplace=True)
    assert torch.equal(X, want)


def test_diff_more_than_2_31_outputs(dev):
    Nq, Hq, d = (1 << 17) + 5, 256, 32
    g = torch.Generator("cuda").manual_seed(22)
    q = torch.zeros(1, Nq, 2 * Hq, d, dtype=BF, device="cuda")
    k, v = rnd(g, 1, 40, 2, d, dtype=BF), rnd(g, 1, 40, 1, 2 * d, dtype=BF)
    o = H.diff_attention(q, k, v, torch.tensor(0.5, device="cuda"), kv_len=torch.tensor([1], dtype=torch.int32, device="cuda"))
    want = 0.5 * v[:, :1]
    for part in (o[:, :3000], o[:, 65000:68000], o[:, -3000:]):
        assert torch.equal(part, want.expand_as(part))


def test_diff_more_blocks_than_a_launch_holds(dev):
    """129 queries of one key each in 2^21 - 1 entries: 16 rows a block would be 2^32 threads and more"""
    B, Nq, d = (1 << 21) - 1, 129, 32
    g = torch.Generator("cuda").manual_seed(25)
    q, k, v = torch.zeros(1, Nq, 2, d, dtype=BF, device="cuda"), torch.zeros(1, 1, 2, d, dtype=BF, device="cuda"), rnd(g, B, 1, 1, 2 * d, dtype=BF)
    lam, o = torch.tensor(0.5, device="cuda"), torch.full((B, Nq, 1, 2 * d), math.nan, dtype=BF, device="cuda")
    # (the C call: q and k of one entry stand for all)
    desc = O.DIFF_PACK.pack(O.DIFF_PACK.size, B, Nq, 1, 1, 1, d, O.DTYPE[BF], 0, 0, 0, 0.5, 0, 2 * d, d, 0, 0, d, 2 * d, 0, 0, 0, 0, 0)
    assert O.load().hs_diff_attn_fwd_ws_bytes(desc) == 0
    O.call(0, "hs_diff_attn_fwd", desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), None, None, o.data_ptr(), None, None, None, 0)
    for at in range(0, B, 1 << 17):
        assert torch.equal(o[at:at + (1 << 17)], (0.5 * v[at:at + (1 << 17)]).expand(-1, Nq, -1, -1))


def test_adamw_more_than_2_31_elements(dev):
    n = (1 << 31) + 777
    tail = (n // 256 - 20) * 256
    g = torch.Generator("cuda").manual_seed(23)
    p, grad = torch.zeros(n, dtype=BF, device="cuda"), torch.zeros(n, dtype=BF, device="cuda")
    p[tail:], grad[tail:] = rnd(g, n - tail, dtype=BF), rnd(g, n - tail, dtype=BF)
    small = p[tail:].clone()
    small.grad = grad[tail:].clone()
    p.grad = grad
    big, other = H.AdamW([p], state_bits=8, **NUM), H.AdamW([small], state_bits=8, **NUM)
    big.step(), other.step()
    assert torch.equal(p[tail:], small) and not p[:1 << 20].any() and not p[tail - (1 << 20):tail].any()
    for name in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(big.state[p][name][tail:], other.state[small][name]) and not big.state[p][name][tail - (1 << 20):tail].any()


# ---- the three together ----------------------------------------------------------------------------------------------------------
def test_one_training_step_of_an_attention_layer(dev):
    """projection -> rotary positions of a volume's tokens -> differential attention -> output projection -> loss -> AdamW on all weights, beside the
    same layer in 64 bits.  The gradients agree to bf16's roundings (the layer's four products and the operators: 12 roundings of 2^-9 at random would
    be 7e-3 of a gradient's norm; the bound is four times that), and the step on given gradients is the formula's."""
    g = torch.Generator("cuda").manual_seed(8)
    B, side, Hq, d = 2, (3, 4, 4), 2, 32
    N, W = 48, 2 * Hq * d
    grid = torch.stack(torch.meshgrid(*[torch.arange(s) for s in side], indexing="ij")).reshape(3, N).to("cuda", torch.int32)
    plan = H.RotaryAxes((4, 6, 6))
    x, target = rnd(g, B, N, W), rnd(g, B, N, W)
    ws = [rnd(g, 3 * W, W, scale=W ** -0.5).requires_grad_(), rnd(g, W, W, scale=W ** -0.5).requires_grad_(), torch.rand(Hq, generator=g, device="cuda").requires_grad_()]
    xs = [w.detach().double().requires_grad_() for w in ws]
    qkv = (x.bfloat16() @ ws[0].bfloat16().t())
    q, k = H.rotary_axes(qkv[..., :W].view(B, N, 2 * Hq, d), qkv[..., W:2 * W].view(B, N, 2 * Hq, d), grid, plan)
    o = H.diff_attention(q, k, qkv[..., 2 * W:].view(B, N, Hq, 2 * d), ws[2])
    loss = ((o.flatten(2) @ ws[1].bfloat16().t()).float() - target).square().sum()
    loss.backward()
    y = x.double() @ xs[0].t()
    ang = (grid.double()[plan.axis.long()].t() * plan.freq)[None, :, None]
    def turn(z):
        a, b = z.view(B, N, 2 * Hq, d).chunk(2, -1)
        return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1)
    Q, K, V = turn(y[..., :W]), turn(y[..., W:2 * W]), y[..., 2 * W:].view(B, N, Hq, 2 * d)
    maps = [torch.softmax(torch.einsum("bihd,bjhd->bhij", Q[:, :, m::2], K[:, :, m::2]) * d ** -0.5, -1) for m in (0, 1)]
    O = torch.einsum("bhij,bjhc->bihc", maps[0] - xs[2][:, None, None] * maps[1], V)
    ((O.flatten(2) @ xs[1].t()) - target.double()).square().sum().backward()
    for w, z in zip(ws, xs):
        assert float((w.grad.double() - z.grad).norm()) <= 2.8e-2 * float(z.grad.norm())
    before = [w.detach().clone() for w in ws]
    opt = H.AdamW(ws, state_bits=8, **NUM)
    opt.step()
    for w, b in zip(ws, before):
        zero = torch.zeros_like(b, dtype=torch.float64)
        within(w.detach(), *adamw_reference(b, w.grad, zero, zero, 1)[0])
