"""Rotary positions with several axes: the slice, row and column of a volume's tokens (or time, height and width of a video's) turn pairs of
columns of q and k in front of attention (``hs_rotary_axes``)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import _ops as O

_POS = {torch.int32: O.POS_I32, torch.int64: O.POS_I64, torch.float32: O.POS_F32}


class RotaryAxes:
    """The turning rates of a head's column pairs.

    sections: pairs of each axis, in the order of the columns (sum P; a head's first 2 P columns turn, any others pass through).
    ladder: ``"shared"``: pair j of all P turns by pos * theta^(-j / P) (one ladder of rates, cut into the axes' sections); ``"per_axis"``: pair i of an
    axis's n turns by pos * theta^(-i / n) (every axis from the fastest rate down).
    interleaved: pairs are columns (2 j, 2 j + 1) instead of (j, j + P).
    The rates are held in 64 bits on ``device``."""

    def __init__(self, sections: Sequence[int], theta: float = 10000.0, ladder: str = "per_axis", interleaved: bool = False, device="cuda"):
        sections = tuple(int(s) for s in sections)
        if not sections or min(sections) < 0 or not 1 <= sum(sections) <= O.ROTARY_MAX_PAIRS:
            raise ValueError(f"sections must be pair counts >= 0 with a sum of 1 to {O.ROTARY_MAX_PAIRS}, got {sections}")
        if ladder not in ("shared", "per_axis"):
            raise ValueError("ladder must be 'shared' or 'per_axis'")
        if not theta > 0:
            raise ValueError("theta must be positive")
        self.sections, self.theta, self.ladder, self.interleaved = sections, float(theta), ladder, bool(interleaved)
        P = sum(sections)
        rates, axis = [], []
        for a, n in enumerate(sections):
            for i in range(n):
                e = i / n if ladder == "per_axis" else len(rates) / P
                rates.append(self.theta ** -e)
                axis.append(a)
        self.pairs, self.axes = P, len(sections)
        self.freq = torch.tensor(rates, dtype=torch.float64, device=device)
        self.axis = torch.tensor(axis, dtype=torch.int32, device=device)

    def to(self, device) -> "RotaryAxes":
        return RotaryAxes(self.sections, self.theta, self.ladder, self.interleaved, device)


def _turn(xs, positions, plan, inverse, inplace):
    """the turned tensors of xs (one or two [B, N, heads, dh] of one type), new ones or xs themselves"""
    if not isinstance(plan, RotaryAxes):
        raise L.HsError("plan must be a RotaryAxes")
    x0, x1 = xs[0], xs[1] if len(xs) > 1 else None
    with O.on_device(x0, x1, positions, plan.freq):
        if x0.dtype not in O.DTYPE:
            raise L.HsError(f"q and k must be bf16, fp16 or fp32, got {x0.dtype}")
        for x in xs:
            if x.dim() != 4 or x.dtype != x0.dtype or x.shape[:2] != x0.shape[:2] or x.shape[3] != x0.shape[3]:
                raise L.HsError("q and k must be [B, N, heads, columns] of one type, equal in B, N and columns")
        B, N, _, dh = x0.shape
        if dh < 2 * plan.pairs:
            raise L.HsError(f"a head of {dh} columns has no room for {plan.pairs} pairs")
        if positions.dtype not in _POS:
            raise L.HsError(f"positions must be int32, int64 or float32, got {positions.dtype}")
        if tuple(positions.shape) == (plan.axes, N):
            pa, pn, pb = positions.stride(0), positions.stride(1), 0
        elif tuple(positions.shape) == (plan.axes, B, N):
            pa, pb, pn = positions.stride()
        else:
            raise L.HsError(f"positions must be [axes, N] or [axes, B, N] = ({plan.axes}, {B}, {N}), got {tuple(positions.shape)}")
        ins = []
        for x in xs:
            if x.stride(3) != 1 and dh > 1:
                if inplace:
                    raise L.HsError("a tensor that is turned in place must have its columns side by side")
                x = x.contiguous()
            if inplace and x.numel() and any(n > 1 and s == 0 for n, s in zip(x.shape, x.stride())):
                raise L.HsError("a broadcast tensor cannot be turned in place")
            ins.append(x)
        outs = ins if inplace else [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in ins]
        if B * N == 0 or all(x.numel() == 0 for x in ins):
            return outs
        live = [(x, y) for x, y in zip(ins, outs) if x.shape[2]]
        d = O.RotaryDesc(B, N, dh, plan.pairs, plan.axes)
        d.interleaved, d.inverse, d.dtype, d.pos_dtype = plan.interleaved, inverse, O.DTYPE[x0.dtype], _POS[positions.dtype]
        for i, (x, y) in enumerate(live):
            d.heads[i] = x.shape[2]
            d.x_b[i], d.x_n[i], d.x_h[i] = O.bnh(x)
            d.y_b[i], d.y_n[i], d.y_h[i] = O.bnh(y)
        d.pos_a, d.pos_b, d.pos_n = pa, pb, pn
        ptr = [p.data_ptr() for xy in live for p in xy] + [None, None]
        O.call("hs_rotary_axes", C.byref(d), *ptr[:4], positions.data_ptr(), plan.freq.data_ptr(), plan.axis.data_ptr(), O.stream())
        return outs


class RotaryAxesFn(torch.autograd.Function):
    """q and k turned by their positions; the gradient is turned back."""

    @staticmethod
    def forward(ctx, positions, plan, *xs):
        ctx.save_for_backward(positions)
        ctx.plan = plan
        return tuple(_turn(xs, positions, plan, False, False))

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        (positions,) = ctx.saved_tensors
        want = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[2 + i]]
        out = [None] * len(grads)
        if want:
            for i, g in zip(want, _turn([grads[i] for i in want], positions, ctx.plan, True, False)):
                out[i] = g
        return (None, None, *out)


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, plan: RotaryAxes, inplace: bool = False):
    """q [B, N, H, dh] and k [B, N, Hkv, dh] (or None) turned by ``positions`` ([axes, N], or [axes, B, N] where the batch entries differ; int32, int64
    or float32) in one launch: (q', k'), or q' where k is None.  bf16, fp16 or fp32; angles are held in 64 bits.  The tensors may be
    views with their columns side by side (the q and k thirds of one projection); the results are dense.  Differentiable in q and k.
    ``inplace``: the tensors themselves are turned and returned, without a graph (a new token's q and k)."""
    xs = (q,) if k is None else (q, k)
    if inplace:
        if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
            raise L.HsError("turning in place is not differentiable: call it under no_grad, or without inplace")
        out = _turn(xs, positions, plan, False, True)
        for x in xs:
            torch.autograd.graph.increment_version(x)
    elif torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        out = RotaryAxesFn.apply(positions, plan, *xs)
    else:
        out = _turn(xs, positions, plan, False, False)
    return out[0] if k is None else (out[0], out[1])
