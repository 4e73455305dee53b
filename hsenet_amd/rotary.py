"""Rotary positions with several axes: the slice, row and column of a volume's tokens (or time, height and width of a video's) turn pairs of
columns of q and k in front of attention (``hs_rotary_axes``)."""
from __future__ import annotations

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


def _apart(B, N, dh, live) -> bool:
    """a quick proof, for the usual layouts, that no two elements of one or two tensors lie in the same place: entries, tokens and heads step over each
    other in that order, and the tensors lie behind one another, or both inside each row of the same larger tensor"""
    spans = []
    for h, _, (sb, sn, sh), _, _ in live:
        head = (h - 1) * sh + dh
        entry = (N - 1) * sn + head
        if (h > 1 and sh < dh) or (N > 1 and sn < head) or (B > 1 and sb < entry):
            return False
        spans.append((head, (B - 1) * sb + entry))
    if len(live) == 1:
        return True
    (_, x, (sb, sn, _), _, _), (_, y, (tb, tn, _), _, _) = live
    gap, size = y.data_ptr() - x.data_ptr(), x.element_size()
    if gap >= spans[0][1] * size or -gap >= spans[1][1] * size:
        return True
    row = sn if N > 1 else sb
    at, part = divmod(gap % (row * size), size) if row else (0, 1)
    return not part and row == (tn if N > 1 else tb) and sb % row == 0 == tb % row and spans[0][0] <= at <= row - spans[1][0]


def _extent(x, below=None):
    """(elements from x's first to its last, whether every stride steps over all that shorter ones reach); of the strides under `below` alone"""
    reach, plain = 1, True
    for s, n in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1 and (below is None or s < below)):
        plain &= s >= reach
        reach += (n - 1) * s
    return reach, plain


def _share_memory(xs) -> bool:
    """whether two elements of the tensors (one or two [B, N, heads, columns] with their columns side by side) lie in the same place"""
    if all(_extent(x)[1] for x in xs):
        if len(xs) == 1:
            return False
        x, y = sorted(xs, key=torch.Tensor.data_ptr)
        size = x.element_size()
        gap, part = divmod(y.data_ptr() - x.data_ptr(), size)
        if gap >= _extent(x)[0]:
            return False
        # views of the same rows (the thirds of a projection): where all longer strides are multiples of one, places modulo it tell them apart
        for m in {s for s, n in zip(x.stride(), x.shape) if n > 1 and s > 1} if part == 0 else ():
            if all(s < m or s % m == 0 for t in xs for s, n in zip(t.stride(), t.shape) if n > 1):
                at, left, right = gap % m, _extent(x, m)[0], _extent(y, m)[0]
                if left <= at and at + right <= m:
                    return False
    # rows of `columns` elements side by side share some where two starts are nearer than that
    starts = []
    for x in xs:
        at = torch.tensor(x.data_ptr(), dtype=torch.int64)
        for s, n in zip(x.stride()[:3], x.shape[:3]):
            at = at[..., None] + torch.arange(n, dtype=torch.int64) * (s * x.element_size())
        starts.append(at.flatten())
    at = torch.cat(starts).sort().values
    return bool((at.diff() < xs[0].shape[3] * xs[0].element_size()).any())


def _turn(xs, positions, plan, inverse, inplace):
    """the turned tensors of xs (one or two [B, N, heads, dh] of one type), new ones or xs themselves"""
    if not isinstance(plan, RotaryAxes):
        raise L.HsError("plan must be a RotaryAxes")
    dev = O.device_of(*xs, positions, plan.freq)
    x0 = xs[0]
    dt, dtype = x0.dtype, O.DTYPE.get(x0.dtype)
    if dtype is None:
        raise L.HsError(f"q and k must be bf16, fp16 or fp32, got {dt}")
    shape = x0.shape
    if len(shape) != 4:
        raise L.HsError("q and k must be [B, N, heads, columns]")
    B, N, _, dh = shape
    if dh < 2 * plan.pairs:
        raise L.HsError(f"a head of {dh} columns has no room for {plan.pairs} pairs")
    pos_dtype = _POS.get(positions.dtype)
    if pos_dtype is None:
        raise L.HsError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    pshape, pos = positions.shape, positions.stride()
    if pshape == (plan.axes, N):
        pos = (pos[0], 0, pos[1])
    elif pshape != (plan.axes, B, N):
        raise L.HsError(f"positions must be [axes, N] or [axes, B, N] = ({plan.axes}, {B}, {N}), got {tuple(positions.shape)}")
    outs, live = [], []
    for x in xs:
        xshape = x.shape
        if x.dtype is not dt or len(xshape) != 4 or xshape[0] != B or xshape[1] != N or xshape[3] != dh:
            raise L.HsError("q and k must be [B, N, heads, columns] of one type, equal in B, N and columns")
        stride, h = x.stride(), xshape[2]
        if stride[3] != 1 and dh > 1:
            if inplace:
                raise L.HsError("a tensor that is turned in place must have its columns side by side")
            x = x.contiguous()
            stride = x.stride()
        if inplace:
            if any(n > 1 and s == 0 for n, s in zip(xshape, stride)):
                raise L.HsError("a broadcast tensor cannot be turned in place")
            y, ystride = x, stride
        else:
            y = torch.empty_like(x, memory_format=torch.contiguous_format)
            ystride = (N * h * dh, h * dh, dh, 1)
        outs.append(y)
        if B * N * h * dh:
            live.append((h, x, O.bnh(xshape, stride), y, O.bnh(xshape, ystride)))
    if inplace and live and not _apart(B, N, dh, live) and _share_memory([x for _, x, _, _, _ in live]):
        raise L.HsError("tensors that overlap, or one that overlaps itself, cannot be turned in place")
    if live:
        h0, x0, s0, y0, t0 = live[0]
        h1, x1, s1, y1, t1 = live[1] if len(live) > 1 else (0, None, (0, 0, 0), None, (0, 0, 0))
        desc = O.ROTARY_PACK.pack(O.ROTARY_PACK.size, B, N, dh, plan.pairs, plan.axes, h0, h1, plan.interleaved, inverse, dtype, pos_dtype,
                                  s0[0], s1[0], s0[1], s1[1], s0[2], s1[2], t0[0], t1[0], t0[1], t1[1], t0[2], t1[2], *pos)
        O.call(dev, "hs_rotary_axes", desc, x0.data_ptr(), y0.data_ptr(), None if x1 is None else x1.data_ptr(), None if y1 is None else y1.data_ptr(),
               positions.data_ptr(), plan.freq.data_ptr(), plan.axis.data_ptr())
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
    views with their columns side by side (the q and k thirds of one projection); the results are dense.  Differentiable in q and k (backward).
    ``inplace``: the tensors themselves are turned and returned, without a graph (a new token's q and k); no two of their elements may share a place."""
    xs = (q,) if k is None else (q, k)
    O.refuse_tangents(*xs, positions)
    if inplace:
        if k is not None and k.numel() and k.data_ptr() == q.data_ptr():
            raise L.HsError("one tensor cannot be turned in place twice in a call")
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
