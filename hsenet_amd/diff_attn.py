"""Differential attention (``hs_diff_attn_fwd`` / ``hs_diff_attn_bwd``): softmax(q1 k1^T) v - lam softmax(q2 k2^T) v, the difference of two softmax
maps with a learned weight."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L
from . import _ops as O


def _per_entry(t, what, B):
    if t is not None and (not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous()):
        raise L.HsError(f"{what} must be a dense int32 tensor of one number per batch entry ({B})")


def _placed(t):
    """(t, its strides) where the kernels can read it: itself, or a dense copy"""
    shape, stride = t.shape, t.stride()
    if not O.rows_of_heads(shape, stride, t.data_ptr()):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
        stride = t.stride()
    return t, O.bnh(shape, stride)


def _prepare(q, k, v, lam, scale, causal, q_start, kv_len):
    """(device, descriptor's numbers and strides, q, k, v, lam) with the operands where the kernels can read them; HsError for what they cannot take"""
    dev = O.device_of(q, k, v, lam, q_start, kv_len)
    qs, ks, vs, dt = q.shape, k.shape, v.shape, q.dtype
    if not len(qs) == len(ks) == len(vs) == 4:
        raise L.HsError("q, k and v must have 4 axes: [B, tokens, heads, columns]")
    if (dt is not torch.bfloat16 and dt is not torch.float16) or k.dtype is not dt or v.dtype is not dt:
        raise L.HsError("q, k and v must all be bf16 or all fp16")
    B, Nq, H2, d = qs
    Nk, Hk2 = ks[1], ks[2]
    H, Hkv = H2 // 2, Hk2 // 2
    if H2 % 2 or Hk2 % 2 or H < 1 or Hkv < 1 or H % Hkv:
        raise L.HsError(f"q needs 2 H heads and k 2 Hkv, H a multiple of Hkv: got {H2} and {Hk2}")
    if d not in (32, 64, 128):
        raise L.HsError(f"heads of 32, 64 or 128 columns, got {d}")
    if tuple(ks) != (B, Nk, Hk2, d) or tuple(vs) != (B, Nk, Hkv, 2 * d):
        raise L.HsError(f"for q {tuple(qs)} and k {tuple(ks)} v must be {(B, Nk, Hkv, 2 * d)}, got {tuple(vs)}")
    if lam.dtype is not torch.float32 or not (lam.numel() == 1 or tuple(lam.shape) == (H,)):
        raise L.HsError(f"lam must be fp32, one number or one per head ({H},), got {lam.dtype} {tuple(lam.shape)}")
    _per_entry(q_start, "q_start", B)
    _per_entry(kv_len, "kv_len", B)
    scale = d ** -0.5 if scale is None else float(scale)
    if not 1e-30 < scale < 1e6:
        raise L.HsError(f"scale must be positive (between 1e-30 and 1e6), got {scale}")
    (q, sq), (k, sk), (v, sv) = _placed(q), _placed(k), _placed(v)
    lam = lam.contiguous()
    numbers = (O.DIFF_PACK.size, B, Nq, Nk, H, Hkv, d, O.DTYPE[dt], bool(causal), Nk - Nq, int(H > 1 and lam.numel() > 1), scale)
    return dev, numbers, (*sq, *sk, *sv), q, k, v, lam


def _forward(q, k, v, lam, scale, causal, q_start, kv_len, keep):
    """-> (o, and for a backward pass the descriptor's numbers, the operands as they were read, the maps' outputs and statistics)"""
    dev, numbers, strides, q, k, v, lam = _prepare(q, k, v, lam, scale, causal, q_start, kv_len)
    _, B, Nq, Nk, H, _, d = numbers[:7]
    o = q.new_empty((B, Nq, H, 2 * d))
    maps = q.new_empty((2, B, Nq, H, 2 * d)) if keep else None
    lse = torch.empty(B, H, 4, Nq, dtype=torch.float32, device=q.device) if keep else None
    if B * Nq:
        if Nk == 0:
            o.zero_()
        else:
            desc = O.DIFF_PACK.pack(*numbers, *strides, 0, 0, 0)
            n = O.load().hs_diff_attn_fwd_ws_bytes(desc)
            ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
            O.call(dev, "hs_diff_attn_fwd", desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _ptr(q_start), _ptr(kv_len),
                   o.data_ptr(), _ptr(maps), _ptr(lse), _ptr(ws), n)
    return o, numbers, q, k, v, lam, maps, lse


def _ptr(t):
    return None if t is None else t.data_ptr()


class DiffAttnFn(torch.autograd.Function):
    """differential attention and its gradient (q, k, v and lam)."""

    @staticmethod
    def forward(ctx, q, k, v, lam, scale, causal, q_start, kv_len):
        o, numbers, q, k, v, lam, maps, lse = _forward(q, k, v, lam, scale, causal, q_start, kv_len, True)
        ctx.save_for_backward(q, k, v, lam, q_start, kv_len, maps, lse)
        ctx.numbers = numbers
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, lam, q_start, kv_len, maps, lse = ctx.saved_tensors
        dev = O.device_of(q, k, v, lam, q_start, kv_len, maps, lse, go)
        # (what comes back may lie otherwise than what was saved: torch.autograd.graph.save_on_cpu returns dense copies)
        (q, sq), (k, sk), (v, sv), (go, sg) = _placed(q), _placed(k), _placed(v), _placed(go)
        lam, maps, lse = lam.contiguous(), maps.contiguous(), lse.contiguous()
        dq, dk, dv, dlam = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v, lam))
        if q.numel() == 0 or k.numel() == 0:
            return (*(t.zero_() for t in (dq, dk, dv, dlam)), None, None, None, None)
        desc = O.DIFF_PACK.pack(*ctx.numbers, *sq, *sk, *sv, *sg)
        n = O.load().hs_diff_attn_bwd_ws_bytes(desc)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        O.call(dev, "hs_diff_attn_bwd", desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _ptr(q_start), _ptr(kv_len), go.data_ptr(),
               maps.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dlam.data_ptr(), ws.data_ptr(), n)
        return dq, dk, dv, dlam, None, None, None, None


def diff_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor, *, scale: Optional[float] = None, causal: bool = False,
                   q_start: Optional[torch.Tensor] = None, kv_len: Optional[torch.Tensor] = None) -> torch.Tensor:
    """o [B, Nq, H, 2 d] = softmax(scale q1 k1^T) v - lam softmax(scale q2 k2^T) v.

    q [B, Nq, 2 H, d]: heads 2 h and 2 h + 1 are the two queries of head h; k [B, Nk, 2 Hkv, d] likewise; v [B, Nk, Hkv, 2 d]; head h reads key head
    h // (H / Hkv).  bf16 or fp16, d 32, 64 or 128; views with their columns side by side and strides of multiples of 8 elements are read where they lie
    (a cache longer than its tokens, the thirds of one projection), others are copied first.  lam: fp32, one number or [H].  scale: d^-0.5.

    kv_len (int32 [B]): the keys of each entry that count (its first; 0 to Nk); what k and v hold behind them is not used.
    causal: query i of entry b sees the keys j <= q_start[b] + i.  q_start (int32 [B]) is the position of an entry's first query: without it,
    Nk - Nq (the queries are the last tokens).  A query that sees no key gets zeros, and nothing flows back from it, whatever q and
    o's gradient hold there.  What k and v hold at keys that no query of the entry sees is not used either; a NaN at a key that some see may show in all
    queries of the entry.

    Scores, sums and outputs are made in fp32; the softmax weights go through the products with v in 16 bits, an error relative to each map that shows
    beside o where the maps cancel.  A few queries against many keys (a token and its cache) are split over the keys, and there the weights go through in
    two numbers of 16 bits: the same operands may differ by that rounding between the two, which a rule on the sizes chooses.

    Differentiable in q, k, v and lam (backward), without atomics (equal inputs, equal bits); the maps' own outputs are kept for it.  In fp16 a backward
    pass holds P (dP - D), for dk with lam in it, times 16: scale the loss so that |P (dP - D)| max(1, |lam|) stays under 4094."""
    O.refuse_tangents(q, k, v, lam)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (q, k, v, lam)):
        return DiffAttnFn.apply(q, k, v, lam, scale, causal, q_start, kv_len)
    return _forward(q, k, v, lam, scale, causal, q_start, kv_len, False)[0]
