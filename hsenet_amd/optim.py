"""AdamW over many tensors at once, moments in 32 or 8 bits (``hs_adamw_multi``): the optimizer for a module's own parameters, where the engines'
``hs_adamw_fused`` wants one flat fp32 buffer."""
from __future__ import annotations

from array import array
from typing import List, Optional, Sequence, Tuple

import torch

from . import _lib as L
from . import _ops as O

_BYTES = {8: (torch.int8, torch.uint8), 32: (torch.float32, torch.float32)}


def _dense(t: torch.Tensor) -> bool:
    """whether t's elements fill one stretch of memory, in whatever order of its axes"""
    if t.is_contiguous():
        return True
    want = 1
    for s, n in sorted((s, n) for n, s in zip(t.shape, t.stride()) if n > 1):
        if s != want:
            return False
        want *= n
    return True


class AdamW(torch.optim.Optimizer):
    """p *= 1 - lr * weight_decay; m, v the moments of the gradient; p -= lr m^ / (sqrt(v^) + eps), with all tensors of a group in a launch per 56.

    Parameters: bf16, fp16 or fp32 (arithmetic in fp32, one rounding at the end), dense in any order of their axes, no two in the same memory (they are
    updated side by side), gradients of the same type.
    state_bits 32: moments in fp32.  state_bits 8: int8 and uint8 codes with an fp32 scale per 256 elements of a tensor, in its order in memory
    (include/hsenet_ops.h has the formula): 2.03 bytes an element instead of 8.  The step is taken with the new moments before they are rounded.
    A gradient that is not finite makes its element, and with 8 bits its block's moments, NaN: skip such a step, as torch.amp.GradScaler does.

    state[p]: ``step`` (int32 [4] on the device: the count and scratch), ``exp_avg``, ``exp_avg_sq`` and, with 8 bits, ``exp_avg_scale`` and
    ``exp_avg_sq_scale``.  The count lives on the device, so a step can be captured into a graph (its lr, betas, eps and weight_decay as they were at
    the capture).  A parameter without a gradient is left out of a step."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, group) -> None:
        super().add_param_group(group)
        g = self.param_groups[-1]
        try:
            self._check_numbers(g)
            if g["state_bits"] not in (8, 32):
                raise ValueError("state_bits must be 8 or 32")
            for p in g["params"]:
                if p.dtype not in O.DTYPE:
                    raise ValueError(f"parameters must be bf16, fp16 or fp32, got {p.dtype}")
            if len(set(g["params"])) != len(g["params"]):
                raise ValueError("a parameter stands twice in a group")
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check_numbers(g) -> Tuple[float, float, float, float, float]:
        lr, (b1, b2), eps, wd = g["lr"], g["betas"], g["eps"], g["weight_decay"]
        if isinstance(lr, torch.Tensor):
            raise ValueError("lr must be a number, not a tensor")
        if not lr >= 0 or not 0 <= b1 < 1 or not 0 <= b2 < 1 or not eps >= 0 or not wd >= 0:
            raise ValueError(f"bad lr, betas, eps or weight_decay: {lr}, {(b1, b2)}, {eps}, {wd}")
        return float(lr), float(b1), float(b2), float(eps), float(wd)

    def _bits(self, p) -> int:
        for g in self.param_groups:
            if any(q is p for q in g["params"]):
                return g["state_bits"]
        raise L.HsError("not a parameter of this optimizer")

    def set_state(self, p: torch.Tensor, *, step: int, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, exp_avg_scale: Optional[torch.Tensor] = None,
                  exp_avg_sq_scale: Optional[torch.Tensor] = None) -> None:
        """takes the given tensors as p's state (they are updated in place from now on): of p's shape and memory order, scales [ceil(n / 256)]"""
        bits, new = self._bits(p), {"exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}
        if bits == 8:
            new.update(exp_avg_scale=exp_avg_scale, exp_avg_sq_scale=exp_avg_sq_scale)
        elif exp_avg_scale is not None or exp_avg_sq_scale is not None:
            raise L.HsError("32-bit moments have no scales")
        if not 0 <= int(step) < 1 << 31:
            raise L.HsError(f"step must be the number of steps done, 0 or more, got {step}")
        rec = torch.zeros(4, dtype=torch.int32)
        rec[0] = int(step)
        st = {"step": rec.to(p.device), **new}
        self._check_state(p, st, bits)
        self.state[p] = st

    @staticmethod
    def _check_state(p, st, bits) -> None:
        if not _dense(p):
            raise L.HsError("a parameter's elements must fill one stretch of memory")
        dm, dv = _BYTES[bits]
        for name, dt in (("exp_avg", dm), ("exp_avg_sq", dv)):
            t = st.get(name)
            if not isinstance(t, torch.Tensor) or t.dtype != dt or t.shape != p.shape or t.device != p.device or (t.stride() != p.stride() and p.numel() > 1):
                raise L.HsError(f"{name} must be a {dt} tensor of its parameter's shape, strides and device")
        if bits == 8:
            n = -(-p.numel() // O.ADAMW_BLOCK)
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                t = st.get(name)
                if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != (n,) or t.device != p.device or not t.is_contiguous():
                    raise L.HsError(f"{name} must be a dense fp32 tensor ({n},) on its parameter's device")
        t = st.get("step")
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or tuple(t.shape) != (4,) or t.device != p.device or not t.is_contiguous():
            raise L.HsError("step must be a dense int32 tensor (4,) on its parameter's device")

    def _init_state(self, p, bits) -> dict:
        if torch.cuda.is_current_stream_capturing():
            raise L.HsError("the first step makes the states: take it before a graph is captured")
        dm, dv = _BYTES[bits]
        st = {"step": torch.zeros(4, dtype=torch.int32, device=p.device), "exp_avg": torch.zeros_like(p, dtype=dm),
              "exp_avg_sq": torch.zeros_like(p, dtype=dv)}
        if bits == 8:
            n = -(-p.numel() // O.ADAMW_BLOCK)
            st.update(exp_avg_scale=torch.zeros(n, dtype=torch.float32, device=p.device), exp_avg_sq_scale=torch.zeros(n, dtype=torch.float32, device=p.device))
        self._check_state(p, st, bits)
        self.state[p] = st
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        launches, changed = [], []                             # (a step that is refused for one parameter is taken for none)
        for group in self.param_groups:
            numbers, bits = self._check_numbers(group), group["state_bits"]
            tables, state, key, words, (dm, dv), block = {}, self.state, None, None, _BYTES[bits], O.ADAMW_BLOCK      # (device, type) -> (addresses, gradients)
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                dev, dtype, n = p.get_device(), p.dtype, p.numel()
                if dev < 0:
                    raise L.HsError("hsenet_amd kernels need tensors on an MI355X ('cuda') device; there is no CPU fallback")
                if g.dtype is not dtype or g.get_device() != dev or g.numel() != n:
                    raise L.HsError("a gradient must be of its parameter's type and size and on its device")
                st = state.get(p) or self._init_state(p, bits)
                m, v, t = st["exp_avg"], st["exp_avg_sq"], st["step"]
                # what can be seen without the state's shapes; where it is not as usual, all is looked at
                usual = m.dtype is dm and v.dtype is dv and m.numel() == n == v.numel() and t.numel() == 4 \
                    and m.get_device() == dev == v.get_device() == t.get_device()
                if usual and bits == 8:
                    sm, su = st["exp_avg_scale"], st["exp_avg_sq_scale"]
                    usual = sm.numel() == -(-n // block) == su.numel() and sm.get_device() == dev == su.get_device()
                if not (usual and p.is_contiguous() and g.is_contiguous() and m.is_contiguous() and v.is_contiguous()):
                    if g.layout is not torch.strided or g.shape != p.shape:
                        raise L.HsError("a gradient must be dense and of its parameter's shape")
                    self._check_state(p, st, bits)
                    if g.stride() != p.stride():
                        g = torch.empty_like(p).copy_(g)
                if key != (dev, dtype):
                    key = (dev, dtype)
                    if key not in tables:
                        if dtype not in O.DTYPE:
                            raise L.HsError(f"parameters must be bf16, fp16 or fp32, got {dtype}")
                        tables[key] = (array("q"), [])
                    words, held = tables[key]
                held.append(g)                                 # (a gradient that was copied lives until the launch)
                words.extend((p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), sm.data_ptr(), su.data_ptr(), t.data_ptr(), n) if bits == 8 else
                             (p.data_ptr(), g.data_ptr(), m.data_ptr(), v.data_ptr(), 0, 0, t.data_ptr(), n))
                changed.append(p)
            launches += [(dev, words, held, O.DTYPE[dtype], bits, numbers) for (dev, dtype), (words, held) in tables.items()]
        for dev, words, _, dtype, bits, numbers in launches:
            O.call(dev, "hs_adamw_multi", words.buffer_info()[0], len(words) // 8, dtype, bits, *numbers)
        if changed:
            torch.autograd.graph.increment_version(changed)
        return loss

    @torch.no_grad()
    def read_moments(self, exp_avg: Sequence[torch.Tensor], exp_avg_sq: Sequence[torch.Tensor]) -> None:
        """writes the moments of every parameter (in the groups' order) into the given dense tensors of its shape and strides, all bf16 or all fp32: the
        values that 8-bit codes stand for, or a copy of 32-bit moments.  A parameter that has no state yet has moments of 0."""
        if not len(exp_avg) == len(exp_avg_sq) == sum(len(g["params"]) for g in self.param_groups):
            raise L.HsError("one pair of tensors per parameter expected")
        tables, i = {}, 0
        dtype = exp_avg[0].dtype if exp_avg else torch.float32
        if dtype is not torch.float32 and dtype is not torch.bfloat16:
            raise L.HsError("moments go into bf16 or fp32 tensors")
        for group in self.param_groups:
            bits = group["state_bits"]
            (dm, dv), block = _BYTES[bits], O.ADAMW_BLOCK
            for p in group["params"]:
                x, y, dev, shape, n, plain = exp_avg[i], exp_avg_sq[i], p.get_device(), p.shape, p.numel(), p.is_contiguous()
                i += 1
                if x.dtype is not dtype or y.dtype is not dtype or x.get_device() != dev or y.get_device() != dev or x.shape != shape or y.shape != shape \
                        or not (plain and x.is_contiguous() and y.is_contiguous() or n < 2 or x.stride() == p.stride() == y.stride()):
                    raise L.HsError("moments go into tensors of one type, each of its parameter's shape, strides and device")
                st = self.state.get(p)
                if not st:
                    x.zero_()
                    y.zero_()
                    continue
                m, v = st["exp_avg"], st["exp_avg_sq"]
                usual = plain and m.dtype is dm and v.dtype is dv and m.numel() == n == v.numel() and m.get_device() == dev == v.get_device() \
                    and m.is_contiguous() and v.is_contiguous()
                if usual and bits == 8:
                    sm, su = st["exp_avg_scale"], st["exp_avg_sq_scale"]
                    usual = sm.numel() == -(-n // block) == su.numel() and sm.get_device() == dev == su.get_device()
                if not usual:
                    self._check_state(p, st, bits)
                if bits == 32:
                    x.copy_(m)
                    y.copy_(v)
                else:
                    words = tables.get(dev)
                    if words is None:
                        words = tables[dev] = array("q")
                    sm, su = st["exp_avg_scale"], st["exp_avg_sq_scale"]
                    words.extend((x.data_ptr(), y.data_ptr(), m.data_ptr(), v.data_ptr(), sm.data_ptr(), su.data_ptr(), 0, n))
        for dev, words in tables.items():
            O.call(dev, "hs_adamw_moments", words.buffer_info()[0], len(words) // 8, O.DTYPE[dtype])

    def moments(self, p: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """the moments (m, v) of one parameter in fp32 or bf16, whatever they are held in"""
        m, v = torch.empty_like(p, dtype=dtype, requires_grad=False), torch.empty_like(p, dtype=dtype, requires_grad=False)
        one = AdamW.__new__(AdamW)
        one.param_groups, one.state = [{"params": [p], "state_bits": self._bits(p)}], {p: self.state.get(p)}
        AdamW.read_moments(one, [m], [v])
        return m, v

    def load_state_dict(self, state_dict) -> None:
        """as torch's, but codes and scales keep their types (torch casts a floating parameter's state to the parameter's type).  Moments of 32 bits go to
        the order that the parameter's elements have in memory; codes have to come in that order, for their scales are those of 256 neighbours there.
        A state_dict that is refused leaves the optimizer as it was."""
        held = self.state, self.param_groups
        try:
            super().load_state_dict(state_dict)
            self._take_states(state_dict)
        except Exception:
            self.state, self.param_groups = held
            raise

    def _take_states(self, state_dict) -> None:
        for g in self.param_groups:
            lost = [k for k in ("lr", "betas", "eps", "weight_decay", "state_bits") if k not in g]
            if lost:
                raise L.HsError(f"a loaded group has no {', '.join(lost)}")
            self._check_numbers(g)
            if g["state_bits"] not in (8, 32):
                raise L.HsError(f"state_bits must be 8 or 32, got {g['state_bits']}")
        saved: List = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, (p, bits) in zip(saved, [(p, g["state_bits"]) for g in self.param_groups for p in g["params"]]):
            st = state_dict["state"].get(i)
            if st is None:
                continue
            new = {}
            for k, t in st.items():
                if k in ("exp_avg", "exp_avg_sq"):
                    if t.shape != p.shape:
                        raise L.HsError(f"{k} must be of its parameter's shape {tuple(p.shape)}, got {tuple(t.shape)}")
                    if bits == 8 and any(n > 1 and a != b for n, a, b in zip(p.shape, p.stride(), t.stride())):
                        raise L.HsError(f"{k}: codes of 8 bits belong to the memory order that they were made in, strides {t.stride()}; their parameter "
                                        f"has {p.stride()}")
                    t = torch.empty_like(p, dtype=t.dtype, requires_grad=False).copy_(t)
                elif isinstance(t, torch.Tensor):
                    t = t.detach().to(p.device, copy=True).contiguous()
                new[k] = t
            self._check_state(p, new, bits)
            self.state[p] = new
