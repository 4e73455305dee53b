"""ctypes binding of libhsenet_ops.so (include/hsenet_ops.h): the operators beside the encoder path.  As in _lib.py there is no fallback: a
missing library or a negative status raises HsError."""
from __future__ import annotations

import ctypes as C
import os
import struct
import threading

import torch
from torch.autograd import forward_ad

from . import _lib as L

LIB_PATH = os.environ.get("HS_OPS_LIB_PATH") or os.path.join(L.HERE, "lib", "libhsenet_ops.so")
ABI_VERSION = 1
POS_I32, POS_I64, POS_F32 = 0, 1, 2
DTYPE = {torch.bfloat16: L.PREC_BF16, torch.float32: L.PREC_F32, torch.float16: L.PREC_F16}
ADAMW_BLOCK = 256
ROTARY_MAX_PAIRS = 512

_vp, _i, _i64, _sz, _d, _i64x2 = C.c_void_p, C.c_int, C.c_int64, C.c_size_t, C.c_double, C.c_int64 * 2


class _Packed(struct.Struct):
    def pack(self, *numbers) -> bytes:
        try:
            return super().pack(*numbers)
        except struct.error as e:
            raise L.HsError(f"a size does not fit 32 bits: {e}") from e


class RotaryDesc(L._Desc):
    _fields_ = [("struct_size", C.c_uint32), ("B", _i), ("N", _i), ("dh", _i), ("pairs", _i), ("axes", _i), ("heads", _i * 2), ("interleaved", _i),
                ("inverse", _i), ("dtype", _i), ("pos_dtype", _i), ("x_b", _i64x2), ("x_n", _i64x2), ("x_h", _i64x2), ("y_b", _i64x2),
                ("y_n", _i64x2), ("y_h", _i64x2), ("pos_a", _i64), ("pos_b", _i64), ("pos_n", _i64)]


class DiffAttnDesc(L._Desc):
    _fields_ = [("struct_size", C.c_uint32), ("B", _i), ("Nq", _i), ("Nk", _i), ("H", _i), ("Hkv", _i), ("d", _i), ("dtype", _i), ("causal", _i),
                ("q_start0", _i), ("lam_stride", _i), ("scale", C.c_float)] + [(f"{t}_{s}", _i64) for t in ("q", "k", "v", "go") for s in "bnh"]


# descriptors are packed in one go where a call builds them (setting a structure's fields one by one costs more than the launch)
ROTARY_PACK, DIFF_PACK = _Packed("@I11i15q"), _Packed("@I10if12q")
assert ROTARY_PACK.size == C.sizeof(RotaryDesc) and DIFF_PACK.size == C.sizeof(DiffAttnDesc)

SIGNATURES = {
    "hs_ops_version": [],
    "hs_ops_build_id": [],
    "hs_rotary_axes": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp],
    "hs_diff_attn_fwd_ws_bytes": [_vp],
    "hs_diff_attn_bwd_ws_bytes": [_vp],
    "hs_diff_attn_fwd": [_vp] + [_vp] * 10 + [_sz, _vp],
    "hs_diff_attn_bwd": [_vp] + [_vp] * 14 + [_sz, _vp],
    "hs_adamw_multi": [_vp, _i, _i, _i, _d, _d, _d, _d, _d, _vp],
    "hs_adamw_moments": [_vp, _i, _i, _vp],
}
_RESTYPE = {"hs_ops_build_id": C.c_char_p, "hs_diff_attn_fwd_ws_bytes": _sz, "hs_diff_attn_bwd_ws_bytes": _sz}
_lib = None
_lock = threading.Lock()


def load() -> C.CDLL:
    """Load (once) and type the shared library; HsError if it is absent, of another ABI or lacks a symbol."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise L.HsError(f"{LIB_PATH} is missing: the HIP extension has not been built (run `python -m hsenet_amd.build`); hsenet_amd has "
                            "no CPU/PyTorch fallback")
        try:
            lib = C.CDLL(LIB_PATH)
            for name, args in SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes, fn.restype = args, _RESTYPE.get(name, C.c_int)
        except (OSError, AttributeError) as e:
            raise L.HsError(f"cannot load {LIB_PATH}: {e}") from e
        if lib.hs_ops_version() != ABI_VERSION:
            raise L.HsError(f"{LIB_PATH} speaks ABI {lib.hs_ops_version()}, this package ABI {ABI_VERSION} (include/hsenet_ops.h): rebuild it "
                            "(`python -m hsenet_amd.build`)")
        _lib = lib
    return _lib


def check_fresh() -> str:
    """raise unless the loaded library was built from the sources in this tree (skipped for an HS_OPS_LIB_PATH build)."""
    from .build import ops_source_id
    have, want = load().hs_ops_build_id().decode(), ops_source_id()
    if have != want and not os.environ.get("HS_OPS_LIB_PATH"):
        raise L.HsError(f"{LIB_PATH} is stale: built from sources {have}, the tree is {want} (run `python -m hsenet_amd.build`)")
    return have


def device_of(*tensors) -> int:
    """the index of the one GPU that the tensors (None: left out) lie on; HsError where they do not"""
    dev = None
    for t in tensors:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise L.HsError(f"expected a tensor, got {type(t).__name__}")
        if not t.is_cuda:
            raise L.HsError("hsenet_amd kernels need tensors on an MI355X ('cuda') device; there is no CPU fallback")
        i = t.get_device()
        if dev is None:
            dev = i
        elif i != dev:
            raise L.HsError(f"the tensors of one call lie on different devices (cuda:{dev} and cuda:{i})")
    return dev


def refuse_tangents(*tensors) -> None:
    """HsError for a tensor that carries a tangent (torch.autograd.forward_ad): a kernel would return a value without one, which reads as a derivative of 0"""
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
                raise L.HsError("forward-mode derivatives are not supported: call this on the primal, or differentiate backward")


_current_device, _raw_stream = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device, None
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream


def stream(dev: int) -> int:
    return _raw_stream(dev) if _raw_stream is not None else torch.cuda.current_stream(dev).cuda_stream


def call(dev: int, name: str, *args) -> None:
    """enqueues an entry point on device `dev`'s current stream (a caller that made a tensor on another stream orders the two, as with any torch
    operation), with that device the current one"""
    fn = getattr(_lib or load(), name)
    if dev == _current_device():
        rc = fn(*args, stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, stream(dev))
    if rc != L.HS_OK:
        raise L.HsError(f"{name} failed: {rc} ({L._ERR.get(rc, 'unknown')})")


def rows_of_heads(shape, stride, ptr: int) -> bool:
    """whether a [B, N, heads, columns] tensor can be read where it lies by the attention kernels: columns side by side, the other strides (of axes longer
    than 1) positive multiples of 8 elements, tokens and heads at most 2^24 apart, its first element on a 16-byte address"""
    (b, n, h, d), (sb, sn, sh, sd) = shape, stride
    return ptr % 16 == 0 and (sd == 1 or d == 1) and (b == 1 or (sb > 0 and sb % 8 == 0)) and (n == 1 or (0 < sn <= 1 << 24 and sn % 8 == 0)) \
        and (h == 1 or (0 < sh <= 1 << 24 and sh % 8 == 0))


def bnh(shape, stride):
    """strides of batch entry, token and head; 0 for an axis of length 1, which no address uses"""
    return (stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0, stride[2] if shape[2] > 1 else 0)
