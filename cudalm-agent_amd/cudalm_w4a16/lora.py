"""Low-rank adapters of many requests beside shared projections
(include/cudalm_lora.h). The reference serves one set of weights and has no
counterpart.

    plan = lora.plan(index, adapters)            # once per batch: which row has which
    q, k, v = w4.gemv_multi(...)                 # per layer, on all rows
    lora.add(x, [q, k, v], [Aq, Ak, Av], [Bq, Bk, Bv], plan, scales)

Tensors are on one GPU; calls run on the current stream, or on `stream` (a torch
stream or a raw handle), and never wait for the device. Arguments that a call cannot
serve raise ValueError, a refused launch RuntimeError. What index and ranks hold is on the
GPU and not checked by the host: a number that names no adapter means none.
"""
from __future__ import annotations

import ctypes
import struct

from . import _I, _P, _SZ, _check, _lib, _stream
from . import paged_kv as _kv
from .paged_kv import _L, _elsewhere, _empty, _type_of

_SIGS = {
    "cudalm_lora_plan_bytes": ([_I, _I], _SZ),
    "cudalm_lora_plan": ([_P, _I, _I, _P, _SZ, _P], _I),
    "cudalm_lora_add": ([_P, _I, _P, _L, _I, _I, _I, _I, _I, _P, _P, _P, _P], _I),
}
for _name, (_args, _ret) in _SIGS.items():
    _fn = getattr(_lib, _name)
    _fn.argtypes = _args
    _fn.restype = _ret

EXPORTED_SYMBOLS = tuple(_SIGS)

MAX_PROJ = 8
MAX_RANK = 256
MAX_ADAPTERS = 4096


class Proj(ctypes.Structure):
    """struct cudalm_lora_proj."""
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("y", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("y_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64), ("N", ctypes.c_int)]


# an array of them as bytes, by their number
_PACK = [struct.Struct("4P2qi4x" * n).pack for n in range(MAX_PROJ + 1)]


def _need(ok, what):
    if not ok:
        raise ValueError("lora: " + what)


class Plan:
    """Rows of a batch in the order of their adapters, on the GPU."""

    def __init__(self, memory, M, adapters):
        self.memory, self.M, self.adapters, self.index = memory, M, adapters, memory.get_device()
        self.at = memory.data_ptr()


def plan(index, adapters: int, out: Plan | None = None, stream=None) -> Plan:
    """The plan of rows with adapters index [M] int32 (outside of 0 .. adapters - 1:
    none), in new memory or in that of `out`, a plan for as many rows and adapters."""
    import torch

    gpu = index.get_device()
    _need(index.dim() == 1 and index.dtype == torch.int32 and index.is_contiguous() and gpu >= 0,
          "index is a contiguous int32 tensor [M] on the GPU")
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return plan(index, adapters, out, stream)
    M = index.shape[0]
    _need(1 <= adapters <= MAX_ADAPTERS and M <= 1 << 22, f"1 to {MAX_ADAPTERS} adapters, at most 2^22 rows")
    if out is None:
        out = Plan(_empty((_lib.cudalm_lora_plan_bytes(M, adapters),), torch.uint8, gpu, stream), M, adapters)
    _need(out.M == M and out.adapters == adapters and out.index == gpu, "out is a plan for as many rows and adapters")
    rc = _lib.cudalm_lora_plan(index.data_ptr(), M, adapters, out.memory.data_ptr(), out.memory.numel(), _stream(stream))
    _check(rc, "cudalm_lora_plan")
    return out


def _bad(name, shape):
    raise ValueError(f"lora: {name} is {shape} in x's type and on its GPU, a row's elements contiguous")


def add(x, ys, a, b, plan: Plan, scales=None, ranks=None, outs=None, stream=None):
    """out_j[m] = y_j[m] + scales[i] * B_j[i] (A_j[i] x[m]) with i the adapter of row m;
    rows of none keep y. x [M, K]; ys, a, b (and outs): one tensor, or a list of up to 8 for
    projections that share x: y [M, N], a [adapters, rank, K], b [adapters, N, rank]. The
    results replace ys, or go to outs, which overlap neither x nor each other. scales [adapters] float32 (None: 1); ranks
    [adapters] int32 (None: all the same): what adapter i uses of the rank, the rest is
    padding. K and rank are multiples of 8. Returns the results, as ys came."""
    if not isinstance(ys, (list, tuple)):
        return add(x, [ys], [a], [b], plan, scales, ranks, None if outs is None else [outs], stream)[0]
    gpu, dtype = x.get_device(), x.dtype
    kind = _type_of(dtype)
    shape = x.shape
    M = plan.M
    if gpu < 0 or len(shape) != 2 or plan.index != gpu or shape[0] != M:
        raise ValueError("lora: x is [M, K] on the GPU of its plan")
    if _elsewhere(gpu):
        import torch

        with torch.cuda.device(gpu):
            return add(x, ys, a, b, plan, scales, ranks, outs, stream)
    K = shape[1]
    s = x.stride()
    if s[1] != 1 and K != 1:
        _bad("x", [M, K])
    x_stride = s[0] if M > 1 else K
    if outs is None:
        outs = ys
    count, L = len(ys), plan.adapters
    if not 1 <= count <= MAX_PROJ or len(a) != count or len(b) != count or len(outs) != count:
        raise ValueError(f"lora: ys, a, b and outs are as many, 1 to {MAX_PROJ}")
    R = a[0].shape[1] if a[0].dim() == 3 else 0
    fields = []
    for y, fa, fb, out in zip(ys, a, b, outs):
        shape, s = y.shape, y.stride()
        if len(shape) != 2 or shape[0] != M or y.dtype != dtype or y.get_device() != gpu or (s[1] != 1 and shape[1] != 1):
            _bad("y", [M, "N"])
        N = shape[1]
        step = to = s[0] if M > 1 else N
        if out is not y:
            s = out.stride()
            if out.shape != shape or out.dtype != dtype or out.get_device() != gpu or (s[1] != 1 and N != 1):
                _bad("out", [M, N])
            to = s[0] if M > 1 else N
        if (fa.shape != (L, R, K) or fb.shape != (L, N, R) or fa.dtype != dtype or fb.dtype != dtype or
                fa.get_device() != gpu or fb.get_device() != gpu or not fa.is_contiguous() or not fb.is_contiguous()):
            raise ValueError(f"lora: a and b are contiguous [{L}, rank, {K}] and [{L}, {N}, rank] in x's type and on its GPU")
        fields += (fa.data_ptr(), fb.data_ptr(), y.data_ptr(), out.data_ptr(), step, to, N)
    sp = rp = None
    if scales is not None:
        if scales.shape != (L,) or scales.dtype != _kv._float32_type or scales.get_device() != gpu or not scales.is_contiguous():
            raise ValueError(f"lora: scales is a contiguous float32 tensor [{L}] on x's GPU")
        sp = scales.data_ptr()
    if ranks is not None:
        if ranks.shape != (L,) or ranks.dtype != _kv._int32_type or ranks.get_device() != gpu or not ranks.is_contiguous():
            raise ValueError(f"lora: ranks is a contiguous int32 tensor [{L}] on x's GPU")
        rp = ranks.data_ptr()
    rc = _lib.cudalm_lora_add(_PACK[count](*fields), count, x.data_ptr(), x_stride, K, M, R, L, kind, sp, rp, plan.at,
                              _stream(stream))
    if rc:
        _check(rc, "cudalm_lora_add")
    return outs
