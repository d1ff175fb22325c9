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
from .paged_kv import _L, _empty, _type_of, _workspace

_SIGS = {
    "cudalm_lora_plan_bytes": ([_I, _I], _SZ),
    "cudalm_lora_plan": ([_P, _I, _I, _P, _SZ, _P], _I),
    "cudalm_lora_workspace_bytes": ([_I, _I, _I, _I], _SZ),
    "cudalm_lora_add": ([_P, _I, _P, _L, _I, _I, _I, _I, _I, _P, _P, _P, _P, _SZ, _P], _I),
}
for _name, (_args, _ret) in _SIGS.items():
    _fn = getattr(_lib, _name)
    _fn.argtypes = _args
    _fn.restype = _ret

EXPORTED_SYMBOLS = tuple(_SIGS)

MAX_PROJ = 8
MAX_RANK = 256
MAX_ADAPTERS = 8192


class Proj(ctypes.Structure):
    """struct cudalm_lora_proj."""
    _fields_ = [("a", ctypes.c_void_p), ("b", ctypes.c_void_p), ("y", ctypes.c_void_p), ("out", ctypes.c_void_p),
                ("y_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64), ("N", ctypes.c_int)]


def _need(ok, what):
    if not ok:
        raise ValueError("lora: " + what)


class Plan:
    """Rows of a batch in the order of their adapters, on the GPU."""

    def __init__(self, memory, M, adapters):
        self.memory, self.M, self.adapters, self.index = memory, M, adapters, memory.get_device()


def _elsewhere(index) -> bool:
    import torch

    return index >= 0 and index != torch.cuda.current_device()


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


def _matrix(t, M, N, dtype, gpu, name):
    """Row stride of t [M, N]; N where there is one row."""
    if (t.dim() != 2 or t.shape[0] != M or (N and t.shape[1] != N) or t.dtype != dtype or t.get_device() != gpu or
            (t.stride(1) != 1 and t.shape[1] != 1)):
        raise ValueError(f"lora: {name} is [{M}, {N or 'N'}] in x's type and on its GPU, a row's elements contiguous")
    return t.stride(0) if M > 1 else t.shape[1]


def add(x, ys, a, b, plan: Plan, scales=None, ranks=None, outs=None, workspace=None, stream=None):
    """out_j[m] = y_j[m] + scales[i] * B_j[i] (A_j[i] x[m]) with i the adapter of row m;
    rows of none keep y. x [M, K]; ys, a, b (and outs): one tensor, or a list of up to 8 for
    projections that share x: y [M, N], a [adapters, rank, K], b [adapters, N, rank]. The
    results replace ys, or go to outs. scales [adapters] float32 (None: 1); ranks
    [adapters] int32 (None: all the same): what adapter i uses of the rank, the rest is
    padding. Returns the results, as ys came."""
    import torch

    gpu, dtype = x.get_device(), x.dtype
    kind = _type_of(dtype)
    if gpu < 0 or x.dim() != 2 or plan.index != gpu or plan.M != x.shape[0]:
        raise ValueError("lora: x is [M, K] on the GPU of its plan")
    if _elsewhere(gpu):
        with torch.cuda.device(gpu):
            return add(x, ys, a, b, plan, scales, ranks, outs, workspace, stream)
    if isinstance(ys, torch.Tensor):
        return add(x, [ys], [a], [b], plan, scales, ranks, None if outs is None else [outs], workspace, stream)[0]
    if outs is None:
        outs = ys
    count, L = len(ys), plan.adapters
    if not 1 <= count <= MAX_PROJ or len(a) != count or len(b) != count or len(outs) != count:
        raise ValueError(f"lora: ys, a, b and outs are as many, 1 to {MAX_PROJ}")
    M, K = x.shape
    x_stride = _matrix(x, M, K, dtype, gpu, "x")
    R = a[0].shape[1] if a[0].dim() == 3 else 0
    fields = []
    for y, fa, fb, out in zip(ys, a, b, outs):
        ysd = _matrix(y, M, 0, dtype, gpu, "y")
        N = y.shape[1]
        if (fa.shape != (L, R, K) or fb.shape != (L, N, R) or fa.dtype != dtype or fb.dtype != dtype or
                fa.get_device() != gpu or fb.get_device() != gpu or not fa.is_contiguous() or not fb.is_contiguous()):
            raise ValueError(f"lora: a and b are contiguous [{L}, rank, {K}] and [{L}, {N}, rank] in x's type and on its GPU")
        osd = ysd if out is y else _matrix(out, M, N, dtype, gpu, "out")
        fields += (fa.data_ptr(), fb.data_ptr(), y.data_ptr(), out.data_ptr(), ysd, osd, N)
    for t, want, name in ((scales, torch.float32, "scales"), (ranks, torch.int32, "ranks")):
        if t is not None and (t.shape != (L,) or t.dtype != want or t.get_device() != gpu or not t.is_contiguous()):
            raise ValueError(f"lora: {name} is a contiguous {want} tensor [{L}] on x's GPU")
    need = 0
    if workspace is None:
        need = _lib.cudalm_lora_workspace_bytes(count, M, R, kind)
    at, size, held = _workspace(need, workspace, gpu, stream)
    rc = _lib.cudalm_lora_add(struct.pack("4P2qi4x" * count, *fields), count, x.data_ptr(), x_stride, K, M, R, L, kind,
                              None if scales is None else scales.data_ptr(), None if ranks is None else ranks.data_ptr(),
                              plan.memory.data_ptr(), at, size, _stream(stream))
    _check(rc, "cudalm_lora_add")
    return outs
