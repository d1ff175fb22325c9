"""Rotary positions (include/cudalm_rotary.h): rows of heads rotated by their
positions, and new tokens' keys rotated on their way into the paged cache. What the
reference does here: a partial rotation of one axis in a pass of its own
(qwen35_kernels.cu:40-479).

A Rotary is what a model says of its positions: the pairs' frequencies, which
channels make a pair, and which of several axes (time, height, width) a pair goes
by. Tensors are on one GPU; calls run on the current stream, or on `stream` (a torch
stream or a raw handle), and never wait for the device. Arguments that a call cannot
serve raise ValueError, a refused launch RuntimeError.
"""
from __future__ import annotations

import ctypes
import struct

from . import _I, _P, _check, _lib, _stream
from . import paged_kv as _kv
from .paged_kv import _L, _cache, _elsewhere, _empty, _int32, _rows, _type_of

_SIGS = {
    "cudalm_rotary_rotate": ([_P, _P, _I, _I, _I, _P, _P], _I),
    "cudalm_rotary_append": ([_P, _P, _P, _P, _L, _L, _L, _L, _P, _P, _P, _I, _P], _I),
}
for _name, (_args, _ret) in _SIGS.items():
    _fn = getattr(_lib, _name)
    _fn.argtypes = _args
    _fn.restype = _ret

EXPORTED_SYMBOLS = tuple(_SIGS)

MAX_AXES = 4
MAX_PAIRS = 256


class Plan(ctypes.Structure):
    """struct cudalm_rotary."""
    _fields_ = [("freqs", ctypes.c_void_p), ("pairs", ctypes.c_int), ("adjacent", ctypes.c_int),
                ("axes", ctypes.c_int), ("sections", ctypes.c_int * MAX_AXES), ("turns", ctypes.c_int),
                ("scale", ctypes.c_float)]


class Rows(ctypes.Structure):
    """struct cudalm_rotary_rows."""
    _fields_ = [("x", ctypes.c_void_p), ("out", ctypes.c_void_p), ("x_token_stride", ctypes.c_int64),
                ("x_head_stride", ctypes.c_int64), ("out_token_stride", ctypes.c_int64),
                ("out_head_stride", ctypes.c_int64), ("heads", ctypes.c_int)]


_pack_plan = struct.Struct("P8if4x").pack
_pack_rows = struct.Struct("2P4qi4x").pack


def _need(ok, what):
    if not ok:
        raise ValueError("rotary: " + what)


def frequencies(pairs: int, theta: float, device="cuda"):
    """theta ** (-i / pairs) of pair i, float32."""
    import torch

    i = torch.arange(pairs, dtype=torch.float64)
    return (theta ** (-i / pairs)).to(torch.float32).to(device)


class Rotary:
    """freqs [pairs] float32 on the GPU: radians per position of every pair, as they
    are (scaled for long contexts or not). Pair i is channels i and pairs + i, or,
    adjacent, 2 i and 2 i + 1; further channels are not rotated. sections: pairs of
    each axis; axis 0's come first, then axis 1's, or, with turns, they are dealt to
    the axes in turn, one that has all of its own being passed over. scale multiplies
    the rotated channels."""

    def __init__(self, freqs, sections=None, turns: bool = False, adjacent: bool = False, scale: float = 1.0):
        import torch

        _need(freqs.dim() == 1 and freqs.dtype == torch.float32 and freqs.get_device() >= 0 and
              freqs.is_contiguous() and 1 <= freqs.shape[0] <= MAX_PAIRS,
              f"freqs is a contiguous float32 tensor of 1 to {MAX_PAIRS} pairs on the GPU")
        sections = [freqs.shape[0]] if sections is None else [int(n) for n in sections]
        _need(1 <= len(sections) <= MAX_AXES and min(sections) >= 0 and sum(sections) == freqs.shape[0],
              f"sections are the pairs of 1 to {MAX_AXES} axes, {freqs.shape[0]} in all")
        self.freqs, self.pairs, self.axes, self.index = freqs, freqs.shape[0], len(sections), freqs.get_device()
        self._bytes = _pack_plan(freqs.data_ptr(), self.pairs, bool(adjacent), self.axes,
                                 *sections, *[0] * (MAX_AXES - self.axes), bool(turns), scale)


def _positions(rot, positions, T, index):
    """Their address: [axes, T], or [T] for one axis."""
    if (positions.shape != ((T,) if positions.dim() == 1 and rot.axes == 1 else (rot.axes, T)) or
            positions.dtype != _kv._int32_type or positions.get_device() != index or not positions.is_contiguous()):
        raise ValueError(f"rotary: positions is a contiguous int32 tensor {[rot.axes, T]} on the GPU of the rows")
    return positions.data_ptr()


def _strides(shape, s):
    """(token stride, head stride) of [T, heads, D]; 0 where a dimension has one entry."""
    return s[0] if shape[0] != 1 else 0, s[1] if shape[1] != 1 else 0


def _out(x, shape, dtype, index, out, stream):
    """(out, its token and head strides)."""
    if out is None:
        out = _empty(shape, dtype, index, stream)
    s = out.stride()
    if (out is not x and (out.shape != shape or out.dtype != dtype or out.get_device() != index)) or (
            s[2] != 1 and shape[2] != 1):
        raise ValueError("rotary: out is like the rows, a head's elements contiguous")
    return out, _strides(shape, s)


def rotate(x, positions, rot: Rotary, out=None, stream=None):
    """x [T, heads, D] rotated by positions [axes, T] (or [T] for one axis), int32;
    into `out`, which may be x itself (and else overlaps it nowhere), or a new tensor. Any
    strides of tokens and heads; rows of `out` are apart."""
    index, dtype = x.get_device(), x.dtype
    kind = _type_of(dtype)
    shape, s = x.shape, x.stride()
    if len(shape) != 3 or (s[2] != 1 and shape[2] != 1) or index < 0 or index != rot.index:
        raise ValueError("rotary: x is [T, heads, D] on the GPU of the frequencies, a head's elements contiguous")
    if _elsewhere(index):
        import torch

        with torch.cuda.device(index):
            return rotate(x, positions, rot, out, stream)
    T, heads, D = shape
    out, to = _out(x, shape, dtype, index, out, stream)
    at = _positions(rot, positions, T, index)
    rc = _lib.cudalm_rotary_rotate(rot._bytes, _pack_rows(x.data_ptr(), out.data_ptr(), *_strides(shape, s), *to, heads),
                                   T, D, kind, at, _stream(stream))
    if rc:
        _check(rc, "cudalm_rotary_rotate")
    return out


def append(q, k_new, v_new, k, v, tables, lens, rot: Rotary, positions=None, cu_new=None, weights=None,
           out=None, stream=None):
    """paged_kv.append with keys rotated on the way, and queries q [T, heads, D] (or
    None) rotated by the same positions: into `out`, which may be q itself and overlaps no
    other rows of the call, or a new tensor; it is returned. positions [axes, T] int32; None: a token's place in the
    cache (not its position any more after an eviction). Rows of no sequence are left
    as they are."""
    kv, index = _cache(k, v, tables, lens, weights)
    if index != rot.index:
        raise ValueError("rotary: the frequencies are on the cache's GPU")
    if _elsewhere(index):
        import torch

        with torch.cuda.device(index):
            return append(q, k_new, v_new, k, v, tables, lens, rot, positions, cu_new, weights, out, stream)
    heads = k.shape[1]
    kt, kh = _rows(k_new, 1, heads, k, index, "k_new")
    vt, vh = _rows(v_new, 1, heads, k, index, "v_new")
    T = k_new.shape[0]
    if v_new.shape[0] != T or (q is not None and q.shape[0] != T):
        raise ValueError("rotary: q, k_new and v_new have one row per token")
    rows = None
    if q is not None:
        qt, qh = _rows(q, 1, None, k, index, "q")
        out, to = _out(q, q.shape, q.dtype, index, out, stream)
        rows = _pack_rows(q.data_ptr(), out.data_ptr(), qt, qh, *to, q.shape[1])
    else:
        out = None
    at = None if positions is None else _positions(rot, positions, T, index)
    cu = None
    if cu_new is not None:
        _int32(cu_new, (tables.shape[0] + 1,), "cu_new", index)
        cu = cu_new.data_ptr()
    rc = _lib.cudalm_rotary_append(rot._bytes, kv, k_new.data_ptr(), v_new.data_ptr(), kt, kh, vt, vh, rows, at, cu, T,
                                   _stream(stream))
    _check(rc, "cudalm_rotary_append")
    return out
