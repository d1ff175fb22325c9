"""Paged key-value cache (include/cudalm_paged_kv.h): writing new tokens,
attention over the pages, eviction.

A layer's cache is k [pages, kv_heads, page_size, D], v [pages, kv_heads,
page_size / 8, D, 8] (eight tokens interleaved) and, optionally, weights
[pages, kv_heads, page_size] in fp32; empty_cache() makes one. tables [B, W]
int32 names the page of tokens [i * page_size, (i + 1) * page_size) of every
sequence, -1 where they are absent; lens [B] int32 is the number of its tokens, the
new ones included. All are torch tensors on one GPU; calls run on the current
stream, or on `stream` (a torch stream or a raw handle), and never wait for
the device. What the reference does here: paged_kv.cu:53-180 and
batch_decode.cu:238-599 (writes and attention, other layouts; no window,
sinks, split or eviction).

Arguments that a call cannot serve raise ValueError, a refused launch
RuntimeError. What tables and lens hold is on the GPU and not checked by the
host: the kernels skip pages that are out of range.

max_len is what the caller knows of the longest sequence (else the tables' width
counts): the work is split by it, and decode's weights are zero past it.
"""
from __future__ import annotations

import ctypes
import functools
import struct

from . import _I, _P, _SZ, _check, _lib, _stream

_L = ctypes.c_int64

_SIGS = {
    "cudalm_paged_append": ([_P, _P, _P, _L, _L, _L, _L, _P, _I, _P], _I),
    "cudalm_paged_decode_workspace_bytes": ([_P, _P, _I, _I], _SZ),
    "cudalm_paged_decode": ([_P, _P, _I, _I, _P, _SZ, _P], _I),
    "cudalm_paged_decode_shared_workspace_bytes": ([_P, _P, _P, _I], _SZ),
    "cudalm_paged_decode_shared": ([_P, _P, _P, _I, _P, _SZ, _P], _I),
    "cudalm_paged_prefill_workspace_bytes": ([_P, _P, _I], _SZ),
    "cudalm_paged_prefill": ([_P, _P, _P, _I, _P, _SZ, _P], _I),
    "cudalm_paged_evict_workspace_bytes": ([_P, _I], _SZ),
    "cudalm_paged_evict": ([_P, _P, _I, _I, _I, _I, _P, _P, _I, _P, _SZ, _P], _I),
    "cudalm_paged_kernel_regs": ([_I, _I, _I], _I),
}
for _name, (_args, _ret) in _SIGS.items():
    _fn = getattr(_lib, _name)
    _fn.argtypes = _args
    _fn.restype = _ret

EXPORTED_SYMBOLS = tuple(_SIGS)

BF16 = 0
F16 = 1
WEIGHTS_SET = 1
WEIGHTS_ADD = 2

HEAD_DIMS = (64, 128, 256)

_types = None  # torch's, once a call needs them


def _load_types():
    global _types, _int32_type, _float32_type
    import torch

    _int32_type, _float32_type = torch.int32, torch.float32
    _types = {torch.bfloat16: BF16, torch.float16: F16}  # last: other threads go by it


def _type_of(dtype) -> int:
    if _types is None:
        _load_types()
    try:
        return _types[dtype]
    except KeyError:
        raise ValueError(f"paged_kv: {dtype} is not served (bfloat16 or float16)") from None


class KV(ctypes.Structure):
    """struct cudalm_paged_kv."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("weights", ctypes.c_void_p),
                ("tables", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("num_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("type", ctypes.c_int), ("batch", ctypes.c_int), ("max_pages", ctypes.c_int)]


class Query(ctypes.Structure):
    """struct cudalm_paged_query."""
    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("token_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("heads", ctypes.c_int), ("scale", ctypes.c_float),
                ("window", ctypes.c_int), ("sinks", ctypes.c_int), ("max_len", ctypes.c_int)]


class Groups(ctypes.Structure):
    """struct cudalm_paged_groups."""
    _fields_ = [("cu", ctypes.c_void_p), ("shared", ctypes.c_void_p), ("count", ctypes.c_int),
                ("max_shared", ctypes.c_int)]


# the same as bytes: one pack instead of a ctypes store per field
_pack_kv = struct.Struct("5P7i4x").pack
_pack_query = struct.Struct("2P2qifiii4x").pack
_pack_groups = struct.Struct("2P2i").pack


def _need(ok, what):
    if not ok:
        raise ValueError("paged_kv: " + what)


# The checks of a call are in its time (a decode step's small calls take about ten
# microseconds): device indexes in place of device objects, sizes compared as
# torch.Size, messages made where one is needed.

def _bad_int32(name, shape):
    raise ValueError(f"paged_kv: {name} is a contiguous int32 tensor {list(shape)} on the cache's GPU")


def _int32(t, shape, name, index):
    if t.shape != shape or t.dtype != _int32_type or t.get_device() != index or not t.is_contiguous():
        _bad_int32(name, shape)


def _cache(k, v, tables, lens, weights):
    """(struct cudalm_paged_kv of the tensors as bytes, GPU index)."""
    if _types is None:
        _load_types()
    if k.dim() != 4 or tables.dim() != 2:
        raise ValueError("paged_kv: k is [pages, kv_heads, page_size, D], tables [B, W]")
    pages, heads, size, D = k.shape
    index = k.get_device()
    dtype = k.dtype
    kind = _types.get(dtype)
    if kind is None:
        _type_of(dtype)
    if (v.shape != (pages, heads, size // 8, D, 8) or v.dtype != dtype or v.get_device() != index or
            size % 8 or index < 0 or not k.is_contiguous() or not v.is_contiguous()):
        raise ValueError("paged_kv: k and v are contiguous, of one type and on one GPU, v is [pages, "
                         "kv_heads, page_size / 8, D, 8]")
    B, W = tables.shape
    if (tables.dtype != _int32_type or tables.get_device() != index or not tables.is_contiguous()):
        _bad_int32("tables", (B, W))
    _int32(lens, (B,), "lens", index)
    w = 0
    if weights is not None:
        if (weights.shape != (pages, heads, size) or weights.dtype != _float32_type or
                weights.get_device() != index or not weights.is_contiguous()):
            raise ValueError("paged_kv: weights is a contiguous float32 tensor [pages, kv_heads, "
                             "page_size] on the cache's GPU")
        w = weights.data_ptr()
    return _pack_kv(k.data_ptr(), v.data_ptr(), w, tables.data_ptr(), lens.data_ptr(), pages, size,
                    heads, D, kind, B, W), index


def _rows(x, cols, heads, like, index, name):
    """(token stride, head stride) of x: rows of [heads, D] over its leading dimensions.
    Strides of dimensions of one entry have no meaning; 0 where that is all there is."""
    shape, s = x.shape, x.stride()
    if (len(shape) != cols + 2 or shape[-1] != like.shape[3] or x.dtype != like.dtype or
            x.get_device() != index or (heads and shape[-2] != heads)):
        raise ValueError(f"paged_kv: {name} ({x.dtype} {list(shape)} on {x.device}) does not match the cache")
    between = s[-3] if shape[-3] != 1 else 0
    if cols == 2 and shape[0] != 1:
        if shape[1] == 1:
            between = s[0]
        elif s[0] != shape[1] * s[1]:
            raise ValueError(f"paged_kv: {name}: tokens are equally spaced")
    if s[-1] != 1:
        raise ValueError(f"paged_kv: {name}: a head's elements are contiguous")
    return between, s[-2] if shape[-2] != 1 else 0


def _need_ints(**values):
    """Whole numbers that the C types hold: ctypes would pass the lower 32 bits of others."""
    for name, x in values.items():
        if not -2 ** 31 <= x < 2 ** 31:
            raise ValueError(f"paged_kv: {name} {x} is past 32 bits")


def _query(q, out, token_stride, head_stride, scale, window, sinks, max_len):
    D = q.shape[-1]
    try:
        return _pack_query(q.data_ptr(), out.data_ptr(), token_stride, head_stride, q.shape[-2],
                           D ** -0.5 if scale is None else scale, window, sinks, max_len or 0)
    except struct.error:
        _need_ints(window=window, sinks=sinks, max_len=max_len or 0)
        raise


def _empty(shape, dtype, index, stream):
    """Memory of the stream that the call runs on: what another stream's work may still
    use is not in it, and it is not handed out again before this one has passed."""
    import torch

    if stream is None:
        return torch.empty(shape, dtype=dtype, device=_devices(index))
    if isinstance(stream, int):
        # (handle 0 is the default stream; ExternalStream takes 0 for none given and would
        # give a stream of torch's pool)
        stream = (torch.cuda.ExternalStream(stream, device=_devices(index)) if stream
                  else torch.cuda.default_stream(_devices(index)))
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=_devices(index))


_current_device = None  # torch's accessor, once a call needs it


def _elsewhere(index) -> bool:
    """Whether the GPU of a call's tensors is not the current one, which launches go to."""
    global _current_device
    if _current_device is None:
        import torch

        try:
            _current_device = torch._C._cuda_getDevice
        except AttributeError:  # a torch without GPUs, or without this accessor
            _current_device = torch.cuda.current_device
    return index >= 0 and index != _current_device()


def _workspace(nbytes, workspace, index, stream):
    """(address, bytes) of the caller's workspace or of a new one, with what holds it."""
    if workspace is not None:
        _need(workspace.is_contiguous() and workspace.get_device() == index,
              "workspace is a contiguous tensor on the GPU of the call")
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace
    if nbytes == 0:
        return None, 0, None
    import torch

    w = _empty((nbytes,), torch.uint8, index, stream)
    return w.data_ptr(), nbytes, w


@functools.lru_cache(maxsize=None)
def _devices(index):
    import torch

    return torch.device("cuda", index)


def _out_like(q, out, index, stream):
    if out is None:
        return _empty(q.shape, q.dtype, index, stream)
    if out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous():
        raise ValueError("paged_kv: out is contiguous and like q")
    return out


def empty_cache(num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype, device="cuda",
                weights: bool = False):
    """(k, v) or (k, v, weights) of a layer's cache, uninitialised (weights are zero)."""
    import torch

    _type_of(dtype)
    _need(num_pages >= 1 and kv_heads >= 1 and head_dim in HEAD_DIMS and 16 <= page_size <= 1024 and
          page_size & (page_size - 1) == 0,
          f"head_dim is one of {HEAD_DIMS}, page_size a power of two of 16 .. 1024")
    k = torch.empty(num_pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
    v = torch.empty(num_pages, kv_heads, page_size // 8, head_dim, 8, dtype=dtype, device=device)
    if not weights:
        return k, v
    return k, v, torch.zeros(num_pages, kv_heads, page_size, device=device)


def append(k_new, v_new, k, v, tables, lens, cu_new=None, weights=None, stream=None) -> None:
    """Writes new tokens' keys and values [T, kv_heads, D] (any token and head
    strides that are multiples of 8) into their pages, and zeros into their
    weights. Rows cu_new[b] .. cu_new[b + 1] - 1 are the last tokens of
    sequence b; without cu_new every sequence has T / B of them."""
    kv, index = _cache(k, v, tables, lens, weights)
    heads = k.shape[1]
    kt, kh = _rows(k_new, 1, heads, k, index, "k_new")
    vt, vh = _rows(v_new, 1, heads, k, index, "v_new")
    T = k_new.shape[0]
    if v_new.shape[0] != T:
        raise ValueError("paged_kv: k_new and v_new have one row per token")
    cu = None
    if cu_new is not None:
        _int32(cu_new, (tables.shape[0] + 1,), "cu_new", index)
        cu = cu_new.data_ptr()
    rc = _lib.cudalm_paged_append(kv, k_new.data_ptr(), v_new.data_ptr(), kt, kh, vt, vh, cu, T,
                                  _stream(stream))
    _check(rc, "cudalm_paged_append")



def decode(q, k, v, tables, lens, scale=None, window: int = 0, sinks: int = 0, weights=None,
           accumulate: bool = True, max_len=None, out=None, workspace=None, stream=None):
    """Attention of the last token(s) of every sequence: q [B, heads, D] (one)
    or [B, Q, heads, D] (Q of them), output like q. scale defaults to D ** -0.5.
    window > 0: a token sees the last `window` tokens (itself included) and the
    first `sinks`. With weights, what every cached token received (summed over
    the new tokens and a group's query heads) is added to them, or, with
    accumulate=False, replaces them; max_len then has to hold. (Drafted tokens that are
    refused later count as well.)"""
    kv, index = _cache(k, v, tables, lens, weights)
    one = q.dim() == 3
    ts, hs = _rows(q, 1 if one else 2, None, k, index, "q")
    if q.shape[0] != tables.shape[0]:
        raise ValueError("paged_kv: q has one entry per sequence")
    Q = 1 if one else q.shape[1]
    mode = 0 if weights is None else WEIGHTS_ADD if accumulate else WEIGHTS_SET
    out = _out_like(q, out, index, stream)
    query = _query(q, out, ts, hs, scale, window, sinks, max_len)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_decode_workspace_bytes(kv, query, Q, mode)
    at, size, held = _workspace(need, workspace, index, stream)
    rc = _lib.cudalm_paged_decode(kv, query, Q, mode, at, size, _stream(stream))
    _check(rc, "cudalm_paged_decode")
    return out


def decode_shared(q, k, v, tables, lens, cu_groups, shared, scale=None, window: int = 0, sinks: int = 0,
                  max_len=None, max_shared=None, out=None, workspace=None, stream=None):
    """decode() for a batch in which groups of sequences begin with the same tokens,
    which are read once for all of a group's queries. Group g is sequences cu_groups[g] ..
    cu_groups[g + 1] - 1 (int32 [G + 1], G at most the batch; the others share nothing); its
    first shared[g] tokens (int32 [G], any number) are those in the pages of its first
    sequence, whatever the other sequences' tables hold there. max_shared is what the
    caller knows of the longest prefix. Other arguments as in decode()."""
    kv, index = _cache(k, v, tables, lens, None)
    if _elsewhere(index):
        import torch

        with torch.cuda.device(index):
            return decode_shared(q, k, v, tables, lens, cu_groups, shared, scale, window, sinks, max_len, max_shared,
                                 out, workspace, stream)
    one = q.dim() == 3
    ts, hs = _rows(q, 1 if one else 2, None, k, index, "q")
    if q.shape[0] != tables.shape[0]:
        raise ValueError("paged_kv: q has one entry per sequence")
    G = shared.shape[0] if shared.dim() == 1 else -1
    _int32(shared, (G,), "shared", index)
    _int32(cu_groups, (G + 1,), "cu_groups", index)
    if max_shared is not None:
        _need_ints(max_shared=max_shared)
    Q = 1 if one else q.shape[1]
    out = _out_like(q, out, index, stream)
    query = _query(q, out, ts, hs, scale, window, sinks, max_len)
    groups = _pack_groups(cu_groups.data_ptr(), shared.data_ptr(), G, max_shared or 0)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_decode_shared_workspace_bytes(kv, query, groups, Q)
    at, size, held = _workspace(need, workspace, index, stream)
    rc = _lib.cudalm_paged_decode_shared(kv, query, groups, Q, at, size, _stream(stream))
    _check(rc, "cudalm_paged_decode_shared")
    return out


def prefill(q, cu_new, k, v, tables, lens, scale=None, window: int = 0, sinks: int = 0, max_len=None,
            out=None, workspace=None, stream=None):
    """Attention of a chunk: rows cu_new[b] .. cu_new[b + 1] - 1 of q [T, heads,
    D] are the last tokens of sequence b. Arguments as in decode()."""
    kv, index = _cache(k, v, tables, lens, None)
    ts, hs = _rows(q, 1, None, k, index, "q")
    _int32(cu_new, (tables.shape[0] + 1,), "cu_new", index)
    T = q.shape[0]
    out = _out_like(q, out, index, stream)
    query = _query(q, out, ts, hs, scale, window, sinks, max_len)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_prefill_workspace_bytes(kv, query, T)
    at, size, held = _workspace(need, workspace, index, stream)
    rc = _lib.cudalm_paged_prefill(kv, query, cu_new.data_ptr(), T, at, size, _stream(stream))
    _check(rc, "cudalm_paged_prefill")
    return out


def evict(k, v, tables, lens, weights, dst_tables, keep: int, sinks: int = 4, recent: int = 64,
          max_len=None, kept=None, new_lens=None, workspace=None, stream=None):
    """Keeps `keep` tokens of every sequence and key-value head (the first
    `sinks`, the last `recent`, and those with the largest weights) and copies
    them, in order, into the pages of dst_tables [B, W'], which no sequence of
    the call reads. Returns (kept [B, kv_heads, keep] int32 old positions, -1
    past the last; new_lens [B] int32, which may be given as `lens` itself)."""
    import torch

    _need(weights is not None, "eviction goes by the weights")
    _need_ints(keep=keep, sinks=sinks, recent=recent, max_len=max_len or 0)
    kv, index = _cache(k, v, tables, lens, weights)
    B, heads = tables.shape[0], k.shape[1]
    _need(dst_tables.dim() == 2, "dst_tables is [B, W']")
    _int32(dst_tables, (B, dst_tables.shape[1]), "dst_tables", index)
    _need(keep >= 1, "keep is at least 1")
    if kept is None:
        kept = _empty((B, heads, keep), torch.int32, index, stream)
    else:
        _int32(kept, (B, heads, keep), "kept", index)
    if new_lens is None:
        new_lens = _empty((B,), torch.int32, index, stream)
    else:
        _int32(new_lens, (B,), "new_lens", index)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_evict_workspace_bytes(kv, max_len or 0)
    at, size, held = _workspace(need, workspace, index, stream)
    rc = _lib.cudalm_paged_evict(kv, dst_tables.data_ptr(), dst_tables.shape[1], keep, sinks, recent,
                                 kept.data_ptr(), new_lens.data_ptr(), max_len or 0, at, size,
                                 _stream(stream))
    _check(rc, "cudalm_paged_evict")
    return kept, new_lens


def kernel_regs(dtype, head_dim: int, prefill: bool = False) -> int:
    return _lib.cudalm_paged_kernel_regs(_type_of(dtype), head_dim, int(prefill))
