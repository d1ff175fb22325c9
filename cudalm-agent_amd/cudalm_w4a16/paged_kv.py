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
counts): the work is split by it.
"""
from __future__ import annotations

import ctypes
import struct

from . import _I, _P, _SZ, _check, _lib, _stream

_L = ctypes.c_int64

_SIGS = {
    "cudalm_paged_append": ([_P, _P, _P, _L, _L, _L, _L, _P, _I, _P], _I),
    "cudalm_paged_decode_workspace_bytes": ([_P, _P, _I, _I], _SZ),
    "cudalm_paged_decode": ([_P, _P, _I, _I, _P, _SZ, _P], _I),
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

_types = None


def _type_of(dtype) -> int:
    global _types
    if _types is None:
        import torch

        _types = {torch.bfloat16: BF16, torch.float16: F16}
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


# the same as bytes: one pack instead of a ctypes store per field
_pack_kv = struct.Struct("5P7i4x").pack
_pack_query = struct.Struct("2P2qifiii4x").pack


def _need(ok, what):
    if not ok:
        raise ValueError("paged_kv: " + what)


def _int32(t, shape, name, device):
    import torch

    _need(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous() and
          t.device == device, f"{name} is a contiguous int32 tensor {list(shape)} on {device}")


def _cache(k, v, tables, lens, weights):
    """struct cudalm_paged_kv of the tensors, as bytes."""
    import torch

    _need(k.dim() == 4 and v.dim() == 5 and tables.dim() == 2,
          "k is [pages, kv_heads, page_size, D], v [pages, kv_heads, page_size / 8, D, 8], "
          "tables [B, W]")
    pages, heads, size, D = k.shape
    _need(tuple(v.shape) == (pages, heads, size // 8, D, 8) and size % 8 == 0 and
          v.dtype == k.dtype, "v does not match k")
    _need(k.is_contiguous() and v.is_contiguous(), "k and v are contiguous")
    device = k.device
    _need(device.type == "cuda" and v.device == device, "k and v are on one GPU")
    B, W = tables.shape
    _int32(tables, (B, W), "tables", device)
    _int32(lens, (B,), "lens", device)
    w = 0
    if weights is not None:
        _need(weights.dtype == torch.float32 and tuple(weights.shape) == (pages, heads, size) and
              weights.is_contiguous() and weights.device == device,
              "weights is a contiguous float32 tensor [pages, kv_heads, page_size]")
        w = weights.data_ptr()
    return _pack_kv(k.data_ptr(), v.data_ptr(), w, tables.data_ptr(), lens.data_ptr(), pages, size,
                    heads, D, _type_of(k.dtype), B, W)


def _rows(x, cols, heads, D, like, name):
    """(token stride, head stride) of x, rows of [heads, D] over its leading dimensions."""
    _need(x.dim() == cols + 2 and x.shape[-1] == D and x.dtype == like.dtype and
          x.device == like.device and (heads is None or x.shape[-2] == heads),
          f"{name} is {x.dtype} {list(x.shape)}, which does not match the cache")
    s = x.stride()
    _need(s[-1] == 1 and (cols == 1 or x.shape[0] == 1 or s[0] == x.shape[1] * s[1]),
          f"{name}: heads are contiguous and tokens equally spaced")
    return s[-3], s[-2]


def _query(q, out, token_stride, head_stride, scale, window, sinks, max_len):
    D = q.shape[-1]
    return _pack_query(q.data_ptr(), out.data_ptr(), token_stride, head_stride, q.shape[-2],
                       D ** -0.5 if scale is None else scale, window, sinks, max_len or 0)


def _workspace(nbytes, workspace, device, stream):
    """(address, bytes) of the caller's workspace or of a new one, with what holds it."""
    import torch

    if workspace is not None:
        _need(workspace.is_contiguous() and workspace.device == device,
              "workspace is a contiguous tensor on the cache's GPU")
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace
    if nbytes == 0:
        return None, 0, None
    if stream is None:
        w = torch.empty(nbytes, dtype=torch.uint8, device=device)
    else:  # memory that is not handed out again before this stream has passed
        s = torch.cuda.ExternalStream(stream) if isinstance(stream, int) else stream
        with torch.cuda.stream(s):
            w = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return w.data_ptr(), nbytes, w


def _out_like(q, out):
    import torch

    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _need(out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous() and
          out.device == q.device, "out is contiguous and like q")
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
    kv = _cache(k, v, tables, lens, weights)
    heads, D = k.shape[1], k.shape[3]
    kt, kh = _rows(k_new, 1, heads, D, k, "k_new")
    vt, vh = _rows(v_new, 1, heads, D, k, "v_new")
    T = k_new.shape[0]
    _need(v_new.shape[0] == T, "k_new and v_new have one row per token")
    cu = None
    if cu_new is not None:
        _int32(cu_new, (tables.shape[0] + 1,), "cu_new", k.device)
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
    accumulate=False, replaces them; max_len then has to hold."""
    kv = _cache(k, v, tables, lens, weights)
    D = k.shape[3]
    one = q.dim() == 3
    ts, hs = _rows(q, 1 if one else 2, None, D, k, "q")
    _need(q.shape[0] == tables.shape[0], "q has one entry per sequence")
    Q = 1 if one else q.shape[1]
    mode = 0 if weights is None else WEIGHTS_ADD if accumulate else WEIGHTS_SET
    out = _out_like(q, out)
    query = _query(q, out, ts, hs, scale, window, sinks, max_len)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_decode_workspace_bytes(kv, query, Q, mode)
    at, size, held = _workspace(need, workspace, k.device, stream)
    rc = _lib.cudalm_paged_decode(kv, query, Q, mode, at, size, _stream(stream))
    _check(rc, "cudalm_paged_decode")
    return out


def prefill(q, cu_new, k, v, tables, lens, scale=None, window: int = 0, sinks: int = 0, max_len=None,
            out=None, workspace=None, stream=None):
    """Attention of a chunk: rows cu_new[b] .. cu_new[b + 1] - 1 of q [T, heads,
    D] are the last tokens of sequence b. Arguments as in decode()."""
    kv = _cache(k, v, tables, lens, None)
    ts, hs = _rows(q, 1, None, k.shape[3], k, "q")
    _int32(cu_new, (tables.shape[0] + 1,), "cu_new", k.device)
    T = q.shape[0]
    out = _out_like(q, out)
    query = _query(q, out, ts, hs, scale, window, sinks, max_len)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_prefill_workspace_bytes(kv, query, T)
    at, size, held = _workspace(need, workspace, k.device, stream)
    rc = _lib.cudalm_paged_prefill(kv, query, cu_new.data_ptr(), T, at, size, _stream(stream))
    _check(rc, "cudalm_paged_prefill")
    return out


def evict(k, v, tables, lens, weights, dst_tables, keep: int, sinks: int = 4, recent: int = 64,
          max_len=None, kept=None, new_lens=None, workspace=None, stream=None):
    """Keeps `keep` tokens of every sequence and key-value head (the first
    `sinks`, the last `recent`, and those with the largest weights) and copies
    them, in order, into the pages of dst_tables [B, W'], which no sequence of
    the call reads. Returns (kept [B, kv_heads, keep] int32 old positions, -1
    past the last; new_lens [B] int32)."""
    import torch

    _need(weights is not None, "eviction goes by the weights")
    kv = _cache(k, v, tables, lens, weights)
    B, heads = tables.shape[0], k.shape[1]
    _need(dst_tables.dim() == 2, "dst_tables is [B, W']")
    _int32(dst_tables, (B, dst_tables.shape[1]), "dst_tables", k.device)
    _need(keep >= 1, "keep is at least 1")
    if kept is None:
        kept = torch.empty(B, heads, keep, dtype=torch.int32, device=k.device)
    _int32(kept, (B, heads, keep), "kept", k.device)
    if new_lens is None:
        new_lens = torch.empty(B, dtype=torch.int32, device=k.device)
    _int32(new_lens, (B,), "new_lens", k.device)
    need = 0
    if workspace is None:
        need = _lib.cudalm_paged_evict_workspace_bytes(kv, max_len or 0)
    at, size, held = _workspace(need, workspace, k.device, stream)
    rc = _lib.cudalm_paged_evict(kv, dst_tables.data_ptr(), dst_tables.shape[1], keep, sinks, recent,
                                 kept.data_ptr(), new_lens.data_ptr(), max_len or 0, at, size,
                                 _stream(stream))
    _check(rc, "cudalm_paged_evict")
    return kept, new_lens


def kernel_regs(dtype, head_dim: int, prefill: bool = False) -> int:
    return _lib.cudalm_paged_kernel_regs(_type_of(dtype), head_dim, int(prefill))
