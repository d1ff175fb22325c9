"""Verification of drafted tokens (include/cudalm_draft.h). The reference
decodes one token per step and has no counterpart."""
from __future__ import annotations

import ctypes

from . import _I, _P, _SZ, _check, _lib, _stream
from .paged_kv import _empty, _workspace

_L = ctypes.c_int64

_SIGS = {
    "cudalm_draft_verify_workspace_bytes": ([_I, _I, _I], _SZ),
    "cudalm_draft_verify": ([_P, _L, _P, _L, _I, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _SZ, _P], _I),
}
for _name, (_args, _ret) in _SIGS.items():
    _fn = getattr(_lib, _name)
    _fn.argtypes = _args
    _fn.restype = _ret

EXPORTED_SYMBOLS = tuple(_SIGS)

_types = None


def _need(ok, what):
    if not ok:
        raise ValueError("draft: " + what)


def _probs(p, B, rows, V, dtype, index, name):
    """Row stride of probabilities [B, rows, V]."""
    if rows == 0:
        return V
    s = p.stride()
    if (p.shape != (B, rows, V) or p.dtype != dtype or p.get_device() != index or (s[2] != 1 and V != 1) or
            (B != 1 and rows != 1 and s[0] != rows * s[1])):
        raise ValueError(f"draft: {name} is [{B}, {rows}, {V}] of the target's type and GPU, rows contiguous "
                         "and equally spaced")
    # one row per sequence is always equally spaced; the stride of a single row has no meaning
    return s[1] if rows != 1 else s[0] if B != 1 else V


def _plain(t, shape, dtype, index, name):
    if t.shape != shape or t.dtype != dtype or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"draft: {name} is a contiguous {dtype} tensor {list(shape)} on the target's GPU")


def verify(target, draft_probs, tokens, u_accept, u_next, counts=None, out=None, accepted=None,
           workspace=None, stream=None):
    """target [B, G + 1, V] and draft_probs [B, G, V] (None: the draft was
    certain) hold probabilities in float32, bfloat16 or float16; tokens [B, G]
    int32 are the drafted ones, counts [B] int32 how many are valid (None: G),
    u_accept [B, G] and u_next [B] float32 random numbers of [0, 1). Returns
    (out [B, G + 1] int32: the accepted tokens, the next one, -1 after it;
    accepted [B] int32, which may be given as `counts` itself)."""
    global _types
    import torch

    if _types is None:
        _types = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    index, dtype = target.get_device(), target.dtype
    _need(target.dim() == 3 and index >= 0 and dtype in _types,
          "target is [B, G + 1, V] in float32, bfloat16 or float16 on the GPU")
    B, G, V = target.shape
    G -= 1
    _need(B >= 1 and G >= 0 and V >= 1, "target has a row per drafted token and one more")
    ts = _probs(target, B, G + 1, V, dtype, index, "target")
    ds, dp = 0, None
    if draft_probs is not None:
        ds = _probs(draft_probs, B, G, V, dtype, index, "draft_probs")
        dp = draft_probs.data_ptr()
    _plain(tokens, (B, G), torch.int32, index, "tokens")
    _plain(u_accept, (B, G), torch.float32, index, "u_accept")
    _plain(u_next, (B,), torch.float32, index, "u_next")
    if counts is not None:
        _plain(counts, (B,), torch.int32, index, "counts")
    if out is None:
        out = _empty((B, G + 1), torch.int32, index, stream)
    else:
        _plain(out, (B, G + 1), torch.int32, index, "out")
    if accepted is None:
        accepted = _empty((B,), torch.int32, index, stream)
    else:
        _plain(accepted, (B,), torch.int32, index, "accepted")
    need = 0
    if workspace is None:
        need = _lib.cudalm_draft_verify_workspace_bytes(B, G, V)
    at, size, held = _workspace(need, workspace, index, stream)
    rc = _lib.cudalm_draft_verify(target.data_ptr(), ts, dp, ds, _types[dtype],
                                  tokens.data_ptr(), None if counts is None else counts.data_ptr(),
                                  u_accept.data_ptr(), u_next.data_ptr(), out.data_ptr(),
                                  accepted.data_ptr(), B, G, V, at, size, _stream(stream))
    _check(rc, "cudalm_draft_verify")
    return out, accepted
