"""Interface checks of the paged cache and of draft verification that need no
GPU: the library exports what the headers declare, the Python structs match,
and calls that cannot be served are refused before any HIP call."""
import ctypes
import os
import re
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x100000


@pytest.fixture(scope="module")
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


@pytest.fixture(scope="module")
def draft():
    from cudalm_w4a16 import draft

    return draft


@pytest.mark.parametrize("header,module", [("cudalm_paged_kv.h", "paged_kv"), ("cudalm_draft.h", "draft")])
def test_library_exports_every_declared_symbol(w4, header, module):
    import importlib

    text = open(os.path.join(REPO, "include", header)).read()
    syms = set(re.findall(r"\b(cudalm_[a-z0-9_]+)\s*\(", text))
    mod = importlib.import_module("cudalm_w4a16." + module)
    assert syms == set(mod.EXPORTED_SYMBOLS)
    assert all(hasattr(w4.lib(), s) for s in syms)


def test_headers_compile_and_struct_layouts(tmp_path, pk, w4):
    fields = [("kv", "cudalm_paged_kv", pk.KV), ("query", "cudalm_paged_query", pk.Query)]
    src = '#include "cudalm_paged_kv.h"\n#include "cudalm_draft.h"\n#include <cstddef>\n#include <cstdio>\n'
    src += "int main() {\n"
    for _, name, cls in fields:
        src += f'  std::printf("%zu", sizeof({name}));\n'
        for f, _t in cls._fields_:
            src += f'  std::printf(" %zu", offsetof({name}, {f}));\n'
        src += '  std::printf("\\n");\n'
    src += "  return cudalm_draft_verify_workspace_bytes(1, 1, 4097) == 32 ? 0 : 1;\n}\n"
    (tmp_path / "use.cpp").write_text(src)
    libdir = os.path.dirname(w4.LIB_PATH)
    cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-I", os.path.join(REPO, "include"),
           str(tmp_path / "use.cpp"), "-L", libdir, "-lcudalm_w4a16", f"-Wl,-rpath,{libdir}", "-o",
           str(tmp_path / "use")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([str(tmp_path / "use")], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0
    for line, (_, _, cls) in zip(out.stdout.splitlines(), fields):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(cls)] + [
            getattr(cls, f).offset for f, _t in cls._fields_]
    # the packed bytes that the calls pass are these structs
    assert len(pk._pack_kv(*range(12))) == ctypes.sizeof(pk.KV)
    s = pk.Query.from_buffer_copy(pk._pack_query(1, 2, 3, 4, 5, 0.5, 7, 8, 9))
    assert [getattr(s, f) for f, _t in pk.Query._fields_] == [1, 2, 3, 4, 5, 0.5, 7, 8, 9]


GOOD_KV = dict(k=FAKE, v=FAKE, weights=FAKE, tables=FAKE, lens=FAKE, num_pages=10, page_size=16,
               kv_heads=2, head_dim=128, type=0, batch=3, max_pages=4)
GOOD_Q = dict(q=FAKE, out=FAKE, token_stride=1024, head_stride=128, heads=8, scale=0.1, window=0, sinks=0,
              max_len=0)


def _structs(pk, kv=(), q=()):
    return (ctypes.byref(pk.KV(**{**GOOD_KV, **dict(kv)})), ctypes.byref(pk.Query(**{**GOOD_Q, **dict(q)})))


BAD_KV = [(dict(num_pages=0), "EINVAL"), (dict(page_size=8), "EINVAL"), (dict(page_size=48), "EINVAL"),
          (dict(page_size=2048), "EINVAL"), (dict(kv_heads=0), "EINVAL"), (dict(head_dim=96), "EINVAL"),
          (dict(type=2), "EINVAL"), (dict(batch=0), "EINVAL"), (dict(max_pages=0), "EINVAL"),
          (dict(k=None), "ENULL"), (dict(v=None), "ENULL"), (dict(tables=None), "ENULL"),
          (dict(lens=None), "ENULL"), (dict(k=FAKE + 8), "EALIGN"), (dict(v=FAKE + 2), "EALIGN"),
          (dict(tables=FAKE + 2), "EALIGN"), (dict(weights=FAKE + 1), "EALIGN"),
          (dict(max_pages=1 << 27), "ERANGE"), (dict(batch=1 << 24), "ERANGE")]


@pytest.mark.parametrize("bad,code", BAD_KV)
def test_bad_cache_is_refused_by_every_call(pk, w4, bad, code):
    lib, want = w4.lib(), getattr(w4, code)
    kv, q = _structs(pk, kv=bad)
    big = 1 << 40
    assert lib.cudalm_paged_append(kv, FAKE, FAKE, 256, 128, 256, 128, FAKE, 5, None) == want
    assert lib.cudalm_paged_decode(kv, q, 1, 0, FAKE, big, None) == want
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 5, FAKE, big, None) == want
    assert lib.cudalm_paged_evict(kv, FAKE, 4, 5, 1, 1, FAKE, FAKE, 0, FAKE, big, None) == want
    assert lib.cudalm_paged_decode_workspace_bytes(kv, q, 1, 0) == 0
    assert lib.cudalm_paged_prefill_workspace_bytes(kv, q, 5) == 0
    assert lib.cudalm_paged_evict_workspace_bytes(kv, 0) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(heads=0), "EINVAL"), (dict(heads=7), "EINVAL"), (dict(heads=130), "EINVAL"), (dict(q=None), "ENULL"),
    (dict(out=None), "ENULL"), (dict(q=FAKE + 8), "EALIGN"), (dict(out=FAKE + 4), "EALIGN"),
    (dict(token_stride=1028), "EALIGN"), (dict(head_stride=132), "EALIGN")])
def test_bad_query_is_refused(pk, w4, bad, code):
    lib, want = w4.lib(), getattr(w4, code)
    kv, q = _structs(pk, q=bad)
    assert lib.cudalm_paged_decode(kv, q, 1, 0, FAKE, 1 << 40, None) == want
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 5, FAKE, 1 << 40, None) == want


def test_decode_refusals(pk, w4):
    lib = w4.lib()
    kv, q = _structs(pk)
    assert lib.cudalm_paged_decode(kv, q, 0, 0, FAKE, 1 << 40, None) == w4.EINVAL
    assert lib.cudalm_paged_decode(kv, q, 257, 0, FAKE, 1 << 40, None) == w4.EINVAL  # 1028 rows
    assert lib.cudalm_paged_decode(kv, q, 1, 3, FAKE, 1 << 40, None) == w4.EINVAL
    assert lib.cudalm_paged_decode(None, q, 1, 0, FAKE, 1 << 40, None) == w4.ENULL
    assert lib.cudalm_paged_decode(kv, None, 1, 0, FAKE, 1 << 40, None) == w4.ENULL
    need = lib.cudalm_paged_decode_workspace_bytes(kv, q, 1, 1)
    assert need > 0
    assert lib.cudalm_paged_decode(kv, q, 1, 1, None, 1 << 40, None) == w4.ENULL
    assert lib.cudalm_paged_decode(kv, q, 1, 1, FAKE + 8, 1 << 40, None) == w4.EALIGN
    assert lib.cudalm_paged_decode(kv, q, 1, 1, FAKE, need - 1, None) == w4.ERANGE
    kv, q = _structs(pk, kv=dict(weights=None))
    assert lib.cudalm_paged_decode(kv, q, 1, 1, FAKE, 1 << 40, None) == w4.ENULL


def test_prefill_refusals(pk, w4):
    lib = w4.lib()
    kv, q = _structs(pk)
    assert lib.cudalm_paged_prefill(kv, q, FAKE, -1, FAKE, 1 << 40, None) == w4.EINVAL
    assert lib.cudalm_paged_prefill(kv, q, None, 5, FAKE, 1 << 40, None) == w4.ENULL
    assert lib.cudalm_paged_prefill(kv, q, FAKE + 1, 5, FAKE, 1 << 40, None) == w4.EALIGN
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 1 << 24, FAKE, 1 << 60, None) == w4.ERANGE
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 0, None, 0, None) == w4.OK  # nothing to do
    kv, q = _structs(pk, kv=dict(max_pages=4000))  # long enough to be split
    need = lib.cudalm_paged_prefill_workspace_bytes(kv, q, 5)
    assert need > 0
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 5, None, 1 << 40, None) == w4.ENULL
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 5, FAKE + 4, 1 << 40, None) == w4.EALIGN
    assert lib.cudalm_paged_prefill(kv, q, FAKE, 5, FAKE, need - 1, None) == w4.ERANGE


def test_append_refusals(pk, w4):
    lib = w4.lib()
    kv, _ = _structs(pk)
    call = lambda k=FAKE, v=FAKE, s=(256, 128, 256, 128), cu=FAKE, n=5: (  # noqa: E731
        lib.cudalm_paged_append(kv, k, v, *s, cu, n, None))
    assert call(n=-1) == w4.EINVAL
    assert call(cu=None, n=5) == w4.EINVAL  # 5 tokens over 3 sequences
    assert call(n=0) == w4.OK
    assert call(k=None) == w4.ENULL and call(v=None) == w4.ENULL
    assert call(k=FAKE + 2) == w4.EALIGN and call(cu=FAKE + 2) == w4.EALIGN
    for i in range(4):
        s = [256, 128, 256, 128]
        s[i] += 4
        assert call(s=s) == w4.EALIGN
    assert call(n=(1 << 31) - 1) == w4.ERANGE


def test_evict_refusals(pk, w4):
    lib = w4.lib()
    kv, _ = _structs(pk)
    need = lib.cudalm_paged_evict_workspace_bytes(kv, 0)
    assert need > 0
    call = lambda dst=FAKE, pages=4, keep=5, sinks=1, recent=1, kept=FAKE, lens=FAKE, ws=FAKE, size=1 << 40: (  # noqa: E731
        lib.cudalm_paged_evict(kv, dst, pages, keep, sinks, recent, kept, lens, 0, ws, size, None))
    assert call(keep=0) == w4.EINVAL and call(sinks=-1) == w4.EINVAL and call(recent=-1) == w4.EINVAL
    assert call(pages=0) == w4.EINVAL and call(keep=65) == w4.EINVAL
    assert call(dst=None) == w4.ENULL and call(kept=None) == w4.ENULL and call(lens=None) == w4.ENULL
    assert call(ws=None) == w4.ENULL and call(ws=FAKE + 4) == w4.EALIGN and call(dst=FAKE + 1) == w4.EALIGN
    assert call(size=need - 1) == w4.ERANGE
    kv, _ = _structs(pk, kv=dict(weights=None))
    assert call() == w4.ENULL


def test_verify_refusals(draft, w4):
    lib = w4.lib()
    good = dict(target=FAKE, ts=100, dp=FAKE, ds=100, type=0, tokens=FAKE, counts=None, ua=FAKE, un=FAKE,
                out=FAKE, n=FAKE, batch=2, draft=3, vocab=100, ws=FAKE, size=1 << 40, stream=None)
    call = lambda **bad: lib.cudalm_draft_verify(*{**good, **bad}.values())  # noqa: E731
    for bad in (dict(batch=0), dict(draft=-1), dict(vocab=0), dict(type=3), dict(type=-1), dict(ts=99),
                dict(ds=99)):
        assert call(**bad) == w4.EINVAL, bad
    for name in ("target", "tokens", "ua", "un", "out", "n", "ws"):
        assert call(**{name: None}) == w4.ENULL, name
        assert call(**{name: FAKE + 2}) == w4.EALIGN, name
    assert call(dp=FAKE + 2) == w4.EALIGN and call(counts=FAKE + 2) == w4.EALIGN
    assert call(type=1, target=FAKE + 1) == w4.EALIGN
    assert call(size=2 * 16 - 1) == w4.ERANGE
    assert call(vocab=(1 << 22) + 1, ts=1 << 23, ds=1 << 23) == w4.ERANGE
    assert call(batch=65536) == w4.ERANGE
    assert call(batch=65535, vocab=1 << 22, ts=1 << 23, ds=1 << 23, size=1 << 60) == w4.ERANGE


def test_python_layer_refuses(pk, draft):
    """On CPU tensors, or with shapes and types that do not match."""
    import torch

    with pytest.raises(ValueError):
        pk.empty_cache(4, 24, 2, 128, torch.bfloat16, device="cpu")
    with pytest.raises(ValueError):
        pk.empty_cache(4, 16, 2, 100, torch.bfloat16, device="cpu")
    with pytest.raises(ValueError):
        pk.empty_cache(4, 16, 2, 128, torch.float32, device="cpu")
    k, v, w = pk.empty_cache(4, 16, 2, 128, torch.bfloat16, device="cpu", weights=True)
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pk.decode(q, k, v, tables, lens)  # no GPU tensors
    with pytest.raises(ValueError):
        pk.decode(q, k, v.float(), tables, lens)
    with pytest.raises(ValueError):
        pk.decode(q, k, k, tables, lens)
    with pytest.raises(ValueError):
        pk.evict(k, v, tables, lens, None, tables, 3)
    with pytest.raises(ValueError):
        draft.verify(torch.zeros(2, 3, 5), None, tables, tables, tables)
