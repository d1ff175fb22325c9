"""Refusals of decode with shared prefixes, and its struct, on the CPU."""
import ctypes
import os
import subprocess

import pytest

from test_paged_abi import BAD_KV, FAKE, _structs

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


def _groups(pk, **bad):
    return ctypes.byref(pk.Groups(**{**dict(cu=FAKE, shared=FAKE, count=2, max_shared=0), **bad}))


def test_struct(tmp_path, pk):
    src = '#include "cudalm_paged_kv.h"\n#include <cstddef>\n#include <cstdio>\nint main() {\n'
    src += '  std::printf("%zu", sizeof(cudalm_paged_groups));\n'
    for f, _t in pk.Groups._fields_:
        src += f'  std::printf(" %zu", offsetof(cudalm_paged_groups, {f}));\n'
    (tmp_path / "use.cpp").write_text(src + "}\n")
    cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-I", os.path.join(REPO, "include"), str(tmp_path / "use.cpp"), "-o",
           str(tmp_path / "use")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([str(tmp_path / "use")], capture_output=True, text=True, timeout=120).stdout
    assert [int(x) for x in out.split()] == [ctypes.sizeof(pk.Groups)] + [getattr(pk.Groups, f).offset for f, _t in pk.Groups._fields_]
    g = pk.Groups.from_buffer_copy(pk._pack_groups(1, 2, 3, 4))
    assert (g.cu, g.shared, g.count, g.max_shared) == (1, 2, 3, 4)


@pytest.mark.parametrize("bad,code", BAD_KV)
def test_bad_cache_is_refused(pk, w4, bad, code):
    kv, q = _structs(pk, kv=bad)
    assert w4.lib().cudalm_paged_decode_shared(kv, q, _groups(pk), 1, FAKE, 1 << 40, None) == getattr(w4, code)
    assert w4.lib().cudalm_paged_decode_shared_workspace_bytes(kv, q, _groups(pk), 1) == 0


def test_refusals(pk, w4):
    lib = w4.lib()
    kv, q = _structs(pk)
    need = lib.cudalm_paged_decode_shared_workspace_bytes(kv, q, _groups(pk), 1)
    assert need > 0
    call = lambda g=None, kv=kv, q=q, n=1, ws=FAKE, size=1 << 40: lib.cudalm_paged_decode_shared(  # noqa: E731
        kv, q, _groups(pk) if g is None else g, n, ws, size, None)
    assert call(n=0) == w4.EINVAL and call(n=257) == w4.EINVAL  # 1028 rows
    assert call(g=_groups(pk, count=0)) == w4.EINVAL and call(g=_groups(pk, count=4)) == w4.EINVAL  # of three sequences
    assert lib.cudalm_paged_decode_shared(kv, q, None, 1, FAKE, 1 << 40, None) == w4.ENULL
    assert call(g=_groups(pk, cu=None)) == w4.ENULL and call(g=_groups(pk, shared=None)) == w4.ENULL
    assert call(g=_groups(pk, cu=FAKE + 2)) == w4.EALIGN and call(g=_groups(pk, shared=FAKE + 1)) == w4.EALIGN
    assert call(ws=None) == w4.ENULL and call(ws=FAKE + 8) == w4.EALIGN and call(size=need - 1) == w4.ERANGE
    for bad, code in ((dict(heads=7), w4.EINVAL), (dict(q=None), w4.ENULL), (dict(out=None), w4.ENULL),
                      (dict(token_stride=1028), w4.EALIGN)):
        assert call(q=_structs(pk, q=bad)[1]) == code, bad
    kv = _structs(pk, kv=dict(batch=33, max_pages=2 ** 26))[0]  # tiles that 31 bits do not number
    assert call(kv=kv) == w4.ERANGE
    kv = _structs(pk, kv=dict(batch=1 << 22))[0]  # rows past a launch
    assert call(kv=kv) == w4.ERANGE


def test_python_layer_refuses(pk):
    import torch

    k, v = pk.empty_cache(4, 16, 2, 128, torch.bfloat16, device="cpu")
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        pk.decode_shared(torch.zeros(3, 8, 128, dtype=torch.bfloat16), k, v, tables, lens, lens[:2], lens[:1])
