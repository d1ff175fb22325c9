"""Interface checks of rotary positions that need no GPU: the library exports what the
header declares, the Python structs match, and calls that cannot be served are refused
before any HIP call."""
import ctypes
import os
import re
import subprocess

import pytest

from test_paged_abi import BAD_KV, FAKE, GOOD_KV

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rot():
    from cudalm_w4a16 import rotary

    return rotary


@pytest.fixture(scope="module")
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


def test_library_exports_every_declared_symbol(w4, rot):
    text = open(os.path.join(REPO, "include", "cudalm_rotary.h")).read()
    syms = set(re.findall(r"\b(cudalm_[a-z0-9_]+)\s*\(", text)) - {"cudalm_paged_append"}
    assert syms == set(rot.EXPORTED_SYMBOLS)
    assert all(hasattr(w4.lib(), s) for s in syms)


def test_struct_layouts(tmp_path, rot):
    pairs = [("cudalm_rotary", rot.Plan), ("cudalm_rotary_rows", rot.Rows)]
    src = '#include "cudalm_rotary.h"\n#include <cstddef>\n#include <cstdio>\nint main() {\n'
    for name, cls in pairs:
        src += f'  std::printf("%zu", sizeof({name}));\n'
        for f, _t in cls._fields_:
            src += f'  std::printf(" %zu", offsetof({name}, {f}));\n'
        src += '  std::printf("\\n");\n'
    (tmp_path / "use.cpp").write_text(src + "}\n")
    cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-I", os.path.join(REPO, "include"), str(tmp_path / "use.cpp"),
           "-o", str(tmp_path / "use")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([str(tmp_path / "use")], capture_output=True, text=True, timeout=120)
    for line, (_, cls) in zip(out.stdout.splitlines(), pairs):
        assert [int(x) for x in line.split()] == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _t in cls._fields_]
    p = rot.Plan.from_buffer_copy(rot._pack_plan(1, 2, 3, 4, 5, 6, 7, 8, 9, 0.5))
    assert (p.freqs, p.pairs, p.adjacent, p.axes, list(p.sections), p.turns, p.scale) == (1, 2, 3, 4, [5, 6, 7, 8], 9, 0.5)
    r = rot.Rows.from_buffer_copy(rot._pack_rows(1, 2, 3, 4, 5, 6, 7))
    assert [getattr(r, f) for f, _t in rot.Rows._fields_] == [1, 2, 3, 4, 5, 6, 7]


def _plan(rot, sections=(11, 11, 10, 0), **bad):
    p = rot.Plan(**{**dict(freqs=FAKE, pairs=32, adjacent=0, axes=3, turns=1, scale=1.0), **bad})
    for i, n in enumerate(sections):
        p.sections[i] = n
    return ctypes.byref(p)


def _rows(rot, **bad):
    return ctypes.byref(rot.Rows(**{**dict(x=FAKE, out=FAKE + (1 << 20), x_token_stride=2048, x_head_stride=256,
                                           out_token_stride=2048, out_head_stride=256, heads=8), **bad}))


BAD_PLAN = [(dict(pairs=0), "EINVAL"), (dict(pairs=257), "EINVAL"), (dict(axes=0), "EINVAL"), (dict(axes=5), "EINVAL"),
            (dict(adjacent=2), "EINVAL"), (dict(turns=-1), "EINVAL"), (dict(sections=(11, 11, 11, 0)), "EINVAL"),
            (dict(sections=(40, -8, 0, 0)), "EINVAL"), (dict(freqs=None), "ENULL"), (dict(freqs=FAKE + 2), "EALIGN")]


@pytest.mark.parametrize("bad,code", BAD_PLAN)
def test_bad_plan_is_refused_by_both_calls(rot, pk, w4, bad, code):
    lib, want = w4.lib(), getattr(w4, code)
    assert lib.cudalm_rotary_rotate(_plan(rot, **bad), _rows(rot), 5, 256, 0, FAKE, None) == want
    kv = ctypes.byref(pk.KV(**{**GOOD_KV, "head_dim": 256}))
    assert lib.cudalm_rotary_append(_plan(rot, **bad), kv, FAKE, FAKE, 512, 256, 512, 256, _rows(rot), FAKE, FAKE, 5,
                                    None) == want


def test_rotate_refusals(rot, w4):
    lib = w4.lib()
    call = lambda plan=None, rows=None, T=5, D=256, t=0, p=FAKE: lib.cudalm_rotary_rotate(  # noqa: E731
        plan or _plan(rot), rows or _rows(rot), T, D, t, p, None)
    assert call(T=-1) == w4.EINVAL and call(D=63) == w4.EINVAL and call(D=513) == w4.EINVAL
    assert call(t=2) == w4.EINVAL and call(rows=_rows(rot, heads=-1)) == w4.EINVAL
    assert call(rows=_rows(rot, out=FAKE, out_head_stride=264)) == w4.EINVAL  # in place, elsewhere
    # rows that would be written to one place
    assert call(rows=_rows(rot, out_head_stride=0)) == w4.EINVAL and call(rows=_rows(rot, out_token_stride=255)) == w4.EINVAL
    assert call(T=0) == w4.OK and call(rows=_rows(rot, heads=0)) == w4.OK
    assert call(rows=_rows(rot, x=None)) == w4.ENULL and call(rows=_rows(rot, out=None)) == w4.ENULL
    assert call(p=None) == w4.ENULL and call(p=FAKE + 2) == w4.EALIGN
    assert call(rows=_rows(rot, x=FAKE + 1)) == w4.EALIGN
    assert call(T=2 ** 31 - 1) == w4.ERANGE
    assert lib.cudalm_rotary_rotate(None, _rows(rot), 5, 256, 0, FAKE, None) == w4.ENULL
    assert lib.cudalm_rotary_rotate(_plan(rot), None, 5, 256, 0, FAKE, None) == w4.ENULL


@pytest.mark.parametrize("bad,code", [b for b in BAD_KV if "head_dim" not in b[0]])
def test_append_refuses_a_bad_cache(rot, pk, w4, bad, code):
    kv = ctypes.byref(pk.KV(**{**GOOD_KV, "head_dim": 256, **bad}))
    assert w4.lib().cudalm_rotary_append(_plan(rot), kv, FAKE, FAKE, 512, 256, 512, 256, _rows(rot), FAKE, FAKE, 5,
                                         None) == getattr(w4, code)


def test_append_refusals(rot, pk, w4):
    lib = w4.lib()
    kv = ctypes.byref(pk.KV(**{**GOOD_KV, "head_dim": 256}))
    call = lambda plan=None, kv=kv, k=FAKE, v=FAKE, s=(512, 256, 512, 256), q=_rows(rot), p=FAKE, cu=FAKE, n=5: (  # noqa: E731
        lib.cudalm_rotary_append(plan or _plan(rot), kv, k, v, *s, q, p, cu, n, None))
    assert call(n=-1) == w4.EINVAL and call(cu=None, n=5) == w4.EINVAL
    assert call(plan=_plan(rot, pairs=36, axes=1)) == w4.EINVAL  # not a multiple of 8
    assert call(plan=_plan(rot, pairs=136, axes=1)) == w4.EINVAL  # more than the head has
    assert call(q=_rows(rot, heads=0)) == w4.EINVAL
    assert call(q=_rows(rot, out=FAKE, out_token_stride=0)) == w4.EINVAL
    assert call(q=_rows(rot, out_head_stride=8)) == w4.EINVAL
    assert call(n=0) == w4.OK
    assert call(k=None) == w4.ENULL and call(v=None) == w4.ENULL
    assert call(q=_rows(rot, x=None)) == w4.ENULL and call(q=_rows(rot, out=None)) == w4.ENULL
    assert call(k=FAKE + 2) == w4.EALIGN and call(cu=FAKE + 2) == w4.EALIGN and call(p=FAKE + 1) == w4.EALIGN
    assert call(q=_rows(rot, x=FAKE + 8)) == w4.EALIGN and call(q=_rows(rot, out_head_stride=260)) == w4.EALIGN
    for i in range(4):
        s = [512, 256, 512, 256]
        s[i] += 4
        assert call(s=s) == w4.EALIGN
    assert call(n=2 ** 31 - 1) == w4.ERANGE and call(q=_rows(rot, heads=1 << 22)) == w4.ERANGE


def test_python_layer_refuses(rot):
    import torch

    with pytest.raises(ValueError):
        rot.Rotary(torch.zeros(32))  # not on a GPU
    f = rot.frequencies(32, 1e4, device="cpu")
    assert f.dtype == torch.float32 and f[0] == 1 and abs(float(f[16]) - 0.01) < 1e-9
    r = rot.Rotary.__new__(rot.Rotary)
    r.index, r.axes, r.pairs = 0, 1, 32
    with pytest.raises(ValueError):
        rot.rotate(torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32), r)
    with pytest.raises(ValueError):
        rot.rotate(torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), r)
