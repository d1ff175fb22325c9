"""Interface checks of low-rank adapters that need no GPU: the library exports what the
header declares, the Python struct matches, and calls that cannot be served are refused
before any HIP call."""
import ctypes
import os
import re
import struct
import subprocess

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAKE = 0x100000


@pytest.fixture(scope="module")
def lora():
    from cudalm_w4a16 import lora

    return lora


def test_library_exports_every_declared_symbol(w4, lora):
    text = open(os.path.join(REPO, "include", "cudalm_lora.h")).read()
    assert set(re.findall(r"\b(cudalm_[a-z0-9_]+)\s*\(", text)) - {"cudalm_lora_plan"} == set(lora.EXPORTED_SYMBOLS) - {"cudalm_lora_plan"}
    assert all(hasattr(w4.lib(), s) for s in lora.EXPORTED_SYMBOLS)


def test_struct_layout(tmp_path, lora):
    src = '#include "cudalm_lora.h"\n#include <cstddef>\n#include <cstdio>\nint main() {\n'
    src += '  std::printf("%zu", sizeof(cudalm_lora_proj));\n'
    for f, _t in lora.Proj._fields_:
        src += f'  std::printf(" %zu", offsetof(cudalm_lora_proj, {f}));\n'
    (tmp_path / "use.cpp").write_text(src + "}\n")
    cmd = ["/opt/rocm/bin/hipcc", "-std=c++17", "-I", os.path.join(REPO, "include"), str(tmp_path / "use.cpp"),
           "-o", str(tmp_path / "use")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    out = subprocess.run([str(tmp_path / "use")], capture_output=True, text=True, timeout=120).stdout
    assert [int(x) for x in out.split()] == [ctypes.sizeof(lora.Proj)] + [
        getattr(lora.Proj, f).offset for f, _t in lora.Proj._fields_]
    p = lora.Proj.from_buffer_copy(struct.pack("4P2qi4x", *range(1, 8)))
    assert [getattr(p, f) for f, _t in lora.Proj._fields_] == list(range(1, 8))


def _projs(lora, count=1, **bad):
    arr = (lora.Proj * count)()
    for i in range(count):
        at = FAKE + (i << 20)
        arr[i] = lora.Proj(**dict(a=FAKE, b=FAKE, y=at, out=at, y_stride=512, out_stride=512, N=512))
    for f, v in bad.items():
        setattr(arr[count - 1], f, v)
    return arr


def test_plan_refusals(lora, w4):
    lib = w4.lib()
    need = lib.cudalm_lora_plan_bytes(100, 7)
    assert need > 400
    call = lambda i=FAKE, M=100, L=7, p=FAKE, n=need: lib.cudalm_lora_plan(i, M, L, p, n, None)  # noqa: E731
    assert call(M=-1) == w4.EINVAL and call(L=0) == w4.EINVAL
    assert call(L=4097, n=1 << 40) == w4.ERANGE and call(M=(1 << 22) + 1, n=1 << 40) == w4.ERANGE
    assert call(i=None) == w4.ENULL and call(p=None) == w4.ENULL
    assert call(i=FAKE + 2) == w4.EALIGN and call(p=FAKE + 8) == w4.EALIGN
    assert call(n=need - 1) == w4.ERANGE
    assert lib.cudalm_lora_plan_bytes(-1, 7) == 0 and lib.cudalm_lora_plan_bytes(5, 0) == 0


def test_plan_bytes_hold_every_tile(w4):
    """A tile per 16 rows of an adapter: at most one that is not full for each, and for the rows of none."""
    lib = w4.lib()
    for M in (0, 1, 2, 15, 16, 17, 100, 1000):
        for L in (1, 2, 15, 16, 100, 2000):
            # as many groups of one row as there are, the rest in one
            groups = min(M, L + 1)
            tiles = groups - 1 + -(-(M - groups + 1) // 16) if groups else 0
            assert lib.cudalm_lora_plan_bytes(M, L) >= 16 + (8 + 64) * tiles


def test_add_refusals(lora, w4):
    lib = w4.lib()
    good = dict(p=None, count=2, x=FAKE + (7 << 20), xs=1024, K=1024, M=30, rank=16, L=7, type=0, scales=FAKE, ranks=FAKE, plan=FAKE,
                stream=None)

    def call(proj=(), **bad):
        args = {**good, **bad}
        if "p" not in bad:
            args["p"] = _projs(lora, 2, **dict(proj))
        return lib.cudalm_lora_add(*args.values())

    for bad in (dict(count=0), dict(count=9), dict(K=0), dict(K=1020), dict(M=-1), dict(rank=0), dict(rank=12),
                dict(rank=264), dict(L=0), dict(type=2), dict(proj=dict(N=0)), dict(proj=dict(out_stride=520))):
        assert call(**bad) == w4.EINVAL, bad
    for bad in (dict(p=None), dict(x=None), dict(plan=None), dict(proj=dict(a=None)), dict(proj=dict(b=None)),
                dict(proj=dict(y=None)), dict(proj=dict(out=None))):
        assert call(**bad) == w4.ENULL, bad
    for bad in (dict(x=FAKE + (7 << 20) + 8), dict(xs=1028), dict(plan=FAKE + 4), dict(scales=FAKE + 2),
                dict(ranks=FAKE + 2), dict(proj=dict(a=FAKE + 2)), dict(proj=dict(b=FAKE + 8)),
                dict(proj=dict(y=FAKE + 1)), dict(proj=dict(out=FAKE + 1))):
        assert call(**bad) == w4.EALIGN, bad
    # results where others are read or written
    for bad in (dict(out=FAKE + (7 << 20)), dict(out=FAKE), dict(out_stride=511, out=FAKE + (9 << 20)),
                dict(out_stride=0, out=FAKE + (9 << 20))):
        assert call(proj=bad, x=FAKE + (7 << 20)) == w4.EINVAL, bad
    assert call(L=4097) == w4.ERANGE and call(M=(1 << 22) + 1) == w4.ERANGE
    assert call(proj=dict(N=(1 << 28) + 1, y_stride=1 << 29, out_stride=1 << 29)) == w4.ERANGE
    assert call(M=0) == w4.OK


def test_python_layer_refuses(lora):
    import torch

    with pytest.raises(ValueError):
        lora.plan(torch.zeros(3, dtype=torch.int32), 2)  # not on a GPU
    p = lora.Plan(torch.zeros(3), 3, 2)
    with pytest.raises(ValueError):
        lora.add(torch.zeros(3, 64, dtype=torch.bfloat16), [], [], [], p)
    with pytest.raises(ValueError):
        lora.add(torch.zeros(3, 64), [], [], [], p)
