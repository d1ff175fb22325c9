"""Low-rank adapters in the forms that the launch chooses for many workgroups, each by the
kernel that runs and its grid: 64 columns per wave, one step of them or several, one, two and
four rank tiles. Against float64, as in test_gpu_lora.py."""
import ctypes
import re

import pytest
import torch

import lora_reference as lr
from launched_kernels import _KernelNodeParams, _runtime
from test_gpu_lora import _case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def lora(dev):
    if torch.cuda.get_device_properties(dev).multi_processor_count != 256:
        pytest.skip("the sizes stand for forms of a 256-CU part")
    from cudalm_w4a16 import lora

    return lora


def _launch(call):
    """(kernel name, workgroups) of the one kernel of call(), recorded and not run."""
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    hip, raw = _runtime(), ctypes.c_void_p(graph.raw_cuda_graph())
    hip.hipKernelNameRefByPtr.restype = ctypes.c_char_p
    n = ctypes.c_size_t(1)
    node = (ctypes.c_void_p * 1)()
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(n)) == 0 and n.value == 1
    assert hip.hipGraphGetNodes(raw, node, ctypes.byref(n)) == 0
    p = _KernelNodeParams()
    assert hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node[0]), ctypes.byref(p)) == 0
    return hip.hipKernelNameRefByPtr(ctypes.c_void_p(p.func), None).decode(), p.grid.x


def _form(launch, M, L, Ns):
    """(rank tiles, halves of 32 columns, steps of them) that a launch stands for."""
    name, grid = launch
    rt, halves = (int(x) for x in re.findall(r"Li(\d+)E", name))
    groups = -(-min(M, -(-M // 16) + (L + 1 if L < M else M)) // 8) * 8
    assert grid % groups == 0
    steps = [s for s in range(1, 200) if groups * sum(-(-n // (256 * halves * s)) for n in Ns) == grid]
    return rt, halves, steps


# M, K, Ns, rank, adapters, type, which adapters; rank tiles, steps
FORMS = [(64, 1024, [4096, 512, 513], 16, 48, "bf16", "each", 1, 1), (64, 1024, [4096, 512, 512], 16, 48, "f16", "each", 1, 1),
         (64, 512, [4104, 520, 512], 32, 48, "bf16", "each", 2, 1), (64, 512, [4096, 500, 520], 24, 48, "f16", "each", 2, 1),
         (64, 264, [4096, 512, 513], 40, 48, "f16", "each", 4, 1), (64, 256, [4096, 520, 512], 200, 48, "bf16", "each", 4, 1),
         (1100, 512, [4104, 2056, 1000], 16, 5, "bf16", "prompts", 1, 2), (1100, 200, [4101, 2000], 8, 5, "f16", "prompts", 1, 2),
         (1100, 512, [9000, 1000], 32, 5, "f16", "prompts", 2, 3), (1100, 136, [9000, 1030], 24, 5, "bf16", "each", 2, 3),
         (1100, 256, [4101, 1000], 64, 5, "bf16", "prompts", 4, 2), (1100, 136, [4104, 2000], 40, 5, "f16", "each", 4, 2),
         (1100, 128, [4096, 2000], 200, 5, "f16", "prompts", 4, 2), (1100, 2048, [3000], 64, 5, "bf16", "prompts", 4, 1)]


@pytest.mark.parametrize("M,K,Ns,R,L,dtype,index,rt,steps", FORMS)
@pytest.mark.parametrize("place", ["ys", "outs"])
def test_add(lora, dev, M, K, Ns, R, L, dtype, index, rt, steps, place):
    x, ys, a, b, s, who = _case(M + K + R, M, K, Ns, R, L, dtype, index)
    who[M // 2] = -1
    plan = lora.plan(who.to(dev), L)
    d = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    yd, xd, ad, bd, sd = d(ys), x.to(dev), d(a), d(b), s.to(dev)
    outs = [torch.full_like(y, float("nan")) for y in yd] if place == "outs" else yd
    got = lora.add(xd, yd, ad, bd, plan, scales=sd, outs=outs)
    none = (who < 0) | (who >= L)
    for j in range(len(Ns)):
        want, tol = lr.added(x, ys[j], a[j], b[j], who, s)
        lr.check(got[j], want, tol, j)
        assert torch.equal(got[j][none.to(dev)].cpu(), ys[j][none]), "rows of no adapter"
    if place == "outs":
        assert all(torch.equal(p.cpu(), q) for p, q in zip(yd, ys))
    form = _form(_launch(lambda: lora.add(xd, yd, ad, bd, plan, scales=sd, outs=outs)), M, L, Ns)
    assert form[:2] == (rt, 2) and steps in form[2], form


@pytest.mark.parametrize("dtype,R", [("bf16", 16), ("f16", 32), ("f16", 40)])
def test_inf_and_nan_stay_with_their_rows(lora, dev, dtype, R):
    """Several steps of 64 columns, ranks of which some are padding, columns that are no multiple of 8."""
    M, K, L, N = 1100, 128, 5, 7003
    x, ys, a, b, s, who = _case(21 + R, M, K, [N], R, L, dtype, "prompts")
    ranks = torch.tensor([R, 8, R - 3, R, 0], dtype=torch.int32)
    for i, r in enumerate(ranks.tolist()):
        a[0][i, r:], b[0][i, :, r:] = float("nan"), float("inf")
    x[5, 7], x[600, 100], x[1099, 3] = float("inf"), float("nan"), float("-inf")
    a[0][3, 2, 5] = float("inf")
    b[0][2, 4000, 3] = float("-inf")
    b[0][0, 7002, 4] = float("nan")
    ys[0][40, 6999] = float("inf")
    plan = lora.plan(who.to(dev), L)
    xd, yd, ad, bd = x.to(dev), ys[0].to(dev), a[0].to(dev), b[0].to(dev)
    out = torch.empty_like(yd)
    got = lora.add(xd, yd, ad, bd, plan, s.to(dev), ranks.to(dev), outs=out)
    want, tol = lr.added(x, ys[0], a[0], b[0], who, s, ranks)
    assert want.isinf().any() and want.isnan().any() and want.isfinite().sum() > 3000000
    lr.check(got, want, tol, dtype)
    form = _form(_launch(lambda: lora.add(xd, yd, ad, bd, plan, outs=out)), M, L, [N])
    assert form[1] == 2 and min(form[2]) > 1, form
