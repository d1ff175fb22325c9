"""Adapters of fewer ranks than the factors hold, beside rows that are not finite."""
import pytest
import torch

import lora_reference as lr
from test_gpu_lora import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("R", [40, 32, 8])
def test_padding_makes_no_nan_of_inf(dev, dtype, R):
    """A row with an Inf gives what the ranks in use make of it: the padding would add 0 times Inf."""
    from cudalm_w4a16 import lora

    M, K, N = 60, 256, 72
    ranks = torch.tensor([1, min(R, 8), min(R, 13), R, 0, -2], dtype=torch.int32)
    L = len(ranks)
    x, ys, a, b, s, who = _case(31 + R, M, K, [N], R, L, dtype, "turn")
    # factors of one sign where the Inf meets them, so that sums over several ranks are Inf and not NaN
    a[0][:, :, 7], b[0][:] = a[0][:, :, 7].abs() + 0.01, b[0].abs() + 0.01
    for i, r in enumerate(ranks.clamp(0, R).tolist()):
        a[0][i, r:], b[0][i, :, r:] = float("nan"), float("inf")
    for m in range(0, 24):  # four rows of each adapter; others stay finite
        x[m, 7] = float("inf") if m % 4 < 3 else float("-inf")
    x[26, 9] = float("nan")
    plan = lora.plan(who.to(dev), L)
    got = lora.add(x.to(dev), ys[0].to(dev), a[0].to(dev), b[0].to(dev), plan, s.to(dev), ranks.to(dev))
    want, tol = lr.added(x, ys[0], a[0], b[0], who, s, ranks)
    used = ranks[who.long()] > 0
    assert want[:24][used[:24]].isinf().all() and want[:24][~used[:24]].isfinite().all()
    assert want[27:].isfinite().all()
    lr.check(got, want, tol, (dtype, R))
