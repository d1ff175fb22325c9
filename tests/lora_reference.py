"""Low-rank adapters in float64, for their tests."""
import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step relative to the value


def added(x, y, a, b, index, scales=None, ranks=None):
    """One projection, all on the CPU: (values, tolerance) in float64. The tolerance is the
    output's rounding (half a step; 2^-25 below fp16's normal range); of sum_r |b_r| sum_k |a_k x_k|
    the first sum's in fp32 (K 2^-24), what h loses as two bf16 numbers (2^-16 of it) and
    fp16 factors as three products of four (2^-16), the second sum's (4 rank 2^-24 and three for scale
    and sum, all terms twice over)."""
    M, K = x.shape
    R = a.shape[1]
    out, tol = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64)
    near = K * 2.0 ** -24 + 2.0 ** -15 + (8 * R + 6) * 2.0 ** -24
    for m in range(M):
        i = int(index[m])
        if not 0 <= i < a.shape[0]:
            continue
        r = R if ranks is None else min(R, max(0, int(ranks[i])))
        s = 1.0 if scales is None else float(scales[i])
        A, B, v = a[i, :r].double(), b[i, :, :r].double(), x[m].double()
        out[m] += s * (B @ (A @ v))
        size = abs(s) * (B.abs() @ (A.abs() @ v.abs()))
        tol[m] = near * size + 2.0 ** -24 * (y[m].double().abs() + size)
    return out, tol + out.abs() * UNIT[x.dtype] + 2.0 ** -25


def check(got, out, tol, what):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), out.isnan()), (what, "NaN places")
    inf = out.isinf()
    assert torch.equal(got[inf], out[inf]), (what, "infinities")
    bad = ((got - out).abs() > tol) & ~inf & ~out.isnan()
    assert not bad.any(), (what, int(bad.sum()), float((got - out).abs()[bad].max()))
