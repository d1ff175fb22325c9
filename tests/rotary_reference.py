"""Rotary positions in float64, for their tests."""
import torch

# a rounding's largest error relative to the value, half a step: 8 (11) bits of significand, steps of
# 2^-7 (2^-10) at 1
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def axis_of(pairs, sections, turns):
    """Axis of every pair."""
    if not turns:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while len(out) < pairs:
        for a in range(len(sections)):
            if left[a] > 0:
                left[a] -= 1
                out.append(a)
    return out


def rotated(x, positions, freqs, sections, turns, adjacent, scale=1.0):
    """x [T, heads, D] (CPU) by positions [axes, T]: (values, tolerance), float64. The
    tolerance is the output's rounding (half a step of the result, 2^-25 below fp16's
    normal range), and of each of the two inputs 2^-21: the reduced angle's rounding (pi
    2^-25), the sine's last places (2^-22), a product's and the sum's (2^-23)."""
    pairs, f = len(freqs), freqs.double()
    axis = axis_of(pairs, sections, turns)
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    for i in range(pairs):
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + pairs)
        w = positions[axis[i]].double() * f[i]
        c, s = torch.cos(w)[:, None] * scale, torch.sin(w)[:, None] * scale
        x0, x1 = x[:, :, a].double(), x[:, :, b].double()
        y[:, :, a], y[:, :, b] = x0 * c - x1 * s, x1 * c + x0 * s
        near = (x0.abs() + x1.abs()) * abs(scale) * 2.0 ** -21
        for ch in (a, b):
            tol[:, :, ch] = near * 1.01 + y[:, :, ch].abs() * UNIT[x.dtype] + 2.0 ** -25
    return y, tol


def check(got, y, tol, what):
    got = got.double().cpu()
    bad = ~((got - y).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got - y).abs()[bad].max()))
