"""Decode with shared prefixes where a sequence has more rows (new tokens times query heads of a
key-value head) than one tile: two tiles of 16, four, and more than one round of four, each by the kernel
that runs. Against float64, as in test_gpu_paged_shared.py."""
import re

import pytest
import torch

from launched_kernels import launched_kernels
from test_gpu_paged_shared import Shared

pytestmark = pytest.mark.gpu

# new tokens, query heads of a key-value head, tiles of rows that have a wave each
ROWS = [(1, 17, 2), (5, 4, 2), (2, 16, 2), (3, 11, 4), (3, 16, 4), (5, 13, 4), (5, 16, 4)]


def _tiles(names, D):
    found = [re.findall(r"Li(\d+)E", n) for n in names if "paged_shared_kernel" in n]
    assert len(found) == 1 and int(found[0][0]) == D, names
    return int(found[0][1])


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 35)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("Q,group,rt", ROWS)
def test_rows(dev, Q, group, rt, dtype, D, window, sinks):
    """Two groups and a sequence of none; sequences that end inside the prefix; lengths of a new token
    alone and of none at all."""
    from cudalm_w4a16 import paged_kv as pk

    kv = 2 if group == 4 else 1
    t = Shared(dev, Q + group + D, [150, 131, 90, 203, 77, 1, 0], [0, 3, 5], [129, 33], kv, kv * group, D, 16, dtype, Q=Q,
               others="nan")
    k, v, tables, lens = t.c.upload()
    q = t.q.to(dev)
    call = lambda: pk.decode_shared(q, k, v, tables, lens, t.cu, t.shared, window=window, sinks=sinks)  # noqa: E731
    t.check(call(), D ** -0.5, window, sinks, "rows")
    assert _tiles(launched_kernels(call), D) == rt


@pytest.mark.parametrize("D,dtype,Q,group,rt", [(256, "bf16", 5, 4, 2), (128, "f16", 2, 16, 2), (64, "bf16", 1, 20, 2),
                                                (256, "f16", 3, 16, 4), (128, "bf16", 5, 13, 4), (64, "f16", 3, 11, 4)])
def test_ranges_of_many_tiles(dev, D, dtype, Q, group, rt):
    """More own tiles than ranges: a range is several tiles, of one segment or of two."""
    from cudalm_w4a16 import paged_kv as pk

    B = 24
    lens = [900 + (b * 131) % 800 for b in range(B)]
    t = Shared(dev, D + rt, lens, [0, 9, B], [70, 45], 2, 2 * group, D, 32, dtype, Q=Q)
    k, v, tables, tl = t.c.upload()
    q = t.q.to(dev)
    call = lambda: pk.decode_shared(q, k, v, tables, tl, t.cu, t.shared, max_shared=70)  # noqa: E731
    got = call()
    t.check(got, D ** -0.5, 0, 0, "many")
    assert _tiles(launched_kernels(call), D) == rt
    # shorter expectations: fewer ranges, of more tiles each
    again = pk.decode_shared(q, k, v, tables, tl, t.cu, t.shared, max_shared=70, max_len=100)
    t.check(again, D ** -0.5, 0, 0, "expected short")


@pytest.mark.parametrize("dtype,D,Q,group,rt", [("bf16", 256, 5, 4, 2), ("f16", 128, 2, 16, 2), ("f16", 256, 5, 13, 4),
                                                ("bf16", 64, 3, 16, 4)])
def test_inf_and_nan(dev, dtype, D, Q, group, rt):
    """In the prefix, in own tokens, in the new tokens that only the later ones see; behind a window."""
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 60 + D, [120, 110, 100, 300], [0, 3], [65], 1, group, D, 16, dtype, Q=Q, others="nan")
    inf, nan = float("inf"), float("nan")
    for b in range(3):
        t.v[b] = t.v[b].clone()
        t.v[b][10, 0, 3], t.v[b][64, 0, 5] = inf, nan
    t.c.v[0][10, 0, 3], t.c.v[0][64, 0, 5] = inf, nan
    t.v[1][109, 0, 7], t.v[1][105, 0, 8] = -inf, inf
    t.c.v[1] = t.v[1]
    t.v[3][200, 0, 9], t.v[3][299, 0, 11] = inf, nan
    t.c.v[3] = t.v[3]
    k, v, tables, lens = t.c.upload()
    q = t.q.to(dev)
    call = lambda w=0: pk.decode_shared(q, k, v, tables, lens, t.cu, t.shared, window=w)  # noqa: E731
    t.check(call(), D ** -0.5, 0, 0, "all")
    t.check(call(20), D ** -0.5, 20, 0, "window")
    assert _tiles(launched_kernels(call), D) == rt
