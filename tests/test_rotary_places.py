"""Rotated rows that would be written over each other, or over rows that are still read, are
refused before any launch."""
import ctypes

import pytest

from test_paged_abi import FAKE, GOOD_KV
from test_rotary_abi import _plan, _rows


@pytest.fixture(scope="module")
def rot():
    from cudalm_w4a16 import rotary

    return rotary


# heads, out's token and head stride, in heads of 256 channels: two rows share a place
SHARED = [(2, 1, 1), (3, 2, 1), (8, 1, 1), (8, 7, 1), (4, 1, 3), (3, 1, 2)]


@pytest.mark.parametrize("heads,token,head", SHARED)
def test_rows_of_one_place(rot, w4, heads, token, head):
    from cudalm_w4a16 import paged_kv as pk

    lib = w4.lib()
    kv = ctypes.byref(pk.KV(**{**GOOD_KV, "head_dim": 256}))
    for more in (dict(), dict(x=FAKE + (1 << 20), x_token_stride=256 * token, x_head_stride=256 * head)):  # in place
        rows = _rows(rot, heads=heads, out_token_stride=256 * token, out_head_stride=256 * head, **more)
        assert lib.cudalm_rotary_rotate(_plan(rot), rows, 5, 256, 0, FAKE, None) == w4.EINVAL
        assert lib.cudalm_rotary_append(_plan(rot), kv, FAKE + (2 << 20), FAKE + (3 << 20), 512, 256, 512, 256, rows, FAKE,
                                        FAKE, 5, None) == w4.EINVAL


def test_rows_that_others_read(rot, w4):
    """A token or a head further than they are read, or a few channels (where strides are the same)."""
    from cudalm_w4a16 import paged_kv as pk

    lib = w4.lib()
    kv = ctypes.byref(pk.KV(**{**GOOD_KV, "head_dim": 256}))
    append = lambda rows, k=FAKE + (2 << 20), v=FAKE + (3 << 20), stride=2048: lib.cudalm_rotary_append(  # noqa: E731
        _plan(rot), kv, k, v, stride, 256, stride, 256, rows, FAKE, FAKE, 5, None)
    for off in (2 * 2048, 2 * 256, 16, -2 * 2048, -16, 4 * 2 * 2048, 2 * 2048 - 512):
        rows = _rows(rot, x=FAKE, out=FAKE + off)
        assert lib.cudalm_rotary_rotate(_plan(rot), rows, 5, 256, 0, FAKE, None) == w4.EINVAL, off
        assert append(rows) == w4.EINVAL, off
    # queries written over keys or values of the same rows
    out = FAKE + (1 << 20)
    for at in (out, out + 2 * 7 * 256, out + 2 * 2048):
        assert append(_rows(rot), k=at) == w4.EINVAL and append(_rows(rot), v=at) == w4.EINVAL, at
