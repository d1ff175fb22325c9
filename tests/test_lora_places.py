"""Adapters' results that would lie over rows that are still read, or over each other, are refused
before any launch."""
import pytest

from test_lora_abi import FAKE, _projs

X = FAKE + (7 << 20)
Y0, Y1 = FAKE, FAKE + (1 << 20)  # of the two projections, 512 columns in rows of 512


@pytest.fixture(scope="module")
def lora():
    from cudalm_w4a16 import lora

    return lora


# what of the second projection, further arguments
PART = [  # its result over a part of its own y, of the other's y and result
    (dict(out=Y1 + 2), {}), (dict(out=Y1 - 2 * 511), {}), (dict(out=Y1 + 2 * 512), {}), (dict(out=Y0 + 2 * 100), {}),
    (dict(out=Y0 + 2 * 512 * 29), {}), (dict(out=Y0 + 2 * 512 * 29 + 2 * 511), {}), (dict(out=Y0 - 2 * 512 * 29 - 2 * 511), {}),
    # inside of x, in its first and last columns; one row of each
    (dict(out=X + 16, out_stride=1024), {}), (dict(out=X + 2 * 1023, out_stride=1024), {}),
    (dict(out=X - 2 * 511, out_stride=1024), {}), (dict(out=X + 2 * 1023, out_stride=600), dict(M=1)),
    (dict(out=Y0 + 2 * 511, out_stride=600), dict(M=1)), (dict(out=Y1 + 2 * 300, out_stride=600), dict(M=1))]


@pytest.mark.parametrize("proj,more", PART)
def test_results_over_parts(lora, w4, proj, more):
    args = dict(p=_projs(lora, 2, **proj), count=2, x=X, xs=1024, K=1024, M=30, rank=16, L=7, type=0, scales=FAKE, ranks=FAKE,
                plan=FAKE, stream=None)
    assert w4.lib().cudalm_lora_add(*{**args, **more}.values()) == w4.EINVAL


def test_another_y_over_the_first_result(lora, w4):
    """The other way round: the first projection's result is given in place, the second one reads it in part."""
    for y in (Y0 + 2, Y0 + 2 * 512 * 29, Y0 - 2 * 500):
        p = _projs(lora, 2, y=y)
        assert w4.lib().cudalm_lora_add(p, 2, X, 1024, 1024, 30, 16, 7, 0, FAKE, FAKE, FAKE, None) == w4.EINVAL
