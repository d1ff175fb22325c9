"""Queries and probabilities that are one row per sequence of a longer tensor."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def test_decode_of_the_last_token_of_longer_queries(dev):
    from cudalm_w4a16 import paged_kv as pk

    c = ref.Cache(61, [50, 7, 200], 2, 128, 16, "bf16", dev)
    k, v, tables, tl = c.upload()
    x = torch.randn(3, 5, 8, 128, device=dev).to(k.dtype)
    expect = pk.decode(x[:, -1].contiguous(), k, v, tables, tl)
    assert torch.equal(pk.decode(x[:, -1:], k, v, tables, tl)[:, 0], expect)
    assert torch.equal(pk.decode(x[:, -1], k, v, tables, tl), expect)
    one = pk.decode(x[:1, -1:], k, v, tables[:1], tl[:1])
    assert torch.equal(one[0, 0], expect[0])
