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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_of_one_row_of_longer_probabilities(dev, dtype):
    from cudalm_w4a16 import draft

    g = torch.Generator(device=dev).manual_seed(62)
    p = torch.softmax(torch.randn(4, 6, 5001, device=dev, generator=g) * 2, 2).to(dtype)
    q = torch.softmax(torch.randn(4, 5, 5001, device=dev, generator=g) * 2, 2).to(dtype)
    x = torch.randint(0, 5001, (4, 1), dtype=torch.int32, device=dev, generator=g)
    u, un = torch.rand(4, 1, device=dev, generator=g) * 0.5, torch.rand(4, device=dev, generator=g)
    none = x[:, :0]
    two = p[:, :2].contiguous()
    for target, probs, tokens in ((p[:, :1], None, none), (p[:, :1], q[:, :0], none), (two, q[:, :1], x)):
        got = draft.verify(target, probs, tokens, u[:, :tokens.shape[1]], un)
        expect = draft.verify(target.contiguous(), None if probs is None else probs.contiguous(), tokens,
                              u[:, :tokens.shape[1]].contiguous(), un)
        assert all(torch.equal(a, b) for a, b in zip(got, expect))
