"""The paged cache's calls and draft verification on the default stream by its
raw handle, 0: results are those of the plain call, in memory of that stream."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def test_default_stream_by_handle(dev):
    from cudalm_w4a16 import draft, paged_kv as pk

    c = ref.Cache(31, [1500, 90], 2, 64, 16, "bf16", dev, spare=60)
    k, v, tables, tl = c.upload()
    q = torch.randn(2, 8, 64, device=dev).to(k.dtype)
    qp = torch.randn(40, 8, 64, device=dev).to(k.dtype)
    cu = torch.tensor([0, 25, 40], dtype=torch.int32, device=dev)
    w = torch.rand(c.num_pages, 2, 16, device=dev)
    dst = torch.full((2, 2), -1, dtype=torch.int32, device=dev)  # (nothing is copied)
    p = torch.softmax(torch.randn(3, 5, 9000, device=dev), 2)
    d = torch.softmax(torch.randn(3, 4, 9000, device=dev), 2)
    x = torch.randint(0, 9000, (3, 4), dtype=torch.int32, device=dev)
    u, un = torch.rand(3, 4, device=dev), torch.rand(3, device=dev)
    handle = torch.cuda.default_stream().cuda_stream
    assert handle == 0

    def calls(stream):
        return [pk.decode(q, k, v, tables, tl, stream=stream), pk.prefill(qp, cu, k, v, tables, tl, stream=stream),
                *pk.evict(k, v, tables, tl, w, dst, 20, stream=stream),
                *draft.verify(p, d, x, u, un, stream=stream)]

    expect = calls(None)
    torch.cuda.synchronize()
    got = calls(handle)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    # what is given back on the default stream is what the next such call gets
    big = torch.empty(7 << 20, dtype=torch.uint8, device=dev)
    at = big.data_ptr()
    del big
    again = pk._empty((7 << 20,), torch.uint8, dev.index or 0, handle)
    assert again.data_ptr() == at
