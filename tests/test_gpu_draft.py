"""Verification of drafted tokens against plain whole-number arithmetic: every
output is exact. Refusal at every place, drafts that were certain, tokens
outside the vocabulary, NaN, rows without any probability, vocabularies of 1
and of odd sizes, strides, and the distribution of what comes out."""
import numpy as np
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def draft():
    from cudalm_w4a16 import draft

    return draft


def _check(draft, dev, p, q, tokens, u, u_next, counts=None):
    B, G = tokens.shape
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    out, n = draft.verify(to(p), to(q), to(tokens), to(u), to(u_next), counts=to(counts))
    torch.cuda.synchronize()
    P, Q = p.float().numpy(), None if q is None else q.float().numpy()
    for b in range(B):
        g = G if counts is None else min(max(int(counts[b]), 0), G)
        want, nxt = ref.verify(P[b], None if Q is None else Q[b], tokens[b, :g].tolist(),
                               u[b].numpy(), float(u_next[b]))
        assert int(n[b]) == want, (b, int(n[b]), want)
        assert out[b].tolist() == tokens[b, :want].tolist() + [nxt] + [-1] * (G - want), b


def _case(seed, B, G, V, dtype, certain=False, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(B, G + 1, V, generator=g) * sharp
    p = torch.softmax(l, 2).to(TYPES[dtype])
    q = torch.softmax(l[:, :G] + torch.randn(B, G, V, generator=g) * 0.7, 2)
    tokens = torch.zeros(B, G, dtype=torch.int32)
    if G:
        tokens = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, G).to(torch.int32)
    return (p, None if certain else q.to(TYPES[dtype]), tokens, torch.rand(B, G, generator=g),
            torch.rand(B, generator=g))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,G,V", [(1, 4, 1000), (7, 3, 4096), (5, 1, 4097), (3, 8, 12289), (4, 2, 1), (6, 0, 50),
                                   (9, 5, 7)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(draft, dev, dtype, B, G, V, certain):
    _check(draft, dev, *_case(B + G + V, B, G, V, dtype, certain))


def test_verify_edges(draft, dev):
    p, q, x, u, un = _case(1, 12, 4, 300, "f32")
    un[:4] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, float("nan")])
    x[0, 0], x[1, 2], x[2, 1] = -1, 300, 2 ** 31 - 1  # not in the vocabulary
    q[3, 0] = 0.0  # a draft that gave its token nothing
    p[4] = 0.0  # nothing to draw from
    p[5, 0] *= 0.0
    u[5, 0] = 0.5  # refused, and nothing is left of the target
    p[6] = q[6, 0] * 0.5
    u[6] = 0.9  # refused, and the draft covers all of it: the target's own
    p[7, :, 5] = float("nan")
    u[8] = 0.0
    counts = torch.tensor([4, 4, 4, 4, 4, 4, 4, 4, 4, 0, 2, 9], dtype=torch.int32)
    ref_un = un.clone()
    ref_un[3] = 0.0  # NaN counts as 0
    B = 12
    out, n = draft.verify(p.to(dev), q.to(dev), x.to(dev), u.to(dev), un.to(dev), counts=counts.to(dev))
    for b in range(B):
        g = min(int(counts[b]), 4)
        want, nxt = ref.verify(p[b].numpy(), q[b].numpy(), x[b, :g].tolist(), u[b].numpy(), float(ref_un[b]))
        assert int(n[b]) == want and out[b].tolist() == x[b, :want].tolist() + [nxt] + [-1] * (4 - want), b
    # the same with a draft that was certain
    out, n = draft.verify(p.to(dev), None, x.to(dev), u.to(dev), un.to(dev))
    for b in range(B):
        want, nxt = ref.verify(p[b].numpy(), None, x[b].tolist(), u[b].numpy(), float(ref_un[b]))
        assert int(n[b]) == want and out[b].tolist() == x[b, :want].tolist() + [nxt] + [-1] * (4 - want), b


def test_verify_strided(draft, dev):
    p, q, x, u, un = _case(2, 5, 3, 1001, "bf16")
    wide_p = torch.full((5, 4, 1030), float("nan"), dtype=p.dtype, device=dev)
    wide_q = torch.full((5, 3, 1003), float("nan"), dtype=p.dtype, device=dev)
    wide_p[:, :, :1001], wide_q[:, :, :1001] = p.to(dev), q.to(dev)
    a = draft.verify(wide_p[:, :, :1001], wide_q[:, :, :1001], x.to(dev), u.to(dev), un.to(dev))
    b = draft.verify(p.to(dev), q.to(dev), x.to(dev), u.to(dev), un.to(dev))
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_verify_vocabulary(draft, dev):
    # the model's vocabulary, one token of many with a tiny share each
    p, q, x, u, un = _case(3, 2, 2, 248320, "f32", sharp=0.5)
    u[1, 0] = 0.999999
    _check(draft, dev, p, q, x, u, un)


def test_output_is_distributed_as_the_target(draft, dev):
    """Whatever the draft, the first token that comes out follows the target.
    40000 draws: each share is within 5 standard deviations."""
    B, V = 40000, 6
    p = torch.tensor([0.05, 0.4, 0.0, 0.25, 0.2, 0.1])
    q = torch.tensor([0.3, 0.1, 0.2, 0.05, 0.2, 0.15])
    g = torch.Generator().manual_seed(5)
    x = torch.multinomial(q, B, replacement=True, generator=g).to(torch.int32).view(B, 1)
    u, un = torch.rand(B, 1, generator=g), torch.rand(B, generator=g)
    out, n = draft.verify(p.expand(B, 2, V).contiguous().to(dev), q.expand(B, 1, V).contiguous().to(dev),
                          x.to(dev), u.to(dev), un.to(dev))
    share = torch.bincount(out[:, 0].cpu().long(), minlength=V).double() / B
    assert bool(((share - p).abs() <= 5 * (p.double() * (1 - p.double()) / B).sqrt() + 1e-6).all()), share
    rate = float(n.double().mean())
    want = float(torch.minimum(p, q).sum())
    assert abs(rate - want) <= 5 * np.sqrt(want * (1 - want) / B)


def test_side_stream_and_graph(draft, dev):
    p, q, x, u, un = (t.to(dev) for t in _case(4, 3, 4, 9999, "f32"))
    expect = draft.verify(p, q, x, u, un)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = draft.verify(p, q, x, u, un, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, expect))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = draft.verify(p, q, x, u, un)
    for i in range(3):
        u.uniform_()
        un.uniform_()
        eager = draft.verify(p, q, x, u, un)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i
