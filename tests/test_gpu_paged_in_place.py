"""Calls that write a result over the argument that it follows from: the new
lengths of eviction, the accepted tokens of verification."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def test_evict_writes_new_lens_over_lens(dev):
    """1200 (sequence, head) pairs, more than run at once: every head selects among all of its
    sequence's tokens, whichever of them is done first."""
    from cudalm_w4a16 import paged_kv as pk

    kv, P, keep = 8, 16, 40
    lens = [(53 * i * i + 29 * i) % 301 for i in range(150)]
    c = ref.Cache(51, lens, kv, 64, P, "bf16", dev)
    k, v, tables, tl = c.upload()
    w = torch.rand(c.num_pages, kv, P, generator=torch.Generator().manual_seed(52)).to(dev)
    dst = torch.full((150, 3), -1, dtype=torch.int32, device=dev)  # (nothing is copied)
    kept, new_lens = pk.evict(k, v, tables, tl, w, dst, keep, 4, 8, new_lens=tl)
    assert new_lens is tl
    assert tl.tolist() == [min(n, keep) for n in lens]
    kept, w = kept.cpu(), w.cpu()
    for b, n in enumerate(lens):
        t = torch.arange(n)
        ww = w[c.tables[b, t // P].long(), :, t % P] if n else torch.empty(0, kv)
        for h in range(kv):
            x = ref.evict_kept(ww[:, h].tolist(), [True] * n, keep, 4, 8)
            assert kept[b, h].tolist() == x + [-1] * (keep - len(x)), (b, h, n)


@pytest.mark.parametrize("certain", [False, True])
def test_verify_writes_accepted_over_counts(dev, certain):
    """600 sequences with several workgroups each read the counts that become what was accepted."""
    from cudalm_w4a16 import draft

    g = torch.Generator(device=dev).manual_seed(53)
    B, G, V = 600, 6, 13000
    p = torch.softmax(torch.randn(B, G + 1, V, device=dev, generator=g) * 2, 2)
    q = None if certain else torch.softmax(p[:, :G].log() + 0.4 * torch.randn(B, G, V, device=dev, generator=g), 2)
    x = p[:, :G].argmax(2).to(torch.int32)
    u, un = torch.rand(B, G, device=dev, generator=g), torch.rand(B, device=dev, generator=g)
    counts = torch.randint(0, G + 1, (B,), device=dev, generator=g, dtype=torch.int32)
    out, n = draft.verify(p, q, x, u, un, counts=counts)
    torch.cuda.synchronize()
    assert bool((n < counts).any()) and bool((n == counts).any())
    again, same = draft.verify(p, q, x, u, un, counts=counts, accepted=counts)
    assert same is counts and torch.equal(counts, n) and torch.equal(again, out)
