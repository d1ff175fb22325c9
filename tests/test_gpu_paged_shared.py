"""Decode for groups of sequences that begin with the same tokens, against float64 and
against decode."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


class Shared:
    """A cache in which the sequences of group g (cu[g] .. cu[g + 1] - 1) have their first shared[g]
    tokens from the group's first one. others: what the tables of the further sequences hold for
    whole shared pages: the same pages, none, or pages of NaN."""

    def __init__(self, dev, seed, lens, cu, shared, kv, heads, D, page, dtype, Q=1, others="same", absent=(), spare=40):
        c = self.c = ref.Cache(seed, lens, kv, D, page, dtype, dev, absent=absent, spare=spare)
        g = torch.Generator().manual_seed(seed + 1)
        self.k, self.v, self.here = list(c.k), list(c.v), [h.clone() for h in c.here]
        W = c.tables.shape[1]
        free = [p for p in range(c.num_pages) if not (c.tables == p).any()]
        for i, S in enumerate(shared):
            lo, hi = cu[i], cu[i + 1]
            S = max(0, min(S, W * page))
            for b in range(lo + 1, hi):
                n = min(S, lens[b], lens[lo])
                self.k[b], self.v[b] = c.k[b].clone(), c.v[b].clone()
                self.k[b][:n], self.v[b][:n] = c.k[lo][:n], c.v[lo][:n]
                self.here[b][:n] = c.here[lo][:n]
                # past the first one's end: what its last page holds there (the cache's pages are of NaN
                # before tokens are written), and where it has no page, nothing
                held = min(S, lens[b], -(-lens[lo] // page) * page)
                if n < held:
                    self.k[b][n:held] = self.v[b][n:held] = float("nan")
                    self.here[b][n:held] = c.here[lo][n - 1]
                self.here[b][max(n, held):min(S, lens[b])] = False
                for w in range(W):
                    if (w + 1) * page <= S:
                        c.tables[b, w] = {"same": c.tables[lo, w], "none": -1, "nan": free[0]}[others]
                # nothing is uploaded for the shared places: they stay NaN in pages of its own
                c.here[b][:min(S, lens[b])] = False
        self.lens, self.Q = lens, Q
        self.q = torch.randn(len(lens), Q, heads, D, generator=g).to(c.dtype)
        self.cu = torch.tensor(cu, dtype=torch.int32, device=dev)
        self.shared = torch.tensor(shared, dtype=torch.int32, device=dev)

    def check(self, got, scale, window, sinks, what):
        for b, n in enumerate(self.lens):
            pos = torch.arange(n - self.Q, n)
            out, _, mag, big = ref.attention(self.q[b], self.k[b], self.v[b], self.here[b], pos, scale, window, sinks)
            vmax = float(self.v[b].double().abs().nan_to_num(0, 0, 0).max()) if n else 1.0
            dtype = "bf16" if self.c.dtype == torch.bfloat16 else "f16"
            ref.check_out(got[b], out, mag, big, max(n, 1), vmax, dtype, self.c.D, (what, b))


CASES = [
    # lens, cu, shared, kv, heads, D, page, type
    dict(lens=[300, 270, 257, 400], cu=[0, 4], shared=[256], kv=2, heads=8, D=256, page=16, dtype="bf16"),
    dict(lens=[130, 90, 500, 97, 33], cu=[0, 3, 5], shared=[77, 33], kv=2, heads=8, D=128, page=32, dtype="f16"),
    # nothing shared, an empty group, sequences of no group on either side
    dict(lens=[50, 60, 70, 80, 90, 1, 0], cu=[1, 3, 3, 5], shared=[0, 40, 79], kv=1, heads=5, D=64, page=16, dtype="bf16"),
    # sequences that end inside the prefix, and before they begin
    dict(lens=[200, 150, 96, 97, 3, 0], cu=[0, 6], shared=[97], kv=2, heads=2, D=64, page=64, dtype="f16"),
    # drafted tokens; their first ones may lie in the prefix
    dict(lens=[205, 201, 340, 203, 1200], cu=[0, 5], shared=[200], kv=2, heads=16, D=128, page=16, dtype="bf16", Q=5),
    # rows of several workgroups, many tiles of rows per sequence
    dict(lens=[700] * 9 + [650] * 3, cu=[0, 9, 12], shared=[600, 615], kv=1, heads=40, D=64, page=32, dtype="bf16", Q=3),
    # more sequences than a wave has lanes, and groups
    dict(lens=[40 + b for b in range(140)], cu=list(range(0, 141, 2)), shared=[30 + g for g in range(70)], kv=1, heads=4,
         D=64, page=16, dtype="f16"),
    dict(lens=[1100 + 3 * b for b in range(70)], cu=[0, 70], shared=[1024], kv=2, heads=8, D=256, page=64, dtype="bf16"),
    # numbers past the tables' end, below zero
    dict(lens=[64, 64, 50, 20], cu=[0, 2, 4], shared=[1000, -8], kv=1, heads=8, D=128, page=16, dtype="bf16"),
    # a prefix and nothing else but the new token
    dict(lens=[129, 129, 129], cu=[0, 3], shared=[128], kv=4, heads=16, D=128, page=128, dtype="f16"),
    # a long prefix of many parts
    dict(lens=[5000, 4900, 4801], cu=[0, 3], shared=[4800], kv=2, heads=8, D=128, page=64, dtype="bf16"),
    # 64 heads to a key-value head, 16 new tokens: the most rows
    dict(lens=[90, 80], cu=[0, 2], shared=[60], kv=1, heads=64, D=64, page=16, dtype="bf16", Q=16),
]


@pytest.mark.parametrize("others", ["same", "none", "nan"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 0), (40, 35), (500, 4)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_decode_shared(dev, case, window, sinks, others):
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 50 + case, others=others, **CASES[case])
    k, v, tables, lens = t.c.upload()
    q = t.q.to(dev)
    got = pk.decode_shared(q, k, v, tables, lens, t.cu, t.shared, window=window, sinks=sinks)
    t.check(got, t.c.D ** -0.5, window, sinks, others)
    # what is expected of the lengths decides about speed alone
    for expect in (dict(max_shared=1), dict(max_shared=max(1, max(CASES[case]["shared"])), max_len=max(t.lens))):
        again = pk.decode_shared(q, k, v, tables, lens, t.cu, t.shared, window=window, sinks=sinks, **expect)
        t.check(again, t.c.D ** -0.5, window, sinks, (others, expect))


def test_many_groups_some_of_them_empty(dev):
    # bounds: runs of the same one around places 63, 64 and 128; sequences before the first group
    # and behind the last
    cu = [3] * 60 + [5, 8] + [9] * 10 + list(range(10, 66)) + [70] * 5 + list(range(90, 121, 2))
    lens = [20 + b % 31 for b in range(150)]
    shared = [5 + g % 23 for g in range(len(cu) - 1)]
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 77, lens, cu, shared, 1, 2, 64, 16, "bf16")
    k, v, tables, lens = t.c.upload()
    t.check(pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared), 64 ** -0.5, 0, 0, "many groups")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_scales_and_one_token(dev, dtype, scale):
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 7, [120, 200, 77], [0, 3], [75], 2, 6, 64, 16, dtype)
    k, v, tables, lens = t.c.upload()
    one = t.q[:, 0].to(dev)
    got = pk.decode_shared(one, k, v, tables, lens, t.cu, t.shared, scale=scale)
    assert got.shape == one.shape
    t.check(got[:, None], scale, 0, 0, scale)


def test_absent_pages(dev):
    """Of the prefix, for all of the group; of a sequence, for itself."""
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 9, [150, 140, 130, 60], [0, 3], [100], 2, 8, 128, 16, "bf16", absent=[(0, 0), (0, 3), (1, 7), (3, 0), (3, 2)])
    k, v, tables, lens = t.c.upload()
    t.check(pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared), 128 ** -0.5, 0, 0, "absent")
    tables[:, :] = -1
    got = pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared)
    assert (got == 0).all()


@pytest.mark.parametrize("dtype,D", [("bf16", 64), ("f16", 256)])
def test_inf_and_nan(dev, dtype, D):
    """In values that are seen they count whatever their weight; behind the ends of sequences, in hidden
    places and in the further tables' copies of the prefix they do not."""
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 10, [90, 80, 70, 300], [0, 3], [65], 1, 4, D, 16, dtype, others="nan")
    inf, nan = float("inf"), float("nan")
    for b in range(3):
        t.v[b] = t.v[b].clone()
        t.v[b][10, 0, 3], t.v[b][64, 0, 5] = inf, nan
    t.c.v[0][10, 0, 3], t.c.v[0][64, 0, 5] = inf, nan
    t.v[1][75, 0, 7] = -inf
    t.c.v[1] = t.v[1]
    t.v[3][200, 0, 9] = inf
    t.c.v[3] = t.v[3]
    k, v, tables, lens = t.c.upload()
    t.check(pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared), D ** -0.5, 0, 0, "all")
    t.check(pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared, window=20), D ** -0.5, 20, 0, "window")


def test_rows_without_weight(dev):
    """Scores of -inf everywhere give zeros, in a prefix alone they give what the other tokens do."""
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 11, [60, 55], [0, 2], [32], 1, 2, 64, 16, "bf16")
    t.q[:, :, :, 0] = 1.0
    for b in range(2):
        t.k[b][:32, 0, 0] = float("-inf")
    t.c.k[0][:32, 0, 0] = float("-inf")
    k, v, tables, lens = t.c.upload()
    got = pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared)
    t.check(got, 64 ** -0.5, 0, 0, "prefix")
    lens[:] = 32
    assert (pk.decode_shared(t.q.to(dev), k, v, tables, lens, t.cu, t.shared) == 0).all()


def test_strided_queries_and_given_memory(dev):
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 12, [150, 140, 260], [0, 2, 3], [128, 17], 2, 8, 128, 16, "bf16", Q=2)
    k, v, tables, lens = t.c.upload()
    wide = torch.full((3, 2, 12, 160), float("nan"), dtype=t.q.dtype, device=dev)
    q = wide[:, :, 2:10, 16:144]
    q.copy_(t.q.to(dev))
    out = torch.full((3, 2, 8, 128), float("nan"), dtype=t.q.dtype, device=dev)
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8, device=dev)  # NaN as fp32
    got = pk.decode_shared(q, k, v, tables, lens, t.cu, t.shared, out=out, workspace=ws)
    assert got is out
    t.check(got, 128 ** -0.5, 0, 0, "strided")


def test_captured_with_growing_sequences(dev):
    """One graph, replayed as sequences grow and groups change, against the eager call; a side stream."""
    from cudalm_w4a16 import paged_kv as pk

    t = Shared(dev, 13, [400, 390, 380, 370, 360], [0, 5], [256], 2, 8, 128, 16, "bf16")
    k, v, tables, lens = t.c.upload()
    k.nan_to_num_(), v.nan_to_num_()
    q, out = t.q.to(dev), torch.empty_like(t.q, device=dev)
    cu, shared = torch.tensor([0, 5, 5], dtype=torch.int32, device=dev), torch.tensor([256, 0], dtype=torch.int32, device=dev)

    def call(stream=None):
        return pk.decode_shared(q, k, v, tables, lens, cu, shared, max_shared=256, out=out, stream=stream)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        lens += torch.randint(-30, 20, (5,), device=dev, dtype=torch.int32)
        lens.clamp_(0, 400)
        q.normal_()
        if i % 2:
            cu.copy_(torch.tensor([0, 2, 4], dtype=torch.int32))
            shared.copy_(torch.tensor([250, 0], dtype=torch.int32))
        expect = call().clone()
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expect), i
        out.zero_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        call(side)
        side.synchronize()
        assert torch.equal(out, expect), ("side", i)


def test_offsets_past_32_bits(dev):
    """Pages behind 2^31 elements of the cache."""
    from cudalm_w4a16 import paged_kv as pk

    pages, D = 2 ** 31 // (16 * 256) + 64, 256
    k = torch.zeros(pages, 1, 16, D, dtype=torch.float16, device=dev)
    v = torch.zeros(pages, 1, 2, D, 8, dtype=torch.float16, device=dev)
    g = torch.Generator(device=dev).manual_seed(6)
    ids = [pages - 1 - i for i in range(12)]
    small = torch.arange(12, dtype=torch.int32, device=dev)
    for i in ids:
        k[i].normal_(generator=g), v[i].normal_(generator=g)
    kc, vc = k[ids].contiguous(), v[ids].contiguous()
    q = torch.randn(2, 4, D, device=dev, generator=g).half()
    lens = torch.tensor([90, 96], dtype=torch.int32, device=dev)
    cu, shared = torch.tensor([0, 2], dtype=torch.int32, device=dev), torch.tensor([48], dtype=torch.int32, device=dev)
    rows = lambda a: torch.stack([a[:6], torch.cat([a[:3], a[6:9]])]).to(torch.int32).contiguous()  # noqa: E731
    far = rows(torch.tensor(ids, device=dev))
    assert torch.equal(pk.decode_shared(q, k, v, far, lens, cu, shared), pk.decode_shared(q, kc, vc, rows(small), lens, cu, shared))


def test_more_sequences_than_one_list_holds(dev):
    """64 x 4096 sequences and some: against plain decode, two roundings of each apart."""
    from cudalm_w4a16 import paged_kv as pk

    B, D, pages = 64 * 4096 + 130, 64, 40
    g = torch.Generator(device=dev).manual_seed(9)
    k, v = pk.empty_cache(pages, 16, 1, D, torch.bfloat16)
    k.normal_(generator=g), v.normal_(generator=g)
    tables = torch.randint(0, pages, (B, 2), dtype=torch.int32, device=dev, generator=g)
    tables[1000:1040, 0] = tables[1000, 0]
    tables[B - 90:B - 1, 0] = tables[B - 90, 0]
    lens = torch.randint(1, 33, (B,), dtype=torch.int32, device=dev, generator=g)
    q = torch.randn(B, 1, D, device=dev, generator=g).to(torch.bfloat16)
    cu = torch.tensor([1000, 1040, B - 90, B - 1], dtype=torch.int32, device=dev)
    shared = torch.tensor([16, 0, 13], dtype=torch.int32, device=dev)
    got = pk.decode_shared(q, k, v, tables, lens, cu, shared).float()
    want = pk.decode(q, k, v, tables, lens).float()
    # an output's rounding (2^-8 of it) and the weights' (2^-8 of the largest value), of both; scores and
    # exponentials in fp32 are 2^-18 of it or less
    tol = 2 * (2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -17) * float(v.float().abs().max()))
    assert (got - want).abs().le(tol).all()
