"""Low-rank adapters of many rows against float64."""
import pytest
import torch

import lora_reference as lr

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _case(seed, M, K, Ns, R, L, dtype, index):
    g = torch.Generator().manual_seed(seed)
    t = DT[dtype]
    x = torch.randn(M, K, generator=g).to(t)
    a = [(torch.randn(L, R, K, generator=g) * K ** -0.5).to(t) for _ in Ns]
    b = [torch.randn(L, n, R, generator=g).to(t) for n in Ns]
    ys = [torch.randn(M, n, generator=g).to(t) for n in Ns]
    s = torch.rand(L, generator=g) * 3 - 1
    if index == "each":
        who = torch.randint(-1, L, (M,), generator=g)
    elif index == "prompts":
        who = torch.sort(torch.randint(-1, L, (M,), generator=g)).values.roll(M // 3)
    elif index == "one":
        who = torch.full((M,), L - 1)
    elif index == "none":
        who = torch.where(torch.arange(M) % 2 == 0, -7, 2 ** 31 - 1)
    else:
        who = torch.arange(M) % L
    return x, ys, a, b, s, who.to(torch.int32)


# M, K, Ns, rank, adapters, type, which adapters
CASES = [(1, 1024, [4096, 512, 512], 16, 8, "bf16", "one"), (1, 128, [16], 8, 1, "f16", "one"),
         (64, 1024, [512, 128], 16, 48, "bf16", "each"), (33, 1024, [640, 640], 64, 6, "f16", "each"),
         (17, 3584, [1024], 32, 5, "bf16", "turn"), (300, 512, [272], 32, 3, "bf16", "prompts"),
         (1000, 256, [128, 64], 8, 9, "f16", "prompts"), (40, 136, [24], 24, 3, "bf16", "each"),
         (21, 8, [7], 8, 4, "bf16", "each"), (50, 264, [33, 1, 130], 40, 7, "f16", "each"),
         (5, 128, [48], 256, 2, "bf16", "turn"), (18, 256, [96], 200, 2, "f16", "each"),
         (9, 128, [64], 16, 4, "bf16", "none"), (200, 128, [32], 16, 1, "f16", "one"),
         (130, 128, [16] * 8, 16, 130, "bf16", "turn"), (400, 64, [40], 8, 4096, "bf16", "each")]


@pytest.mark.parametrize("M,K,Ns,R,L,dtype,index", CASES)
@pytest.mark.parametrize("place", ["ys", "outs"])
def test_add(dev, M, K, Ns, R, L, dtype, index, place):
    from cudalm_w4a16 import lora

    x, ys, a, b, s, who = _case(M + K + R, M, K, Ns, R, L, dtype, index)
    plan = lora.plan(who.to(dev), L)
    d = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    yd = d(ys)
    outs = [torch.full_like(y, float("nan")) for y in yd] if place == "outs" else None
    got = lora.add(x.to(dev), yd, d(a), d(b), plan, scales=s.to(dev), outs=outs)
    for j in range(len(Ns)):
        want, tol = lr.added(x, ys[j], a[j], b[j], who, s)
        lr.check(got[j], want, tol, j)
        none = (who < 0) | (who >= L)
        assert torch.equal(got[j][none.to(dev)].cpu(), ys[j][none]), "rows of no adapter"
        if outs:
            assert got[j] is outs[j] and torch.equal(yd[j].cpu(), ys[j])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_ranks_hide_the_padding(dev, dtype):
    """Rows of A and columns of B past an adapter's rank may hold anything; rank 0 is no adapter at all."""
    from cudalm_w4a16 import lora

    M, K, L, R = 60, 256, 6, 40
    x, ys, a, b, s, who = _case(9, M, K, [72], R, L, dtype, "each")
    ranks = torch.tensor([8, 40, 0, 13, 400, -3], dtype=torch.int32)
    for i, r in enumerate([8, 40, 0, 13, 40, 0]):
        a[0][i, r:] = float("nan")
        b[0][i, :, r:] = float("inf") if i % 2 else float("nan")
    plan = lora.plan(who.to(dev), L)
    got = lora.add(x.to(dev), ys[0].to(dev), a[0].to(dev), b[0].to(dev), plan, s.to(dev), ranks.to(dev))
    want, tol = lr.added(x, ys[0], a[0], b[0], who, s, ranks)
    assert want.isfinite().all()
    lr.check(got, want, tol, "ranks")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_inf_and_nan_stay_with_their_rows(dev, dtype):
    """Of a row's activations, and of an adapter's factors, in the rows that have it."""
    from cudalm_w4a16 import lora

    M, K, L, R = 48, 128, 5, 16
    x, ys, a, b, s, who = _case(11, M, K, [64], R, L, dtype, "turn")
    x[3, 7], x[14, 9] = float("inf"), float("nan")
    a[0][1, 2, 5] = float("inf")
    b[0][2, 11, 3] = float("-inf")
    b[0][0, 1, 4] = float("nan")
    ys[0][40, 2] = float("inf")
    plan = lora.plan(who.to(dev), L)
    got = lora.add(x.to(dev), ys[0].to(dev), a[0].to(dev), b[0].to(dev), plan, s.to(dev))
    want, tol = lr.added(x, ys[0], a[0], b[0], who, s)
    assert want.isinf().any() and want.isnan().any() and want.isfinite().sum() > 1500
    lr.check(got, want, tol, dtype)


def test_large_sums_of_fp16(dev):
    """A x past fp16's range, brought back by small factors of B, and the other way round."""
    from cudalm_w4a16 import lora

    x, ys, a, b, s, who = _case(12, 20, 512, [96], 16, 3, "f16", "each")
    for big in (600.0, 2.0 ** -12):
        xs, bs = (x.float() * big).half(), [(b[0].float() / (40 * big)).half()]
        a2 = [(a[0].float() * 40).half()]
        plan = lora.plan(who.to(dev), 3)
        got = lora.add(xs.to(dev), ys[0].to(dev), a2[0].to(dev), bs[0].to(dev), plan, s.to(dev))
        want, tol = lr.added(xs, ys[0], a2[0], bs[0], who, s)
        lr.check(got, want, tol, big)


def test_strides_and_no_scales(dev):
    """Rows apart by more than they are long; results beside each other in one tensor; odd bases."""
    from cudalm_w4a16 import lora

    M, K, L, R = 37, 192, 4, 24
    x, ys, a, b, _, who = _case(13, M, K, [48, 30], R, L, "bf16", "each")
    plan = lora.plan(who.to(dev), L)
    xs = torch.full((M, 2 * K), float("nan"), dtype=x.dtype, device=dev)
    xs[:, 8:K + 8] = x.to(dev)
    both = torch.full((M, 90), 3.0, dtype=x.dtype, device=dev)
    both[:, 1:49], both[:, 50:80] = ys[0].to(dev), ys[1].to(dev)
    lora.add(xs[:, 8:K + 8], [both[:, 1:49], both[:, 50:80]], [t.to(dev) for t in a], [t.to(dev) for t in b], plan)
    for j, got in enumerate((both[:, 1:49], both[:, 50:80])):
        want, tol = lr.added(x, ys[j], a[j], b[j], who)
        lr.check(got, want, tol, j)
    rest = both.clone()
    rest[:, 1:49] = rest[:, 50:80] = 3.0
    assert (rest == 3).all(), "written beside the rows"


def test_a_row_does_not_depend_on_the_others(dev):
    """The same row alone, in another order of the batch, and through a plan made again."""
    from cudalm_w4a16 import lora

    M, K, L = 90, 1024, 7
    x, ys, a, b, s, who = _case(14, M, K, [256], 16, L, "bf16", "each")
    xd, yd, ad, bd, sd = x.to(dev), ys[0].to(dev), a[0].to(dev), b[0].to(dev), s.to(dev)
    out = torch.empty_like(yd)
    plan = lora.plan(who.to(dev), L)
    first = lora.add(xd, yd, ad, bd, plan, sd, outs=out).clone()
    lora.plan(who.to(dev), L, out=plan)
    assert torch.equal(lora.add(xd, yd, ad, bd, plan, sd, outs=out), first)
    perm = torch.randperm(M, generator=torch.Generator().manual_seed(2))
    other = lora.add(xd[perm.to(dev)], yd[perm.to(dev)], ad, bd, lora.plan(who[perm].to(dev), L), sd)
    assert torch.equal(other.cpu(), first[perm.to(dev)].cpu())
    for m in (0, 41, 89):
        one = lora.add(xd[m:m + 1], yd[m:m + 1], ad, bd, lora.plan(who[m:m + 1].to(dev), L), sd, outs=torch.empty_like(yd[:1]))
        assert torch.equal(one[0], first[m])


def test_captured_with_other_rows(dev):
    """Plan and sums in a graph, replayed with other adapters between eager calls; a side stream."""
    from cudalm_w4a16 import lora

    M, K, L = 40, 256, 9
    x, ys, a, b, s, who = _case(15, M, K, [128, 72], 16, L, "bf16", "each")
    d = lambda ts: [t.to(dev) for t in ts]  # noqa: E731
    xd, yd, ad, bd, sd, wd = x.to(dev), d(ys), d(a), d(b), s.to(dev), who.to(dev)
    outs = [torch.empty_like(y) for y in yd]
    plan = lora.plan(wd, L)

    def call(stream=None):
        lora.plan(wd, L, out=plan, stream=stream)
        return lora.add(xd, yd, ad, bd, plan, sd, outs=outs, stream=stream)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    g = torch.Generator(device=dev).manual_seed(1)
    for i in range(4):
        xd.normal_(generator=g)
        wd.random_(-1, L, generator=g)
        expect = [t.clone() for t in call()]
        torch.cuda.synchronize()
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(expect, outs)), i
        side = torch.cuda.Stream()
        for t in outs:
            t.zero_()
        side.wait_stream(torch.cuda.current_stream())
        call(side)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(expect, outs)), ("side", i)


def test_no_rows(dev):
    from cudalm_w4a16 import lora

    plan = lora.plan(torch.empty(0, dtype=torch.int32, device=dev), 3)
    y = torch.empty(0, 32, dtype=torch.bfloat16, device=dev)
    a, b = torch.empty(3, 8, 64, dtype=y.dtype, device=dev), torch.empty(3, 32, 8, dtype=y.dtype, device=dev)
    assert lora.add(torch.empty(0, 64, dtype=y.dtype, device=dev), y, a, b, plan) is y
