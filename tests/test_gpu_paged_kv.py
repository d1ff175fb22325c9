"""The paged cache's operators against plain float64 forms, in caches whose
unwritten places hold NaN: lengths of 0 and 1, odd lengths, pages that end
inside a tile, absent pages, windows and sinks that leave rows empty, shared
heads, strided queries, many splits, Inf and NaN in hidden places, side
streams and graphs. Tolerances follow from the roundings (paged_reference.py);
written keys, values and kept positions are exact."""
import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pk():
    from cudalm_w4a16 import paged_kv

    return paged_kv


def _queries(seed, rows, H, D, dtype, dev, fused=False, size=1.0):
    """q [rows, H, D] on the CPU and the GPU, there (fused) every second D of a
    projection that holds a gate beside each head."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(rows, H, D, generator=g) * size).to(ref.DT[dtype])
    if not fused:
        return q, q.to(dev)
    both = torch.full((rows, H, 2 * D), float("nan"), dtype=q.dtype, device=dev)
    both[:, :, :D] = q.to(dev)
    return q, both[:, :, :D]


def _expect(c, b, q, n, scale, window, sinks):
    L = c.lens[b]
    pos = torch.arange(n) + L - n
    return ref.attention(q, c.k[b], c.v[b], c.here[b], pos, scale, window, sinks)


def _check_decode(pk, dev, lens, Q, H, kv, D, P, dtype, window=0, sinks=0, absent=(), weights=None,
                  max_len=None, fused=False, scale=None, seed=0, size=1.0, change=None):
    c = ref.Cache(seed + 17 * D + P, lens, kv, D, P, dtype, dev, absent)
    if change:
        change(c)
    k, v, tables, tl = c.upload()
    q, qd = _queries(seed + 5, len(lens) * Q, H, D, dtype, dev, fused, size)
    qd = qd.unflatten(0, (len(lens), Q))
    w = None
    if weights:
        w = torch.full((c.num_pages, kv, P), 0.25, device=dev)
    out = torch.full((len(lens), Q, H, D), float("nan"), dtype=q.dtype, device=dev)
    pk.decode(qd, k, v, tables, tl, scale=scale, window=window, sinks=sinks, weights=w,
              accumulate=weights == "add", max_len=max_len, out=out)
    torch.cuda.synchronize()
    s = D ** -0.5 if scale is None else scale
    want = torch.full((c.num_pages, kv, P), 0.25, dtype=torch.float64)
    for b, L in enumerate(lens):
        o, ww, mag, big = _expect(c, b, q[b * Q:(b + 1) * Q], Q, s, window, sinks)
        vmax = float(c.v[b].double().nan_to_num(0, 0, 0).abs().max()) if L else 0.0
        ref.check_out(out[b], o, mag, big, L, vmax, dtype, D, ("decode", b, L))
        if w is not None and L:
            t = torch.arange(L)[c.here[b]]
            at = c.tables[b, t // P].long()
            base = 0.25 if weights == "add" else 0.0
            ref.check_weights(w.cpu()[at, :, t % P].t() - base, ww[:, t], big + 4, Q * H, D,
                              ("weights", b, L))
            want[at, :, t % P] = float("nan")
    if w is not None:
        rest = ~want.isnan()
        assert torch.equal(w.cpu().double()[rest], want[rest]), "weights of other places"


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 100, 257]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (256, 16), (128, 128), (256, 64), (64, 1024)])
def test_decode_lengths(pk, dev, dtype, D, P):
    _check_decode(pk, dev, LENS, 1, 8, 2, D, P, dtype)


@pytest.mark.parametrize("Q,H,kv", [(1, 1, 1), (1, 3, 1), (2, 8, 8), (5, 8, 2), (3, 15, 3), (8, 16, 4),
                                    (1, 64, 1), (4, 32, 2), (8, 20, 2), (17, 8, 2), (2, 128, 2)])
def test_decode_rows(pk, dev, Q, H, kv):
    # rows per key-value head from 1 to 128: one, two and four tiles of 16, two groups of 64
    _check_decode(pk, dev, [0, 1, Q, 40, 131], Q, H, kv, 64, 16, "bf16")
    _check_decode(pk, dev, [3, 77], Q, H, kv, 128, 32, "f16", window=9, sinks=2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (16, 0), (33, 40), (64, 16), (100, 3),
                                          (1000, 5), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("D,P,Q", [(64, 16, 1), (256, 32, 5), (128, 64, 3)])
def test_decode_window(pk, dev, window, sinks, D, P, Q):
    _check_decode(pk, dev, LENS, Q, 8, 2, D, P, "bf16", window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_decode_absent_pages(pk, dev, window, sinks):
    absent = [(0, 1), (0, 2), (1, 0), (2, 3), (3, 0), (3, 1)]
    _check_decode(pk, dev, [100, 70, 64, 32], 2, 8, 2, 128, 16, "bf16", window, sinks, absent)
    _check_decode(pk, dev, [100, 70, 64, 32], 1, 8, 2, 256, 16, "f16", window, sinks, absent,
                  weights="set")


@pytest.mark.parametrize("max_len", [None, 64, 4000])
def test_decode_many_splits(pk, dev, max_len):
    # one sequence over many workgroups; an expected length that is too small
    _check_decode(pk, dev, [3333], 1, 4, 1, 256, 16, "bf16", max_len=max_len)
    _check_decode(pk, dev, [5, 2100], 5, 8, 2, 64, 64, "f16", max_len=max_len)


@pytest.mark.parametrize("mode", ["set", "add"])
@pytest.mark.parametrize("D,P,Q,window,sinks", [(64, 16, 1, 0, 0), (128, 32, 5, 0, 0), (256, 64, 3, 50, 4),
                                                (64, 128, 8, 7, 33)])
def test_decode_weights(pk, dev, mode, D, P, Q, window, sinks):
    _check_decode(pk, dev, [0, 1, 3, 31, 64, 200, 1111], Q, 8, 2, D, P, "bf16", window, sinks,
                  weights=mode)


def test_decode_weights_of_many_rows(pk, dev):
    # 68 and 128 rows: two groups of 64, of which each may have its own parts
    _check_decode(pk, dev, [17, 300, 900], 17, 8, 2, 64, 16, "bf16", weights="set")
    _check_decode(pk, dev, [40, 2000], 2, 64, 1, 64, 32, "f16", 500, 4, weights="add")


def test_decode_strided_and_scale(pk, dev):
    _check_decode(pk, dev, [9, 50], 2, 8, 2, 256, 16, "bf16", fused=True, scale=0.11)
    _check_decode(pk, dev, [9, 50], 1, 8, 2, 128, 16, "f16", fused=True, scale=-0.2)
    _check_decode(pk, dev, [9, 50], 1, 8, 2, 64, 16, "f16", scale=0.0)


def test_decode_large_scores(pk, dev):
    # one token takes all the weight, wherever it stands; maxima rise late
    _check_decode(pk, dev, [400, 37], 2, 4, 2, 128, 16, "bf16", size=60.0, weights="set")

    def rise(c):
        for k in c.k:
            k *= torch.linspace(0.1, 8, k.shape[0])[:, None, None].to(k.dtype)

    _check_decode(pk, dev, [700], 1, 4, 1, 64, 16, "f16", size=4.0, change=rise)


def _specials(c):
    """Inf and NaN in values and keys of some tokens: the last one, which only
    the last new token sees, one that leaves the window, and one all rows see."""
    for b, n in enumerate(c.lens):
        if n > 40:
            c.v[b][n - 1, 0, 3] = float("inf")
            c.v[b][n - 1, 0, 5] = float("nan")
            c.v[b][n - 22, :, 7] = float("-inf")
            c.v[b][n - 23, :, 8] = float("nan")
            c.k[b][n - 24, 0] = float("nan")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_specials_in_hidden_places(pk, dev, dtype, D):
    # window 20, four new tokens: the tokens 22 .. 24 back are seen by some of them
    _check_decode(pk, dev, [41, 64, 90], 4, 4, 2, D, 16, dtype, window=20, sinks=1, change=_specials)
    _check_decode(pk, dev, [41, 64, 90], 3, 4, 2, D, 32, dtype, change=lambda c: [
        c.v[b].__setitem__((n - 1, 0, 3), float("inf")) for b, n in enumerate(c.lens)])


def test_decode_shared_pages(pk, dev):
    """Two sequences share their first pages."""
    c = ref.Cache(3, [80, 75], 2, 64, 16, "bf16", dev)
    c.tables[1, :3] = c.tables[0, :3]
    c.k[1][:48], c.v[1][:48] = c.k[0][:48], c.v[0][:48]
    k, v, tables, tl = c.upload()
    q, qd = _queries(4, 2, 4, 64, "bf16", dev)
    out = pk.decode(qd, k, v, tables, tl)
    for b in range(2):
        o, _, mag, big = _expect(c, b, q[b:b + 1], 1, 0.125, 0, 0)
        ref.check_out(out[b:b + 1], o, mag, big, 80, 5.0, "bf16", 64, b)


def _check_prefill(pk, dev, lens, new, H, kv, D, P, dtype, window=0, sinks=0, absent=(), max_len=None,
                   fused=False, extra=0, size=1.0, change=None, seed=0, scale=None):
    c = ref.Cache(seed + 29 * D + P, lens, kv, D, P, dtype, dev, absent)
    if change:
        change(c)
    k, v, tables, tl = c.upload()
    T = sum(new)
    q, qd = _queries(seed + 7, T + extra, H, D, dtype, dev, fused, size)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    out = torch.full((T + extra, H, D), 7.0, dtype=q.dtype, device=dev)
    pk.prefill(qd, torch.tensor(cu, dtype=torch.int32, device=dev), k, v, tables, tl, scale=scale,
               window=window, sinks=sinks, max_len=max_len, out=out)
    s = D ** -0.5 if scale is None else scale
    torch.cuda.synchronize()
    for b, n in enumerate(new):
        o, _, mag, big = _expect(c, b, q[cu[b]:cu[b + 1]], n, s, window, sinks)
        vmax = float(c.v[b].double().nan_to_num(0, 0, 0).abs().max()) if lens[b] else 0.0
        ref.check_out(out[cu[b]:cu[b + 1]], o, mag, big, lens[b], vmax, dtype, D, ("prefill", b, n))
    assert bool((out[T:] == 7.0).all()), "rows of no sequence"


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 32), (256, 16), (128, 128), (256, 64), (64, 512)])
def test_prefill_lengths(pk, dev, dtype, D, P):
    # whole prompts, chunks with earlier context, none, one token, more new
    # tokens than cached ones (the first of them see nothing)
    _check_prefill(pk, dev, [1, 33, 0, 64, 100, 130, 0, 5], [1, 33, 0, 64, 37, 1, 3, 9], 8, 2, D, P, dtype)


@pytest.mark.parametrize("H,kv", [(1, 1), (3, 1), (8, 8), (15, 3), (64, 1), (5, 5)])
def test_prefill_heads(pk, dev, H, kv):
    _check_prefill(pk, dev, [70, 31], [70, 9], H, kv, 64, 16, "bf16")
    _check_prefill(pk, dev, [45], [45], H, kv, 128, 32, "f16", window=11, sinks=2)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 4), (16, 0), (33, 40), (64, 16), (100, 3),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64), (256, 32)])
def test_prefill_window(pk, dev, window, sinks, D, P):
    _check_prefill(pk, dev, [150, 299, 40], [150, 60, 1], 8, 2, D, P, "bf16", window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_prefill_absent_pages(pk, dev, window, sinks):
    absent = [(0, 1), (0, 2), (1, 0), (2, 3), (3, 0), (3, 1)]
    _check_prefill(pk, dev, [100, 70, 64, 32], [100, 30, 40, 32], 8, 2, 128, 16, "bf16", window, sinks,
                   absent)
    _check_prefill(pk, dev, [100, 70, 64, 32], [100, 30, 40, 32], 4, 2, 256, 16, "f16", window, sinks,
                   absent)


@pytest.mark.parametrize("max_len", [None, 100])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_splits(pk, dev, max_len, D):
    # few rows over a long context: the cache's length is split
    _check_prefill(pk, dev, [2100, 900], [12, 3], 4, 2, D, 32, "bf16", max_len=max_len)


def test_prefill_strided_and_extra_rows(pk, dev):
    _check_prefill(pk, dev, [50, 60], [50, 20], 8, 2, 256, 16, "bf16", fused=True, extra=5)
    _check_prefill(pk, dev, [2000], [4], 8, 2, 128, 16, "f16", fused=True, extra=3)


@pytest.mark.parametrize("scale", [0.3, -0.2, 0.0])
def test_prefill_scale(pk, dev, scale):
    _check_prefill(pk, dev, [70, 33], [70, 5], 4, 2, 128, 16, "bf16", window=20, sinks=3, scale=scale)
    _check_prefill(pk, dev, [70, 33], [70, 5], 4, 2, 256, 16, "f16", scale=scale)


def test_prefill_large_scores(pk, dev):
    _check_prefill(pk, dev, [200, 37], [90, 37], 4, 2, 128, 16, "bf16", size=60.0)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefill_specials_in_hidden_places(pk, dev, dtype, D):
    _check_prefill(pk, dev, [41, 64, 90], [30, 64, 25], 4, 2, D, 16, dtype, window=20, sinks=1,
                   change=_specials)
    _check_prefill(pk, dev, [41, 64, 190], [30, 64, 100], 4, 2, D, 32, dtype, change=_specials)


# --- append -----------------------------------------------------------------------


@pytest.mark.parametrize("D,P,dtype", [(64, 16, "bf16"), (128, 32, "f16"), (256, 16, "bf16"), (256, 64, "f16")])
@pytest.mark.parametrize("strided", [False, True])
def test_append(pk, dev, D, P, dtype, strided):
    kv, lens = 3, [1, 9, 0, 40, 33, 100, 17, 8]
    new = [1, 9, 0, 3, 17, 61, 1, 4]
    c = ref.Cache(D + P, lens, kv, D, P, dtype, dev, absent=[(5, 1)])
    k, v, tables, tl = c.upload()
    want_k, want_v = k.clone(), v.clone()
    old_k, old_v = k.clone(), v.clone()
    T = sum(new)
    # the cache starts without the new tokens, other places hold a pattern
    fill = torch.randn(k.shape, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(k.dtype)
    gone_k, gone_v = torch.zeros_like(k, dtype=torch.bool), torch.zeros_like(v, dtype=torch.bool)
    rows_k, rows_v = [], []
    for b, (n, m) in enumerate(zip(lens, new)):
        rows_k.append(c.k[b][n - m:])
        rows_v.append(c.v[b][n - m:])
        t = torch.arange(n - m, n)
        t = t[c.here[b][t]]
        at = c.tables[b, t // P].long()
        gone_k[at, :, t % P] = True
        gone_v[at, :, t % P // 8, :, t % 8] = True
    k = torch.where(gone_k, fill, old_k)
    v = torch.where(gone_v, fill.view_as(old_v), old_v)
    w = torch.full((c.num_pages, kv, P), 3.0, device=dev)
    nk, nv = torch.cat(rows_k).to(dev), torch.cat(rows_v).to(dev)
    if strided:  # columns of a fused k, v projection
        both = torch.cat([nk.flatten(1), nv.flatten(1)], dim=1)
        nk, nv = (x.unflatten(1, (kv, D)) for x in both.split(kv * D, dim=1))
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev)
    pk.append(nk, nv, k, v, tables, tl, cu_new=cu, weights=w)
    torch.cuda.synchronize()
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))
    assert torch.equal(w == 0, gone_k[..., 0]) and bool((w[w != 0] == 3).all())
    assert T == nk.shape[0]


@pytest.mark.parametrize("Q", [1, 5, 20])
def test_append_uniform(pk, dev, Q):
    lens = [20, 21, 39, 40, 64]
    c = ref.Cache(Q, lens, 2, 128, 16, "bf16", dev)
    k, v, tables, tl = c.upload()
    want_k, want_v = k.clone(), v.clone()
    for b, n in enumerate(lens):
        t = torch.arange(n - Q, n)
        at = c.tables[b, t // 16].long()
        k[at, :, t % 16] = 0
        v[at, :, t % 16 // 8, :, t % 8] = 0
    nk = torch.cat([c.k[b][-Q:] for b in range(5)]).to(dev)
    nv = torch.cat([c.v[b][-Q:] for b in range(5)]).to(dev)
    pk.append(nk, nv, k, v, tables, tl)
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))


# --- eviction -----------------------------------------------------------------------


def _check_evict(pk, dev, lens, kv, D, P, dtype, keep, sinks, recent, weight, absent=(), max_len=None, seed=0):
    c = ref.Cache(seed + D + P + keep, lens, kv, D, P, dtype, dev, absent, spare=len(lens) * -(-keep // P) + 3)
    k, v, tables, tl = c.upload()
    used = set(c.tables[c.tables >= 0].tolist())
    free = [p for p in range(c.num_pages) if p not in used]
    W = -(-keep // P)
    dst = torch.tensor(free[:len(lens) * W], dtype=torch.int32).view(len(lens), W)
    w = torch.full((c.num_pages, kv, P), float("nan"))
    ww = [weight(b, n, kv) for b, n in enumerate(lens)]  # [kv, n]
    for b, n in enumerate(lens):
        t = torch.arange(n)[c.here[b]]
        if len(t):
            w[c.tables[b, t // P].long(), :, t % P] = ww[b][:, t].t()
    w = w.to(dev)
    want_k, want_v, want_w = k.clone(), v.clone(), w.clone()
    kept, new_lens = pk.evict(k, v, tables, tl, w, dst.to(dev), keep, sinks, recent, max_len=max_len)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        for h in range(kv):
            x = ref.evict_kept(ww[b][h].tolist(), c.here[b].tolist(), keep, sinks, recent)
            assert kept[b, h].tolist() == x + [-1] * (keep - len(x)), (b, h, n)
            assert int(new_lens[b]) == len(x)
            src, i = torch.tensor(x, dtype=torch.long), torch.arange(len(x))
            to = dst[b, i // P].long()
            want_k[to, h, i % P] = c.k[b][src, h].to(dev)
            want_v[to, h, i % P // 8, :, i % 8] = c.v[b][src, h].to(dev)
            want_w[to, h, i % P] = ww[b][h][src].to(dev)
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))
    assert torch.equal(w.view(torch.int32), want_w.view(torch.int32))


def _heavy(b, n, kv):
    g = torch.Generator().manual_seed(100 + b)
    return (torch.randn(kv, n, generator=g) * 2).exp()


@pytest.mark.parametrize("D,P,dtype", [(64, 16, "bf16"), (128, 32, "f16"), (256, 64, "bf16")])
@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (7, 4, 2), (40, 4, 16), (64, 0, 64), (33, 50, 50),
                                               (100, 0, 0), (2000, 4, 8)])
def test_evict(pk, dev, D, P, dtype, keep, sinks, recent):
    _check_evict(pk, dev, [0, 1, 30, 64, 129, 1500], 2, D, P, dtype, keep, sinks, recent, _heavy)


def test_evict_ties_and_odd_weights(pk, dev):
    def odd(b, n, kv):
        g = torch.Generator().manual_seed(b)
        pick = torch.tensor([0.0, -0.0, 1.0, 1.0, -2.0, float("inf"), float("-inf"), float("nan"), 1e-42, 0.5])
        return pick[torch.randint(0, 10, (kv, n), generator=g)]

    for keep in (1, 5, 17, 50, 90, 400):
        _check_evict(pk, dev, [10, 77, 300], 2, 64, 16, "bf16", keep, 2, 3, odd)
    _check_evict(pk, dev, [2500], 1, 64, 16, "bf16", 1111, 0, 0, lambda b, n, kv: torch.zeros(kv, n))
    _check_evict(pk, dev, [90], 1, 64, 16, "bf16", 30, 1, 1, lambda b, n, kv: torch.full((kv, n), float("nan")))


def test_evict_absent_pages(pk, dev):
    absent = [(0, 0), (0, 2), (1, 1), (1, 2), (1, 3)]
    for keep in (5, 40, 90):
        _check_evict(pk, dev, [100, 64, 20], 2, 64, 16, "f16", keep, 4, 4, _heavy, absent)


@pytest.mark.parametrize("max_len", [None, 100, 41000])
def test_evict_long(pk, dev, max_len):
    # more tokens than the LDS holds keys for, next to a short sequence
    _check_evict(pk, dev, [41000, 300], 1, 64, 128, "bf16", 5000, 4, 100, _heavy, max_len=max_len)


# --- more sequences than a wave has lanes ----------------------------------------------

MANY = [(37 * i * i + 11 * i) % 501 for i in range(150)]  # 0 .. 500 tokens


@pytest.mark.parametrize("Q,weights", [(1, None), (5, "add")])
def test_decode_many_sequences(pk, dev, Q, weights):
    _check_decode(pk, dev, MANY, Q, 8, 2, 64, 16, "bf16", weights=weights)
    _check_decode(pk, dev, MANY[:65], Q, 8, 2, 128, 32, "f16", window=100, sinks=4, weights=weights)


def test_prefill_append_and_evict_many_sequences(pk, dev):
    new = [min(n, 1 + (7 * i) % 40) for i, n in enumerate(MANY)]
    _check_prefill(pk, dev, MANY, new, 8, 2, 64, 16, "f16")
    _check_prefill(pk, dev, MANY[:129], new[:129], 4, 4, 128, 32, "bf16", window=50, sinks=4)
    _check_evict(pk, dev, MANY, 2, 64, 16, "bf16", 40, 4, 8, _heavy)
    kv, D, P = 2, 64, 16
    c = ref.Cache(7, MANY, kv, D, P, "bf16", dev)
    k, v, tables, tl = c.upload()
    want_k, want_v = k.clone(), v.clone()
    for b, (n, m) in enumerate(zip(MANY, new)):
        t = torch.arange(n - m, n)
        at = c.tables[b, t // P].long()
        k[at, :, t % P] = 0
        v[at, :, t % P // 8, :, t % 8] = 0
    nk, nv = (torch.cat([x[b][n - m:] for b, (n, m) in enumerate(zip(MANY, new))]).to(dev) for x in (c.k, c.v))
    cu = torch.tensor([sum(new[:i]) for i in range(151)], dtype=torch.int32, device=dev)
    pk.append(nk, nv, k, v, tables, tl, cu_new=cu)
    assert torch.equal(k.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), want_v.view(torch.int16))


def test_row_ranges_that_do_not_ascend(pk, dev):
    """Sequences 1 and 2 have ranges that end before they begin and after the last row: sequence 0 gets
    its results, and the others' pages stay as they are."""
    c = ref.Cache(9, [70, 50, 600], 2, 64, 16, "bf16", dev)
    k, v, tables, tl = c.upload()
    cu = torch.tensor([0, 60, 30, 500], dtype=torch.int32, device=dev)
    q, qd = _queries(11, 100, 8, 64, "bf16", dev)
    out = pk.prefill(qd, cu, k, v, tables, tl, max_len=100)
    o, _, mag, big = _expect(c, 0, q[:60], 60, 0.125, 0, 0)
    ref.check_out(out[:60], o, mag, big, 70, float(c.v[0].abs().max()), "bf16", 64, 0)
    before_k, before_v = k.clone(), v.clone()
    nk, nv = (torch.randn(100, 2, 64, device=dev).to(k.dtype) for _ in range(2))
    nk[:60], nv[:60] = c.k[0][10:].to(dev), c.v[0][10:].to(dev)
    pk.append(nk, nv, k, v, tables, tl, cu_new=cu)
    assert torch.equal(k.view(torch.int16), before_k.view(torch.int16))
    assert torch.equal(v.view(torch.int16), before_v.view(torch.int16))
    cu = torch.tensor([50, 0, -7, 100], dtype=torch.int32, device=dev)
    pk.prefill(qd, cu, k, v, tables, tl)
    pk.append(nk, nv, k, v, torch.full_like(tables, -1), tl, cu_new=cu)
    torch.cuda.synchronize()


# --- a pool past 32-bit offsets ------------------------------------------------------


def test_offsets_past_32_bits(pk, dev):
    """Pages beyond 2^32 bytes and 2^31 elements of the pool, for every operator."""
    pages, kv, P, D, L = 5200, 2, 1024, 256, 1500
    k = torch.empty(pages, kv, P, D, dtype=torch.bfloat16, device=dev)
    v = torch.empty(pages, kv, P // 8, D, 8, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(pages, kv, P, device=dev)
    assert (pages - 10) * kv * P * D > 2 ** 31
    c = ref.Cache(11, [L, 70], kv, D, P, "bf16", dev, width=2)
    tables = torch.tensor([[pages - 1, pages - 3], [pages - 2, -1]], dtype=torch.int32, device=dev)
    tl = torch.tensor([L, 70], dtype=torch.int32, device=dev)
    cu = torch.tensor([0, L, L + 70], dtype=torch.int32, device=dev)
    pk.append(torch.cat(c.k).to(dev), torch.cat(c.v).to(dev), k, v, tables, tl, cu_new=cu, weights=w)
    q, qd = _queries(12, 2, 8, D, "bf16", dev)
    out = pk.decode(qd, k, v, tables, tl, weights=w)
    for b in range(2):
        o, ww, mag, big = _expect(c, b, q[b:b + 1], 1, D ** -0.5, 0, 0)
        ref.check_out(out[b:b + 1], o, mag, big, L, 6.0, "bf16", D, ("decode", b))
    q, qd = _queries(13, 40, 8, D, "bf16", dev)
    out = pk.prefill(qd, torch.tensor([0, 33, 40], dtype=torch.int32, device=dev), k, v, tables, tl)
    for b, (a, e) in enumerate(((0, 33), (33, 40))):
        o, _, mag, big = _expect(c, b, q[a:e], e - a, D ** -0.5, 0, 0)
        ref.check_out(out[a:e], o, mag, big, L, 6.0, "bf16", D, ("prefill", b))
    dst = torch.tensor([[pages - 5], [pages - 6]], dtype=torch.int32, device=dev)
    kept, lens = pk.evict(k, v, tables, tl, w, dst, 500, 4, 16)
    assert lens.tolist() == [500, 70]
    for b, n in enumerate((500, 70)):
        for h in range(kv):
            src = kept[b, h, :n].cpu().long()
            i, to = torch.arange(n, device=dev), int(dst[b, 0])
            assert torch.equal(k[to, h, :n].cpu(), c.k[b][src, h])
            assert torch.equal(v[to, h, i // 8, :, i % 8].cpu(), c.v[b][src, h])


# --- streams and graphs ---------------------------------------------------------------


def _step(pk, c, k, v, tables, tl, nk, nv, q, w, stream=None):
    pk.append(nk, nv, k, v, tables, tl, weights=w, stream=stream)
    return pk.decode(q, k, v, tables, tl, weights=w, stream=stream)


def test_side_stream_and_graph(pk, dev):
    lens, kv, D = [300, 1234, 77], 2, 128
    c = ref.Cache(8, lens, kv, D, 16, "bf16", dev)
    k, v, tables, tl = c.upload()
    nk = torch.stack([c.k[b][-1] for b in range(3)]).to(dev)
    nv = torch.stack([c.v[b][-1] for b in range(3)]).to(dev)
    _, q = _queries(1, 3, 8, D, "bf16", dev)
    w = torch.zeros(c.num_pages, kv, 16, device=dev)
    expect = _step(pk, c, k, v, tables, tl, nk, nv, q, w).clone()
    first = w.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for handle in (side, side.cuda_stream):
        w.zero_()
        side.wait_stream(torch.cuda.current_stream())
        got = _step(pk, c, k, v, tables, tl, nk, nv, q, w, stream=handle)
        side.synchronize()
        assert torch.equal(got, expect) and torch.equal(w, first)
    with torch.cuda.stream(side):
        w.zero_()
        got = _step(pk, c, k, v, tables, tl, nk, nv, q, w)
    side.synchronize()
    assert torch.equal(got, expect) and torch.equal(w, first)
    graph = torch.cuda.CUDAGraph()
    q2 = q.clone()
    with torch.cuda.graph(graph):
        out = _step(pk, c, k, v, tables, tl, nk, nv, q2, w)
    for i in range(4):
        q2.copy_(q * (1 + i % 2))
        eager_w = torch.zeros_like(w)
        eager = _step(pk, c, k, v, tables, tl, nk, nv, q2, eager_w)
        w.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(w, eager_w), i
    cu = torch.tensor([0, 100, 260, 277], dtype=torch.int32, device=dev)
    _, qp = _queries(2, 277, 8, D, "bf16", dev)
    expect = pk.prefill(qp, cu, k, v, tables, tl)
    torch.cuda.synchronize()
    got = pk.prefill(qp, cu, k, v, tables, tl, stream=side)
    side.synchronize()
    assert torch.equal(got, expect)


def test_outputs_are_memory_of_their_stream(pk, dev):
    """A call on another stream does not write memory that was freed on the current one,
    whose work may still use it."""
    c = ref.Cache(18, [700, 90], 2, 64, 16, "f16", dev)
    k, v, tables, tl = c.upload()
    _, q = _queries(3, 2, 8, 64, "f16", dev)
    _, qp = _queries(4, 100, 8, 64, "f16", dev)
    cu = torch.tensor([0, 60, 100], dtype=torch.int32, device=dev)
    w = torch.rand(c.num_pages, 2, 16, device=dev)
    dst = torch.full((2, 2), -1, dtype=torch.int32, device=dev)  # (nothing is copied)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def fresh(like, call):
        t = torch.empty_like(like)
        at = t.data_ptr()
        del t
        got = call()
        side.synchronize()
        assert got.shape == like.shape and got.data_ptr() != at

    fresh(q, lambda: pk.decode(q, k, v, tables, tl, stream=side))
    fresh(qp, lambda: pk.prefill(qp, cu, k, v, tables, tl, stream=side))
    kept = torch.empty(2, 2, 20, dtype=torch.int32, device=dev)
    lens = torch.empty(2, dtype=torch.int32, device=dev)
    fresh(kept, lambda: pk.evict(k, v, tables, tl, w, dst, 20, new_lens=lens, stream=side)[0])
    fresh(lens, lambda: pk.evict(k, v, tables, tl, w, dst, 20, kept=kept, stream=side)[1])


def test_prefill_and_eviction_in_a_graph(pk, dev):
    lens, kv, D = [700, 90], 2, 128
    c = ref.Cache(21, lens, kv, D, 16, "f16", dev, spare=40)
    k, v, tables, tl = c.upload()
    used = set(c.tables[c.tables >= 0].tolist())
    free = [p for p in range(c.num_pages) if p not in used]
    dst = torch.tensor(free[:32], dtype=torch.int32, device=dev).view(2, 16)
    w = torch.zeros(c.num_pages, kv, 16, device=dev)
    cu = torch.tensor([0, 60, 100], dtype=torch.int32, device=dev)
    _, qp = _queries(22, 100, 8, D, "f16", dev)
    graph = torch.cuda.CUDAGraph()

    def both():
        return (pk.prefill(qp, cu, k, v, tables, tl), *pk.evict(k, v, tables, tl, w, dst, 250, 4, 32))

    both()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = both()
    for i in range(3):
        w.uniform_()
        qp.mul_(-1.1)
        eager = both()
        first = [t.clone() for t in (k, v, w)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i
        assert torch.equal(w, first[2]) and torch.equal(k.view(torch.int16), first[0].view(torch.int16))


def test_kernel_registers(pk, dev):
    for dtype in (torch.bfloat16, torch.float16):
        for D in pk.HEAD_DIMS:
            assert 0 < pk.kernel_regs(dtype, D) <= 256 and 0 < pk.kernel_regs(dtype, D, prefill=True) <= 256


def test_repeated_calls_give_the_same_bits(pk, dev):
    c = ref.Cache(9, [2500, 3, 700], 2, 256, 32, "bf16", dev)
    k, v, tables, tl = c.upload()
    _, q = _queries(3, 3, 8, 256, "bf16", dev)
    _, qp = _queries(3, 300, 8, 256, "bf16", dev)
    cu = torch.tensor([0, 250, 253, 300], dtype=torch.int32, device=dev)
    w = torch.empty(c.num_pages, 2, 32, device=dev)
    first = None
    for _ in range(3):
        got = [pk.decode(q, k, v, tables, tl), pk.prefill(qp, cu, k, v, tables, tl),
               pk.decode(q, k, v, tables, tl, weights=w, accumulate=False)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
