"""Attention over the paged cache in every form that the calls are cut into: one launch
of eight waves, fixed splits and equal ranges of all tiles, one, two and four tiles of
rows, whole and split chunks, each by the name of the kernel that runs. With windows,
sinks, absent pages and weights; with Inf and NaN in values that rows see, whatever
their weights (one that underflows, one of zero); with rows whose scores are all -inf.
Expected results are float64, by the definition in the header; tolerances follow from the
roundings (paged_reference.py)."""
import pytest
import torch

import paged_reference as ref
from launched_kernels import launched_kernels

pytestmark = pytest.mark.gpu

SCALE = 0.125


@pytest.fixture(scope="module")
def pk(dev):
    if torch.cuda.get_device_properties(dev).multi_processor_count != 256:
        pytest.skip("the sizes stand for forms of a 256-CU part")
    from cudalm_w4a16 import paged_kv

    return paged_kv


def exact(q, k, v, here, pos, window, sinks):
    """As paged_reference.attention, and zeros where every score is -inf; Inf and NaN among the
    values that a row sees count whatever their weights."""
    q, k, v = q.double(), k.double(), v.double()
    n, H, D = q.shape
    L, kv = k.shape[0], k.shape[1]
    t = torch.arange(L)
    see = (t[None] <= pos[:, None]) & here[None]
    if window > 0:
        see &= (t[None] > pos[:, None] - window) | (t[None] < sinks)
    out, mag = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    w, big = torch.zeros(kv, L, dtype=torch.float64), 0.0
    if L == 0 or n == 0:
        return out, w, mag, big
    inf = float("inf")
    for h in range(H):
        g = h // (H // kv)
        size = (q[:, h].abs() @ k[:, g].abs().nan_to_num(0, 0, 0).t()).masked_fill(~see, 0)
        big = max(big, float(size.max()) * SCALE)
        # elementwise where keys are not finite: 0 * Inf of a product would not be theirs
        s = (q[:, h] @ k[:, g].t() * SCALE).masked_fill(~see, -inf)
        m = s.amax(1, keepdim=True)
        some = m[:, 0] != -inf
        p = torch.exp(s - m.clamp(min=-1e300)).masked_fill(~see, 0.0)
        p = torch.where(some[:, None], p / p.sum(1, keepdim=True), torch.zeros_like(p))
        x = v[:, g]
        o = p @ x.nan_to_num(0, 0, 0)
        seen = see.double()
        up = seen @ ((x == inf) | x.isnan()).double() > 0
        down = seen @ ((x == -inf) | x.isnan()).double() > 0
        o = torch.where(up, o + inf, o)
        o = torch.where(down, o - inf, o)
        out[:, h] = torch.where(some[:, None], o, torch.zeros_like(o))
        mag[:, h] = p @ x.nan_to_num(0, 0, 0).abs()
        w[g] += p.sum(0)
    return out, w, mag, big


# --- what the caches hold ---------------------------------------------------------------


def plain(c):
    pass


def specials(c):
    """Inf and NaN in the last token, in the middle and among the first ones; a channel that holds
    both signs of Inf; a key of NaN in the last key-value head."""
    for b, n in enumerate(c.lens):
        if n < 60:
            continue
        c.v[b][n - 1, 0, 3] = float("inf")
        c.v[b][n - 1, 0, 5] = float("nan")
        c.v[b][n // 2, :, 7] = float("-inf")
        c.v[b][n // 2 + 1, :, 8] = float("nan")
        c.v[b][2, :, 9] = float("inf")
        c.v[b][n - 3, :, 9] = float("-inf")
        if c.kv > 1:
            c.k[b][n // 3, c.kv - 1, 1] = float("nan")


def faint(c):
    """Inf and NaN in tokens whose scores are 400 below the others, so that their weights underflow."""
    for b, n in enumerate(c.lens):
        if n < 60:
            continue
        for t, channel, x in ((3, 1, float("inf")), (n // 2, 2, float("-inf")), (n // 2 + 9, 3, float("nan")),
                              (n - 9, 4, float("inf"))):
            c.k[b][t, :, 0] = -200
            c.v[b][t, :, channel] = x


def rise(c):
    """One token takes all the weight; Inf and NaN in ordinary ones before and after it."""
    for b, n in enumerate(c.lens):
        if n < 60:
            continue
        c.k[b][n // 2 + 7, :, 0] = 200
        for t, channel, x in ((1, 1, float("inf")), (n // 2 - 30, 2, float("-inf")), (n // 2 + 12, 3, float("nan")),
                              (n - 7, 4, float("inf"))):
            c.v[b][t, :, channel] = x


def lowest(c):
    """Every score of the first key-value head is -inf; in the last one those of the first half are."""
    for b, n in enumerate(c.lens):
        if n < 60:
            continue
        c.k[b][:, 0, 0] = float("-inf")
        if c.kv > 1:
            c.k[b][:n // 2, c.kv - 1, 0] = float("-inf")
        for t, channel, x in ((5, 1, float("inf")), (n // 2, 2, float("-inf")), (n - 4, 3, float("nan"))):
            c.v[b][t, :, channel] = x


# every query's first channel is 16: with scale 1/8, a key's first channel of -200 gives -400
def _queries(seed, rows, H, D, dtype):
    q = torch.randn(rows, H, D, generator=torch.Generator().manual_seed(seed)).to(ref.DT[dtype])
    q[:, :, 0] = 16
    return q


def _cache(seed, lens, kv, D, P, dtype, dev, absent, change):
    c = ref.Cache(seed, lens, kv, D, P, dtype, dev, absent)
    for k in c.k:  # scores of a few units, whatever the channel that all queries share
        k[:, :, 0] = k[:, :, 0] / 8
    change(c)
    return c


def _largest(c, b):
    return float(c.v[b].double().nan_to_num(0, 0, 0).abs().max()) if c.lens[b] else 0.0


# --- decode -----------------------------------------------------------------------------


def _mixed(B, top):
    """B lengths: the longest, short ones of 0 and 1, and others down to a third of it."""
    return [top - (i * 7 % B) * 2 * top // (3 * B) if i % 9 < 7 else i % 9 - 7 for i in range(B)]


# (D, P, dtype, new tokens, heads, kv heads, lengths, window, sinks): kernel <D, RT, WV, RANGES>
DECODE = {
    "one-1": ((64, 16, "bf16", 1, 4, 2, [70, 500, 33, 1, 1000], 0, 0), (64, 1, 8, 0)),
    "one-2": ((64, 16, "f16", 6, 8, 2, [600, 90, 0], 0, 0), (64, 2, 8, 0)),
    "splits-1": ((256, 16, "bf16", 1, 4, 1, [3333], 0, 0), (256, 1, 4, 0)),
    "splits-2": ((128, 32, "f16", 5, 16, 4, [1500, 800], 0, 0), (128, 2, 4, 0)),
    "splits-4": ((64, 64, "bf16", 10, 16, 4, [900, 300, 4], 0, 0), (64, 4, 4, 0)),
    "splits-window": ((128, 32, "bf16", 2, 8, 2, [2400, 1100, 77], 900, 5), (128, 1, 4, 0)),
    "ranges-1-64": ((64, 16, "f16", 1, 8, 8, _mixed(12, 1500), 0, 0), (64, 1, 4, 1)),
    "ranges-1-128": ((128, 32, "bf16", 1, 8, 2, _mixed(9, 5601), 0, 0), (128, 1, 4, 1)),
    "ranges-1-256": ((256, 64, "f16", 1, 8, 2, _mixed(9, 4500), 0, 0), (256, 1, 4, 1)),
    "ranges-2-128": ((128, 16, "f16", 5, 32, 8, _mixed(9, 901), 0, 0), (128, 2, 4, 1)),
    "ranges-4-256": ((256, 32, "bf16", 5, 16, 2, _mixed(9, 1500), 0, 0), (256, 4, 4, 1)),
    "ranges-4-64": ((64, 128, "f16", 9, 40, 4, _mixed(9, 1200), 0, 0), (64, 4, 4, 1)),  # two groups of 64 rows
    "ranges-window-128": ((128, 16, "bf16", 1, 32, 8, _mixed(30, 1500), 600, 40), (128, 1, 4, 1)),
    "ranges-window-256": ((256, 64, "f16", 3, 8, 2, _mixed(64, 900), 500, 4), (256, 1, 4, 1)),
}


def _decode(pk, dev, name, change=plain, absent=False, weights=False):
    (D, P, dtype, Q, H, kv, lens, window, sinks), (d, rt, waves, ranges) = DECODE[name]
    gone = [(b, w) for b, n in enumerate(lens) for w in (0, 2, 3) if w * P < n and (b + w) % 2] if absent else []
    c = _cache(3 * D + P + len(lens), lens, kv, D, P, dtype, dev, gone, change)
    k, v, tables, tl = c.upload()
    q = _queries(41, len(lens) * Q, H, D, dtype)
    qd = q.to(dev).unflatten(0, (len(lens), Q))
    w = torch.full((c.num_pages, kv, P), 0.25, device=dev) if weights else None
    out = torch.full((len(lens), Q, H, D), float("nan"), dtype=q.dtype, device=dev)
    call = lambda add=False: pk.decode(qd, k, v, tables, tl, scale=SCALE, window=window, sinks=sinks,  # noqa: E731
                                       weights=w, accumulate=add, out=out)
    kernel = launched_kernels(call)[0]
    assert "paged_decode_kernel" in kernel and f"Li{d}ELi{rt}ELi{waves}ELb{ranges}E" in kernel, kernel
    got_w = None if w is None else w.cpu()
    for b, L in enumerate(lens):
        o, ww, mag, big = exact(q[b * Q:(b + 1) * Q], c.k[b], c.v[b], c.here[b], torch.arange(Q) + L - Q, window, sinks)
        ref.check_out(out[b], o, mag, big, L, _largest(c, b), dtype, D, (name, b, L))
        if w is not None and L:
            t = torch.arange(L)[c.here[b]]
            have = got_w[c.tables[b, t // P].long(), :, t % P].t()
            full = ~ww[:, t].isnan().any(1)  # (a key of NaN leaves no weights to compare)
            ref.check_weights(have[full], ww[:, t][full], big + 4, Q * H, D, ("weights", name, b, L))
    if w is None:
        return
    # added: one fp32 sum each, of what the call without it gives; other places stay as they are
    mine = torch.zeros(w.shape, dtype=torch.bool)
    for b, L in enumerate(lens):
        t = torch.arange(L)[c.here[b]]
        mine[c.tables[b, t // P].long(), :, t % P] = True
    assert bool((got_w[~mine] == 0.25).all())
    w.fill_(0.75)
    call(add=True)
    assert torch.equal(w.cpu().nan_to_num(-1), torch.where(mine, 0.75 + got_w, 0.75).nan_to_num(-1))


@pytest.mark.parametrize("name", DECODE)
def test_decode(pk, dev, name):
    _decode(pk, dev, name)


@pytest.mark.parametrize("name", DECODE)
def test_decode_absent_pages(pk, dev, name):
    _decode(pk, dev, name, absent=True)


@pytest.mark.parametrize("absent", [False, True])
@pytest.mark.parametrize("name", DECODE)
def test_decode_weights(pk, dev, name, absent):
    _decode(pk, dev, name, absent=absent, weights=True)


@pytest.mark.parametrize("name", DECODE)
def test_decode_specials(pk, dev, name):
    _decode(pk, dev, name, specials)


@pytest.mark.parametrize("change", [faint, rise])
@pytest.mark.parametrize("name", DECODE)
def test_decode_specials_of_tiny_weight(pk, dev, name, change):
    _decode(pk, dev, name, change)


@pytest.mark.parametrize("name", DECODE)
def test_decode_of_scores_that_are_all_lowest(pk, dev, name):
    _decode(pk, dev, name, lowest, weights=True)


# --- prefill ----------------------------------------------------------------------------

# (D, P, dtype, new tokens, heads, kv heads, lengths, window, sinks): split over the length or not
PREFILL = {
    "whole-64": ((64, 16, "f16", [300, 64, 0, 200], 64, 32, [300, 500, 3, 1100], 0, 0), False),
    "whole-128": ((128, 32, "bf16", [391, 129], 64, 64, [391, 700], 0, 0), False),
    "whole-256": ((256, 64, "f16", [300, 70], 128, 64, [300, 170], 0, 0), False),
    "whole-window": ((128, 16, "f16", [300, 200], 8, 2, [300, 900], 100, 20), False),
    "split-64": ((64, 16, "bf16", [12, 3], 4, 2, [2100, 900], 0, 0), True),
    "split-128": ((128, 32, "f16", [40, 9, 1], 8, 2, [1700, 3001, 1], 0, 0), True),
    "split-256": ((256, 64, "bf16", [130, 20], 8, 2, [1300, 2000], 0, 0), True),
    "split-window": ((128, 32, "bf16", [50], 8, 2, [2400], 900, 40), True),
}


def _prefill(pk, dev, name, change=plain, absent=False):
    (D, P, dtype, new, H, kv, lens, window, sinks), split = PREFILL[name]
    gone = [(b, w) for b, n in enumerate(lens) for w in (0, 2, 3) if w * P < n and (b + w) % 2] if absent else []
    c = _cache(5 * D + P + len(lens), lens, kv, D, P, dtype, dev, gone, change)
    k, v, tables, tl = c.upload()
    q = _queries(43, sum(new), H, D, dtype)
    qd = q.to(dev)
    cu = [sum(new[:i]) for i in range(len(new) + 1)]
    tcu = torch.tensor(cu, dtype=torch.int32, device=dev)
    out = torch.full_like(qd, float("nan"))
    call = lambda: pk.prefill(qd, tcu, k, v, tables, tl, scale=SCALE, window=window, sinks=sinks, out=out)  # noqa: E731
    assert len(launched_kernels(call)) == (2 if split else 1)
    for b, (n, L) in enumerate(zip(new, lens)):
        o, _, mag, big = exact(q[cu[b]:cu[b + 1]], c.k[b], c.v[b], c.here[b], torch.arange(n) + L - n, window, sinks)
        ref.check_out(out[cu[b]:cu[b + 1]], o, mag, big, L, _largest(c, b), dtype, D, (name, b, n, L))


@pytest.mark.parametrize("absent", [False, True])
@pytest.mark.parametrize("name", PREFILL)
def test_prefill(pk, dev, name, absent):
    _prefill(pk, dev, name, absent=absent)


@pytest.mark.parametrize("name", PREFILL)
def test_prefill_specials(pk, dev, name):
    _prefill(pk, dev, name, specials)


@pytest.mark.parametrize("change", [faint, rise])
@pytest.mark.parametrize("name", PREFILL)
def test_prefill_specials_of_tiny_weight(pk, dev, name, change):
    _prefill(pk, dev, name, change)


@pytest.mark.parametrize("name", PREFILL)
def test_prefill_of_scores_that_are_all_lowest(pk, dev, name):
    _prefill(pk, dev, name, lowest)
