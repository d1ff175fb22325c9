"""Rotary positions against float64: rows of heads in any layout, and new tokens'
keys on their way into the pages."""
import pytest
import torch

import paged_reference as ref
import rotary_reference as rr

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _plan(dev, pairs, sections=None, turns=False, adjacent=False, theta=1e4, scale=1.0):
    from cudalm_w4a16 import rotary

    f = rotary.frequencies(pairs, theta)
    return rotary.Rotary(f, sections, turns, adjacent, scale), f.cpu()


def _positions(g, axes, T, top):
    p = torch.randint(-top // 10, top, (axes, T), generator=g).to(torch.int32)
    if T > 2:
        p[:, 0], p[:, 1] = 0, top
    return p


# T, heads, D, pairs, sections, turns, adjacent, type
ROTATE = [(1, 8, 256, 32, None, False, False, "bf16"), (3, 2, 64, 32, None, False, False, "f16"),
          (7, 5, 128, 64, (24, 20, 20), True, False, "bf16"), (9, 1, 80, 40, (20, 20), False, False, "bf16"),
          (33, 16, 72, 36, (12, 12, 12), False, False, "f16"), (600, 3, 128, 64, (16, 24, 24), False, True, "f16"),
          (17, 4, 96, 16, (5, 0, 11), True, True, "bf16"), (2, 3, 72, 8, None, False, False, "bf16"),
          (5, 2, 7, 3, (1, 1, 1), True, False, "f16"), (4, 2, 11, 4, None, False, True, "bf16"),
          (4500, 2, 512, 256, (100, 50, 50, 56), True, False, "bf16"), (1100, 12, 64, 8, None, False, True, "f16"),
          (6, 300, 64, 32, None, False, False, "bf16"), (13, 2, 2, 1, None, False, True, "f16")]


@pytest.mark.parametrize("T,heads,D,pairs,sections,turns,adjacent,dtype", ROTATE)
@pytest.mark.parametrize("layout", ["plain", "in_place", "strided", "odd_base"])
def test_rotate(dev, T, heads, D, pairs, sections, turns, adjacent, dtype, layout):
    from cudalm_w4a16 import rotary

    g = torch.Generator().manual_seed(T * 131 + D)
    rot, f = _plan(dev, pairs, sections, turns, adjacent)
    sections = sections or (pairs,)
    x = torch.randn(T, heads, D, generator=g).to(DT[dtype])
    p = _positions(g, len(sections), T, 50000)
    want, tol = rr.rotated(x, p, f, sections, turns, adjacent)
    xd, pd = x.to(dev), p.to(dev)
    copied = x[:, :, 2 * pairs:]
    if layout == "plain":
        got = rotary.rotate(xd, pd if len(sections) > 1 else pd[0], rot)
        assert torch.equal(xd.cpu(), x)
    elif layout == "in_place":
        got = rotary.rotate(xd, pd, rot, out=xd)
        assert got is xd
    else:
        # heads and tokens apart by more than they are long, heads outside; one element off a line
        off = 1 if layout == "odd_base" else 8
        big = torch.full((heads, T + 1, D + 16), float("nan"), dtype=x.dtype, device=dev)
        xs = big[:, :T, off:off + D].transpose(0, 1)
        xs.copy_(xd)
        to = torch.full((T, heads + 1, D + 24), 7.0, dtype=x.dtype, device=dev)
        got = rotary.rotate(xs, pd, rot, out=to[:, :heads, off:off + D])
        rest = to.clone()
        rest[:, :heads, off:off + D] = 7.0
        assert (rest == 7).all(), "written beside the rows"
    rr.check(got, want, tol, layout)
    assert torch.equal(got[:, :, 2 * pairs:].cpu(), copied)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,heads,D,pairs,adjacent,off", [
    (4500, 3, 72, 36, True, 0), (4500, 3, 96, 20, False, 4), (9, 20, 76, 12, True, 4), (70, 2, 508, 252, False, 0),
    (1, 1, 8, 4, True, 0), (2, 3, 64, 32, False, 4), (6, 2, 72, 36, False, 2)])
def test_rotate_four_at_a_time(dev, T, heads, D, pairs, adjacent, off, dtype):
    from cudalm_w4a16 import rotary

    g = torch.Generator().manual_seed(T + D)
    rot, f = _plan(dev, pairs, None, False, adjacent)
    x = torch.randn(T, heads, D, generator=g).to(DT[dtype])
    p = _positions(g, 1, T, 50000)
    want, tol = rr.rotated(x, p, f, (pairs,), False, adjacent)
    flat = torch.full((T * heads * D + 16,), 7.0, dtype=x.dtype, device=dev)
    xd = flat[off:off + T * heads * D].view(T, heads, D)
    xd.copy_(x)
    out = torch.full_like(flat, 7.0)
    got = rotary.rotate(xd, p.to(dev), rot, out=out[off:off + T * heads * D].view(T, heads, D))
    rr.check(got, want, tol, "apart")
    assert torch.equal(got[:, :, 2 * pairs:].cpu(), x[:, :, 2 * pairs:])
    assert (out[:off] == 7).all() and (out[off + T * heads * D:] == 7).all(), "written beside the rows"
    assert torch.equal(rotary.rotate(xd, p.to(dev), rot, out=xd), got)


def test_far_positions_are_exact(dev):
    """Angles of positions up to 2^24 (2^31 where the angle's last places, 2^-22, allow for it)."""
    from cudalm_w4a16 import rotary

    rot, f = _plan(dev, 64, theta=1e7)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(64, 2, 128, generator=g).to(torch.float16)
    p = torch.randint(2 ** 23, 2 ** 24, (1, 64), generator=g).to(torch.int32)
    p[0, 0], p[0, 1] = -2 ** 24, 2 ** 24 - 1
    want, tol = rr.rotated(x, p, f, (64,), False, False)
    rr.check(rotary.rotate(x.to(dev), p.to(dev), rot), want, tol, "2^24")
    p[0] = 2 ** 31 - 1 - p[0].abs() // 8
    p[0, 5] = -2 ** 31
    want, tol = rr.rotated(x, p, f, (64,), False, False)
    size = x.double().abs().sum(2, keepdim=True)
    rr.check(rotary.rotate(x.to(dev), p.to(dev), rot), want, tol + size * 2.0 ** -20, "2^31")


def test_scale_and_special_values(dev):
    """The scale is of rotated channels only; Inf and NaN stay in their pair."""
    from cudalm_w4a16 import rotary

    rot, f = _plan(dev, 16, scale=0.75)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(20, 3, 64, generator=g).to(torch.bfloat16)
    p = _positions(g, 1, 20, 3000)
    want, tol = rr.rotated(x, p, f, (16,), False, False, 0.75)
    got = rotary.rotate(x.to(dev), p.to(dev), rot)
    rr.check(got, want, tol, "scale")
    bad = x.clone()
    bad[3, 1, 5], bad[4, 2, 40] = float("nan"), float("inf")
    again = rotary.rotate(bad.to(dev), p.to(dev), rot).cpu()
    assert again[3, 1, 5].isnan() and again[3, 1, 21].isnan() and again[4, 2, 40] == float("inf")
    same = torch.ones(20, 3, 64, dtype=torch.bool)
    same[3, 1, 5] = same[3, 1, 21] = same[4, 2, 40] = False
    assert torch.equal(again[same], got.cpu()[same])


def test_nothing_to_rotate(dev):
    from cudalm_w4a16 import rotary

    rot, _ = _plan(dev, 32)
    x = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=dev)
    assert rotary.rotate(x, torch.empty(1, 0, dtype=torch.int32, device=dev), rot).shape == x.shape


def _appended(dev, seed, lens, new, kv, heads, D, page, dtype, pairs, sections=None, turns=False, adjacent=False,
              given=True, cu=True, q_layout="split", absent=(), weights=False, behind=3, theta=1e4):
    """Appends rotated tokens to a cache and checks everything that the call may and may not write."""
    from cudalm_w4a16 import paged_kv as pk, rotary

    g = torch.Generator().manual_seed(seed)
    rot, f = _plan(dev, pairs, sections, turns, adjacent, theta)
    sections = sections or (pairs,)
    c = ref.Cache(seed, lens, kv, D, page, dtype, dev, absent=absent)
    k, v, tables, tl = c.upload()
    k0, v0 = k.clone(), v.clone()
    T = sum(new) + (behind if cu else 0)
    rows = torch.randn(T, heads + 2 * kv, D, generator=g).to(c.dtype)
    q, nk, nv = rows.split([heads, kv, kv], dim=1)
    start = [sum(new[:b]) for b in range(len(new) + 1)]
    place = torch.zeros(T, dtype=torch.int32)
    for b, n in enumerate(new):
        place[start[b]:start[b + 1]] = torch.arange(lens[b] - n, lens[b])
    p = _positions(g, len(sections), T, 30000) if given else place.repeat(len(sections), 1)
    qw, qt = rr.rotated(q, p, f, sections, turns, adjacent)
    kw, kt = rr.rotated(nk, p, f, sections, turns, adjacent)
    w = torch.full((c.num_pages, kv, page), 5.0, device=dev) if weights else None
    rd = rows.to(dev)
    qd, kd, vd = rd.split([heads, kv, kv], dim=1)
    out = None
    if q_layout == "in_place":
        out = qd
    elif q_layout == "given":
        out = torch.full((T, heads, D), 7.0, dtype=c.dtype, device=dev)
    args = dict(positions=p.to(dev) if given else None, weights=w,
                cu_new=torch.tensor(start, dtype=torch.int32, device=dev) if cu else None)
    if q_layout == "none":
        assert rotary.append(None, kd, vd, k, v, tables, tl, rot, **args) is None
    else:
        got = rotary.append(qd, kd, vd, k, v, tables, tl, rot, out=out, **args)
        n = start[-1]
        rr.check(got[:n], qw[:n], qt[:n], "queries")
        assert torch.equal(got[:n, :, 2 * pairs:].cpu(), q[:n, :, 2 * pairs:])
        if q_layout == "given":
            assert (got[n:] == 7).all(), "a row of no sequence was written"
        if q_layout == "in_place":
            assert torch.equal(got[n:].cpu(), q[n:])
    # every place of the cache
    want_k, tol_k = k0.double().cpu(), torch.zeros(k0.shape, dtype=torch.float64)
    want_v, want_w = v0.cpu().clone(), torch.full((c.num_pages, kv, page), 5.0)
    for b, n in enumerate(new):
        for j in range(n):
            t = lens[b] - n + j
            if t < 0:
                continue
            at = int(c.tables[b, t // page])
            if not 0 <= at < c.num_pages:
                continue
            r = start[b] + j
            want_k[at, :, t % page], tol_k[at, :, t % page] = kw[r], kt[r]
            want_v[at, :, t % page // 8, :, t % 8] = nv[r]
            want_w[at, :, t % page] = 0
    gk = k.double().cpu()
    assert torch.equal(gk.isnan(), want_k.isnan()), "places of the keys"
    rr.check(gk.nan_to_num(), want_k.nan_to_num(), tol_k, "keys")
    assert torch.equal(v.view(torch.int16).cpu(), want_v.view(torch.int16)), "values"
    if weights:
        assert torch.equal(w.cpu(), want_w), "weights"
    # the same bits as a rotation and a plain append
    k1, v1 = k0.clone(), v0.clone()
    turned = rotary.rotate(nk.to(dev).contiguous(), p.to(dev), rot)
    pk.append(turned, nv.to(dev).contiguous(), k1, v1, tables, tl, cu_new=args["cu_new"])
    assert torch.equal(k1.view(torch.int16), k.view(torch.int16)) and torch.equal(v1.view(torch.int16), v.view(torch.int16))


APPEND = [
    # a decode step, no cu; queries in place
    dict(lens=[17, 1, 300], new=[1, 1, 1], kv=2, heads=8, D=256, page=16, dtype="bf16", pairs=32, cu=False, q_layout="in_place"),
    dict(lens=[17, 40, 300], new=[4, 4, 4], kv=2, heads=8, D=64, page=16, dtype="f16", pairs=32, cu=False, given=False),
    # prompts, odd lengths, sequences without new tokens, rows behind the last
    dict(lens=[100, 33, 5, 64, 9], new=[100, 20, 0, 7, 9], kv=3, heads=6, D=128, page=32, dtype="bf16", pairs=64,
         sections=(24, 20, 20), turns=True, weights=True, q_layout="given"),
    dict(lens=[100, 33, 5], new=[37, 20, 2], kv=1, heads=5, D=128, page=16, dtype="f16", pairs=16, sections=(6, 5, 5),
         adjacent=True, given=False, q_layout="in_place"),
    dict(lens=[50], new=[50], kv=2, heads=1, D=64, page=128, dtype="bf16", pairs=8, q_layout="none", weights=True),
    # absent pages: queries are rotated all the same
    dict(lens=[90, 70], new=[60, 70], kv=2, heads=4, D=128, page=16, dtype="bf16", pairs=64, absent=[(0, 4), (1, 0)],
         weights=True, q_layout="given"),
    dict(lens=[200], new=[1], kv=40, heads=40, D=256, page=64, dtype="f16", pairs=128, adjacent=True, q_layout="given"),
]


@pytest.mark.parametrize("case", range(len(APPEND)))
def test_append(dev, case):
    _appended(dev, 100 + case, **APPEND[case])


def test_append_past_the_front_and_the_end(dev):
    """More rows than the length has: those before the first place are not cached, their queries are rotated;
    lengths past the tables count as the tables' end, negative ones as zero."""
    from cudalm_w4a16 import paged_kv as pk, rotary

    rot, f = _plan(dev, 32)
    g = torch.Generator().manual_seed(77)
    lens, new, page = [3, 1000, -5], [11, 9, 5], 16
    k = torch.zeros(8, 1, page, 64, dtype=torch.bfloat16, device=dev)
    v = torch.zeros(8, 1, page // 8, 64, 8, dtype=torch.bfloat16, device=dev)
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device=dev)
    tl = torch.tensor(lens, dtype=torch.int32, device=dev)
    x = torch.randn(25, 4, 64, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, 11, 20, 25], dtype=torch.int32, device=dev)
    kn, vn = x[:, :1].contiguous(), x[:, 1:2].contiguous()
    out = rotary.append(x[:, 2:].to(dev), kn.to(dev), vn.to(dev), k, v, tables, tl, rot, cu_new=cu)
    place = torch.cat([torch.arange(-8, 3), torch.arange(23, 32), torch.arange(-5, 0)]).to(torch.int32)[None]
    want, tol = rr.rotated(x, place, f, (32,), False, False)
    rr.check(out, want[:, 2:], tol[:, 2:], "queries")
    rr.check(k[0, 0, :3], want[8:11, 0], tol[8:11, 0], "front")
    rr.check(k[3, 0, 7:], want[11:20, 0], tol[11:20, 0], "end")
    dense = pk_dense(v)
    assert torch.equal(dense[0, 0, :3].cpu(), vn[8:11, 0]) and torch.equal(dense[3, 0, 7:].cpu(), vn[11:20, 0])
    assert int((k != 0).any(3).sum()) == 12 and int((dense != 0).any(3).sum()) == 12


def pk_dense(v):
    return v.permute(0, 1, 2, 4, 3).reshape(v.shape[0], v.shape[1], -1, v.shape[3])


def test_captured_and_on_another_stream(dev):
    """A graph of rotate and append, replayed between eager calls with other inputs; a call on a side stream."""
    from cudalm_w4a16 import rotary

    rot, _ = _plan(dev, 32, (11, 11, 10), True)
    g = torch.Generator(device=dev).manual_seed(3)
    T, kv, D = 24, 2, 256
    rows = torch.randn(T, 12, D, device=dev, generator=g).to(torch.bfloat16)
    p = torch.randint(0, 5000, (3, T), device=dev, generator=g).to(torch.int32)
    k = torch.zeros(T, kv, 16, D, dtype=torch.bfloat16, device=dev)
    v = torch.zeros(T, kv, 2, D, 8, dtype=torch.bfloat16, device=dev)
    tables = torch.arange(T, dtype=torch.int32, device=dev)[:, None]
    lens = torch.randint(1, 17, (T,), device=dev, generator=g).to(torch.int32)
    x = rows[:, :3].contiguous()
    out, y = torch.empty(T, 8, D, dtype=rows.dtype, device=dev), torch.empty_like(x)

    def calls(stream=None):
        rotary.append(rows[:, :8], rows[:, 8:10], rows[:, 10:], k, v, tables, lens, rot, positions=p, out=out, stream=stream)
        rotary.rotate(x, p, rot, out=y, stream=stream)
        return [t.clone() for t in (out, k, v, y)]

    calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rotary.append(rows[:, :8], rows[:, 8:10], rows[:, 10:], k, v, tables, lens, rot, positions=p, out=out)
        rotary.rotate(x, p, rot, out=y)
    for i in range(4):
        rows.normal_(generator=g)
        x.normal_(generator=g)
        p.random_(0, 9000, generator=g)
        lens.random_(1, 17, generator=g)
        k.zero_(), v.zero_()
        expect = calls()
        torch.cuda.synchronize()
        k.zero_(), v.zero_(), out.zero_(), y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(expect, (out, k, v, y))), i
        side = torch.cuda.Stream()
        k.zero_(), v.zero_(), out.zero_(), y.zero_()
        side.wait_stream(torch.cuda.current_stream())
        calls(side)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(expect, (out, k, v, y))), ("side", i)


def test_large_strides_and_offsets(dev):
    """Rows further apart than 32 bits of elements hold."""
    from cudalm_w4a16 import rotary

    rot, f = _plan(dev, 32)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(3, 2, 64, generator=g).to(torch.float16)
    big = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.float16, device=dev)
    xs = big.as_strided((3, 2, 64), (2 ** 30 + 64, 64, 1))
    xs.copy_(x.to(dev))
    p = _positions(g, 1, 3, 100)
    want, tol = rr.rotated(x, p, f, (32,), False, False)
    rr.check(rotary.rotate(xs, p.to(dev), rot, out=xs), want, tol, "far rows")
