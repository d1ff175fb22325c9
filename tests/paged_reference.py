"""Plain float64 forms of the paged cache's operators, for their tests, and
caches whose unwritten places hold NaN."""
import numpy as np
import torch

DT = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # an ulp of 1: twice the rounding error


class Cache:
    """Random keys and values of sequences of the given lengths, dense on the
    CPU and in pages on the GPU. absent: (sequence, table entry) pairs whose
    pages are not there; a negative or a too large page number says so."""

    def __init__(self, seed, lens, kv, D, page, dtype, dev, absent=(), spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.kv, self.D, self.page, self.dtype = list(lens), kv, D, page, DT[dtype]
        self.k = [torch.randn(n, kv, D, generator=g).to(self.dtype) for n in lens]
        self.v = [torch.randn(n, kv, D, generator=g).to(self.dtype) for n in lens]
        need = [-(-n // page) for n in lens]
        W = width or max(1, max(need))
        self.num_pages = sum(need) + spare
        order = torch.randperm(self.num_pages, generator=g)[:sum(need)].to(torch.int32)
        self.tables = torch.full((len(lens), W), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n]
            at += n
        self.here = [torch.ones(n, dtype=torch.bool) for n in lens]
        for i, (b, w) in enumerate(absent):
            self.tables[b, w] = -1 if i % 2 == 0 else self.num_pages + 5
            self.here[b][w * page:(w + 1) * page] = False
        self.dev = dev

    def upload(self):
        """(k, v, tables, lens) on the GPU."""
        pages, kv, D, P = self.num_pages, self.kv, self.D, self.page
        k = torch.full((pages, kv, P, D), float("nan"), dtype=self.dtype)
        v = torch.full((pages, kv, P // 8, D, 8), float("nan"), dtype=self.dtype)
        for b, n in enumerate(self.lens):
            t = torch.arange(n)[self.here[b]]
            if len(t):
                at = self.tables[b, t // P].long()
                k[at, :, t % P] = self.k[b][t]
                v[at, :, t % P // 8, :, t % 8] = self.v[b][t]
        return (k.to(self.dev), v.to(self.dev), self.tables.to(self.dev),
                torch.tensor(self.lens, dtype=torch.int32, device=self.dev))


def attention(q, k, v, here, pos, scale, window, sinks):
    """One sequence: q [n, heads, D] at positions pos (long [n]) over k, v [L,
    kv, D] of which `here` [L] exist. (out, sum of weights [kv, L], sum of
    weights times |v| like out, largest sum |q k| scale), all float64."""
    q, k, v = q.double(), k.double(), v.double()
    n, H, D = q.shape
    L, kv = k.shape[0], k.shape[1]
    t = torch.arange(L)
    see = (t[None] <= pos[:, None]) & here[None]
    if window > 0:
        see &= (t[None] > pos[:, None] - window) | (t[None] < sinks)
    out, mag = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    w, big = torch.zeros(kv, L, dtype=torch.float64), 0.0
    for h in range(H):
        g = h // (H // kv)
        for i in range(n):
            x = torch.nonzero(see[i]).flatten()
            if len(x) == 0:
                continue
            s = k[x, g] @ q[i, h] * scale
            big = max(big, float((k[x, g].abs() @ q[i, h].abs()).nan_to_num(0, 0, 0).max()) * abs(scale))
            p = torch.softmax(s, 0)
            out[i, h] = p @ v[x, g]
            mag[i, h] = p @ v[x, g].abs()
            w[g, x] += p
    return out, w, mag, big


def check_out(got, out, mag, big, L, vmax, dtype, D, what):
    """Elementwise: the output's rounding (u |o|), the weights' (u sum p |v|), the
    scores' and exponentials' in fp32 (twice (D 2^-24 big + 2^-19) sum p |v|:
    numerator and denominator) and, in fp16, weights below 2^-14 (2^-25 each)."""
    u = UNIT[dtype]
    got = got.double().cpu()
    assert torch.equal(got.isnan(), out.isnan()), (what, "NaN places")
    inf = out.isinf()
    assert torch.equal(got[inf], out[inf]), (what, "infinities")
    tol = u * out.abs() + (u + 2 * (D * 2.0 ** -24 * big + 2.0 ** -19)) * mag
    if dtype == "f16":
        tol = tol + L * 2.0 ** -25 * vmax
    bad = ((got - out).abs() > tol) & ~inf & ~out.isnan()
    assert not bad.any(), (what, int(bad.sum()), float((got - out).abs()[bad].max()))


def check_weights(got, w, big, rows, D, what):
    """Relative: the scores' and exponentials' error, sums over the rows in fp32."""
    tol = w * (2 * (D * 2.0 ** -24 * big + 2.0 ** -19) + rows * 2.0 ** -23) + 1e-30
    bad = (got.double().cpu() - w).abs() > tol
    assert not bad.any(), (what, int(bad.sum()))


def evict_kept(weights, here, keep, sinks, recent):
    """Kept positions of one sequence and head, ascending: numpy, by sorting."""
    n = len(weights)
    s = min(sinks, keep)
    r = min(recent, keep - s)
    rank = []
    for t in range(n):
        if not here[t]:
            continue
        w = float(weights[t])
        forced = t < s or t >= n - r
        rank.append((0 if forced else 1 if w == w else 2, 0.0 if forced or w != w else -w, t))
    return sorted(t for _, _, t in sorted(rank)[:keep])


def verify(p, q, tokens, u, u_next):
    """One sequence, exact whole numbers: (accepted, next token). q None: certain."""
    f = np.float32
    n, V = 0, p.shape[1]
    for i, x in enumerate(tokens):
        if not 0 <= x < V:
            break
        qx = f(1) if q is None else f(q[i, x])
        if not f(u[i]) * qx < f(p[i, x]):
            break
        n += 1

    def units(r):
        return [int(min(max(float(x), 0.0), 1.0) * 2.0 ** 40) if x == x else 0 for x in r]

    whole = units(p[n])
    r = whole
    if n < len(tokens):
        if q is None:
            less = np.zeros(V, f)
            if 0 <= tokens[n] < V:
                less[tokens[n]] = 1
        else:
            less = q[n].astype(f)
        r = units(p[n].astype(f) - less)
        if sum(r) == 0:
            r = whole
    total = sum(r)
    if total == 0:
        return n, -1
    U = min(max(int(float(u_next) * 2 ** 24), 0), 2 ** 24 - 1)
    mark, below = total * U // 2 ** 24, 0
    for v in range(V):
        below += r[v]
        if below > mark:
            return n, v
