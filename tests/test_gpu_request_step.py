"""A decode step of a batch of requests as a server runs it: projections with the
requests' adapters, rotated keys on their way into the pages, attention that reads the
shared prefix once, the output projection with its adapters; against float64 from the
same inputs, stage by stage, and one step after another in a graph."""
import math

import pytest
import torch

import lora_reference as lr
import paged_reference as ref
import rotary_reference as rr

pytestmark = pytest.mark.gpu
K, HEADS, KV, D, PAGE, PAIRS = 256, 8, 2, 64, 16, 16
SECTIONS = (6, 5, 5)


def _w4a16(g, N, K, dev):
    """(file-layout weight, scales, weights in float64) of a W4A16 projection."""
    w = torch.randn(N, K // 128, 128, generator=g) * K ** -0.5
    s = (w.abs().amax(2) / 7).half()
    q = torch.round(w / s.float()[:, :, None]).clamp(-7, 7)
    pairs = q.to(torch.int8).view(N, K // 2, 2).bitwise_and(15).view(torch.uint8)
    return (pairs[:, :, 0] | (pairs[:, :, 1] << 4)).to(dev), s.to(dev), (q.double() * s.double()[:, :, None]).view(N, K)


class Step:
    """Weights, adapters, a cache of three chats behind one prompt and two alone."""

    def __init__(self, dev, seed=3, B=5):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.g, self.B = dev, g, B
        self.Ns = (HEADS * D, KV * D, KV * D)
        self.qkv = [_w4a16(g, n, K, dev) for n in self.Ns]
        self.o = _w4a16(g, K, HEADS * D, dev)
        L, R = 3, 16
        self.a = [(torch.randn(L, R, k, generator=g) * k ** -0.5).bfloat16() for k in (K, K, K, HEADS * D)]
        self.b = [(torch.randn(L, n, R, generator=g) * 0.3).bfloat16() for n in (*self.Ns, K)]
        self.scales = torch.tensor([2.0, 0.5, 1.0])
        self.index = torch.tensor([0, 2, -1, 1, 0], dtype=torch.int32)
        # three chats share 40 tokens; room for more
        self.lens, self.shared = [60, 41, 55, 30, 3], 40
        W = 6
        tables = torch.arange(B * W).view(B, W).to(torch.int32)
        tables[1:3, :self.shared // PAGE] = tables[0, :self.shared // PAGE]
        self.k = torch.randn(B * W, KV, PAGE, D, generator=g).bfloat16()
        self.v = torch.randn(B * W, KV, PAGE // 8, D, 8, generator=g).bfloat16()
        for b in (1, 2):  # the prompt's last page is shared in part: the rest is copied
            i = self.shared // PAGE
            self.k[tables[b, i], :, :8] = self.k[tables[0, i], :, :8]
            self.v[tables[b, i], :, 0] = self.v[tables[0, i], :, 0]
        self.tables = tables
        self.freqs = (1e4 ** (-torch.arange(PAIRS, dtype=torch.float64) / PAIRS)).float()

    def upload(self):
        from cudalm_w4a16 import lora, rotary

        dev = self.dev
        self.gk, self.gv, self.gt = self.k.to(dev), self.v.to(dev), self.tables.to(dev)
        self.glens = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        self.cu = torch.tensor([0, 3], dtype=torch.int32, device=dev)
        self.gshared = torch.tensor([self.shared], dtype=torch.int32, device=dev)
        self.ga, self.gb = [t.to(dev) for t in self.a], [t.to(dev) for t in self.b]
        self.gs = self.scales.to(dev)
        self.rot = rotary.Rotary(self.freqs.to(dev), SECTIONS, turns=True)
        self.plan = lora.plan(self.index.to(dev), 3)

    def run(self, x, positions):
        """One step on the GPU: (q, k and v with adapters, rotated q, attention, output)."""
        import cudalm_w4a16 as w4
        from cudalm_w4a16 import lora, paged_kv as pk, rotary

        B = self.B
        ys = w4.gemv_multi([w[0] for w in self.qkv], [w[1] for w in self.qkv], x, self.Ns, K, B)
        base = [y.clone() for y in ys]
        q, k, v = lora.add(x, ys, self.ga[:3], self.gb[:3], self.plan, scales=self.gs)
        turned = rotary.append(q.view(B, HEADS, D), k.view(B, KV, D), v.view(B, KV, D), self.gk, self.gv, self.gt, self.glens,
                               self.rot, positions=positions)
        att = pk.decode_shared(turned, self.gk, self.gv, self.gt, self.glens, self.cu, self.gshared, max_shared=self.shared)
        flat = att.view(B, HEADS * D)
        y = w4.gemv(self.o[0], self.o[1], flat, K, HEADS * D, B)
        before = y.clone()
        lora.add(flat, y, self.ga[3], self.gb[3], self.plan, scales=self.gs)
        return base, (q, k, v), turned, att, before, y


def test_a_step_stage_by_stage(dev):
    s = Step(dev)
    s.upload()
    x = torch.randn(s.B, K, generator=s.g).bfloat16()
    # behind images a token's positions are not its place
    positions = torch.randint(0, 3000, (3, s.B), generator=s.g).to(torch.int32)
    base, qkv, turned, att, before, y = s.run(x.to(dev), positions.to(dev))
    for j, name in enumerate("qkv"):
        want = x.double() @ s.qkv[j][2].t()
        size = x.double().abs() @ s.qkv[j][2].abs().t()
        assert ((base[j].double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + K * 2.0 ** -23 * size).all(), name
        want, tol = lr.added(x, base[j].cpu(), s.a[j], s.b[j], s.index, s.scales)
        lr.check(qkv[j], want, tol, name)
    q, k, v = (t.cpu() for t in qkv)
    want, tol = rr.rotated(q.view(s.B, HEADS, D), positions, s.freqs, SECTIONS, True, False)
    rr.check(turned, want, tol, "rotated q")
    want, tol = rr.rotated(k.view(s.B, KV, D), positions, s.freqs, SECTIONS, True, False)
    gk, gv = s.gk.cpu(), s.gv.cpu()
    for b, n in enumerate(s.lens):
        at = s.tables[b, (n - 1) // PAGE].long()
        rr.check(gk[at, :, (n - 1) % PAGE], want[b], tol[b], "cached k")
        assert torch.equal(gv[at, :, (n - 1) % PAGE // 8, :, (n - 1) % 8], v.view(s.B, KV, D)[b])
    for b, n in enumerate(s.lens):
        pages = s.tables[b].long()
        keys = gk[pages].transpose(0, 1).reshape(KV, -1, D)[:, :n].transpose(0, 1)
        values = gv[pages].permute(1, 0, 2, 4, 3).reshape(KV, -1, D)[:, :n].transpose(0, 1)
        out, _, mag, big = ref.attention(turned[b:b + 1].cpu(), keys, values, torch.ones(n, dtype=torch.bool),
                                         torch.tensor([n - 1]), 1 / math.sqrt(D), 0, 0)
        ref.check_out(att[b:b + 1], out, mag, big, n, float(values.abs().max()), "bf16", D, b)
    want, tol = lr.added(att.view(s.B, -1).cpu(), before.cpu(), s.a[3], s.b[3], s.index, s.scales)
    lr.check(y, want, tol, "output")


def test_steps_of_a_graph(dev):
    """Four steps by replays of one graph, eager work between them, against four eager steps."""
    import cudalm_w4a16 as w4

    def steps(graphed):
        s = Step(dev)
        s.upload()
        g = torch.Generator(device=dev).manual_seed(7)
        x = torch.zeros(s.B, K, dtype=torch.bfloat16, device=dev)
        positions = torch.zeros(3, s.B, dtype=torch.int32, device=dev)
        graph, held = torch.cuda.CUDAGraph(), None
        if graphed:
            keep = s.gk.clone(), s.gv.clone()
            s.run(x, positions)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                held = s.run(x, positions)
            s.gk.copy_(keep[0]), s.gv.copy_(keep[1])
        outs = []
        for i in range(4):
            x.normal_(generator=g)
            positions += 1
            s.glens += 1
            if graphed:
                graph.replay()
            else:
                held = s.run(x, positions)
            outs.append((held[3].clone(), held[5].clone()))
            # other work of the program
            w4.gemv(s.o[0], s.o[1], torch.randn(2, HEADS * D, device=dev).bfloat16(), K, HEADS * D, 2)
            torch.cuda.synchronize()
        return outs, s.gk, s.gv

    eager, replayed = steps(False), steps(True)
    for i, (p, q) in enumerate(zip(eager[0], replayed[0])):
        assert torch.equal(p[0], q[0]) and torch.equal(p[1], q[1]), i
    assert torch.equal(eager[1], replayed[1]) and torch.equal(eager[2], replayed[2])
