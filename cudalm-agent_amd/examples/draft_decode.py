"""Text generation with drafted tokens over a paged cache, on random weights.

A small decoder of the hybrid model's full-attention layers (hidden size 1024, 8
query heads on 2 key-value heads of 256 with an output gate, MLP 3584, bf16 head;
no positions and no tokenizer) runs every operator where a server would:

  prompt   projections of all tokens -> append -> prefill
  step     drafted tokens from an earlier occurrence of the last token ->
           projections of all of them -> append -> decode (with the weight that every
           cached token receives) -> logits -> verify -> accepted tokens + 1
  cache    past `budget` tokens: evict to half of it, into fresh pages

    python cudalm-agent_amd/examples/draft_decode.py
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import cudalm_w4a16 as w4  # noqa: E402
from cudalm_w4a16 import draft, paged_kv  # noqa: E402

HIDDEN, HEADS, KV, D, INTER = 1024, 8, 2, 256, 3584


def _packed(gen, N, K):
    """A W4A16 projection of N(0, 0.03) weights, repacked."""
    w = torch.randn(N, K // 128, 128, device="cuda", generator=gen) * 0.03
    s = (w.abs().amax(dim=2) / 7).to(torch.float16)
    q = torch.round(w / s.float()[:, :, None]).clamp_(-7, 7).to(torch.int8).view(N, K // 2, 2)
    q = q.bitwise_and_(15).view(torch.uint8)
    return w4.repack(q[:, :, 0] | (q[:, :, 1] << 4), s, N, K)


def _norm(x):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Decoder:
    def __init__(self, layers=2, vocab=4096, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.vocab = vocab
        self.embed, self.head = (torch.randn(vocab, HIDDEN, device="cuda", generator=g).to(torch.bfloat16)
                                 for _ in range(2))
        self.layers = [{
            "qkv": [_packed(g, n, HIDDEN) for n in (2 * HEADS * D, KV * D, KV * D)],
            "o": _packed(g, HIDDEN, HEADS * D),
            "gate": _packed(g, INTER, HIDDEN), "up": _packed(g, INTER, HIDDEN),
            "down": _packed(g, HIDDEN, INTER)} for _ in range(layers)]

    def __call__(self, tokens, caches, attend):
        """Logits [T, vocab] of token ids [T]; attend(layer, q, k, v) is the mixer."""
        x = self.embed[tokens]
        T = x.shape[0]
        for i, w in enumerate(self.layers):
            q, k, v = w4.gemv_multi(w["qkv"], None, _norm(x), (2 * HEADS * D, KV * D, KV * D), HIDDEN, T,
                                    prepacked=True)
            # every head's queries and its gate lie side by side: a strided view is read as it is
            q, gate = q.view(T, HEADS, 2 * D).split(D, dim=2)
            a = attend(caches[i], q, k.view(T, KV, D), v.view(T, KV, D)) * torch.sigmoid(gate)
            x = x + w4.gemv_prepacked(w["o"], a.view(T, HEADS * D), HIDDEN, HEADS * D, T).view(T, HIDDEN)
            m = w4.swiglu(w["gate"], None, w["up"], None, _norm(x), INTER, HIDDEN, T, prepacked=True)
            x = x + w4.gemv_prepacked(w["down"], m.view(T, INTER), HIDDEN, INTER, T).view(T, HIDDEN)
        return w4.bf16_gemv_any(self.head, _norm(x), self.vocab, HIDDEN, T).view(T, self.vocab)


class Chat:
    """One sequence: its pages in every layer's cache (the same page numbers)."""

    def __init__(self, model, capacity=4096, page=16, budget=None, window=0, sinks=4):
        self.model, self.page, self.budget, self.window, self.sinks = model, page, budget, window, sinks
        pages = 2 * (capacity // page)
        self.caches = [paged_kv.empty_cache(pages, page, KV, D, torch.bfloat16, weights=True)
                       for _ in model.layers]
        self.free = list(range(pages))
        self.pages, self.length = [], 0

    def _tables(self, new):
        """Room for `new` more tokens; (tables, lens) with them."""
        self.length += new
        while len(self.pages) * self.page < self.length:
            self.pages.append(self.free.pop())
        return (torch.tensor([self.pages], dtype=torch.int32, device="cuda"),
                torch.tensor([self.length], dtype=torch.int32, device="cuda"))

    def prompt(self, tokens):
        T = len(tokens)
        tables, lens = self._tables(T)
        cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")

        def attend(cache, q, k, v):
            paged_kv.append(k, v, *cache[:2], tables, lens, cu_new=cu, weights=cache[2])
            return paged_kv.prefill(q, cu, *cache[:2], tables, lens, window=self.window, sinks=self.sinks)

        return self.model(torch.tensor(tokens, device="cuda"), self.caches, attend)

    def step(self, tokens):
        """Logits after each of the last accepted token and the drafted ones."""
        tables, lens = self._tables(len(tokens))

        def attend(cache, q, k, v):
            paged_kv.append(k, v, *cache[:2], tables, lens, weights=cache[2])
            return paged_kv.decode(q[None], *cache[:2], tables, lens, window=self.window, sinks=self.sinks,
                                   weights=cache[2], max_len=self.length)[0]

        return self.model(torch.tensor(tokens, device="cuda"), self.caches, attend)

    def forget(self, count):
        """Takes back the last tokens, whose drafts were refused (what their queries added to the
        weights of others stays)."""
        self.length -= count

    def evict(self):
        """Past the budget: half of it stays, in fresh pages."""
        if self.budget is None or self.length <= self.budget:
            return
        keep = self.budget // 2
        fresh = [self.free.pop() for _ in range(-(-keep // self.page))]
        tables = torch.tensor([self.pages], dtype=torch.int32, device="cuda")
        lens = torch.tensor([self.length], dtype=torch.int32, device="cuda")
        dst = torch.tensor([fresh], dtype=torch.int32, device="cuda")
        for k, v, weights in self.caches:
            paged_kv.evict(k, v, tables, lens, weights, dst, keep, sinks=self.sinks, recent=16,
                           max_len=self.length)
        self.free += self.pages
        self.pages, self.length = fresh, keep


def _guess(history, count):
    """The tokens after the last earlier occurrence of the newest one that has so many."""
    for i in range(len(history) - 1 - max(count, 1), -1, -1):
        if history[i] == history[-1]:
            return history[i + 1:i + 1 + count]
    return []


def generate(model, prompt, count, drafts=4, temperature=0.0, seed=0, **chat):
    """(`count` tokens after `prompt`, model steps taken, the chat). Without a budget, drafted
    tokens change neither the most likely continuation (temperature 0) nor, otherwise, the
    distribution of the text, only the number of steps. With one they do: the weights that
    eviction goes by are summed before verification, over the queries of refused tokens too,
    and evictions come after steps of another length."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    chat = Chat(model, **chat)
    history, steps = list(prompt), 0
    logits = chat.prompt(prompt)[-1:]
    guess = []
    while True:
        # the target's probabilities after the last accepted token and each drafted one
        if temperature == 0:
            target = torch.nn.functional.one_hot(logits.float().argmax(-1), model.vocab).float()
        else:
            target = torch.softmax(logits.float() / temperature, dim=-1)
        n = len(guess)
        out, accepted = draft.verify(target[None], None, torch.tensor([guess], dtype=torch.int32, device="cuda").view(1, n),
                                     torch.rand(1, n, device="cuda", generator=g),
                                     torch.rand(1, device="cuda", generator=g))
        taken = int(accepted[0])
        history += out[0, :taken + 1].tolist()
        chat.forget(n - taken)
        if len(history) >= len(prompt) + count:
            return history[len(prompt):len(prompt) + count], steps, chat
        chat.evict()
        guess = _guess(history, drafts)
        logits = chat.step(history[-1:] + guess)
        steps += 1


def main():
    model = Decoder()
    prompt = torch.randint(0, model.vocab, (500,), generator=torch.Generator().manual_seed(1)).tolist()
    for name, more in (("one token a step", dict(drafts=0)), ("four drafted tokens", dict(drafts=4)),
                       ("with a budget of 512 cached tokens", dict(drafts=4, budget=512)),
                       ("with a window of 256 tokens and 4 sinks", dict(drafts=4, window=256))):
        generate(model, prompt, 4, **more)
        torch.cuda.synchronize()
        start = time.perf_counter()
        tokens, steps, chat = generate(model, prompt, 200, **more)
        torch.cuda.synchronize()
        print(f"{name}: {len(tokens)} tokens in {steps} steps, {1e3 * (time.perf_counter() - start):.0f} ms, "
              f"{chat.length} cached; first {tokens[:8]}", flush=True)


if __name__ == "__main__":
    main()
