"""The work whose speed is measured around the paged key-value cache of the
full-attention layers and around drafted tokens, and the ranges it stands for.

Operators (package cudalm_w4a16, modules paged_kv and draft):
  append   new tokens' keys and values into the pages of their sequences
  decode   attention of one or a few new tokens of every sequence over its
           pages, split over the length and joined, optionally with a sliding
           window and sinks, optionally with the attention weight that every
           cached token received
  prefill  the same attention for a chunk of every sequence's tokens
  evict    the tokens that keep their place, by accumulated attention weight,
           and their compaction into fresh pages
  verify   acceptance of drafted tokens against the target's probabilities
           and the token that follows the accepted ones

Layouts: keys [pages, kv heads, page size, D], values [pages, kv heads, page
size/8, D, 8], weights [pages, kv heads, page size] in fp32. Head shapes
are those of the 24-layer hybrid decoder (8 query heads on 2 key-value heads
of 256) and generic ones; the vocabulary is its LM head's.
"""
import os
import sys

import torch

own = False  # False: the plain forms; True: this package's operators

VOCAB = 248320
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one new token of one chat: the smallest call, where latency counts
        {"name": "decode_one", "kind": "decode", "B": 1, "Q": 1, "heads": 8, "kv": 2, "D": 256, "page": 16,
         "len": 777, "window": 0, "sinks": 0, "weights": False, "type": "bf16"},
        # a decode step of 64 sequences of mixed lengths
        {"name": "decode_batch", "kind": "decode", "B": 64, "Q": 1, "heads": 8, "kv": 2, "D": 256, "page": 64,
         "len": 8192, "window": 0, "sinks": 0, "weights": False, "type": "bf16"},
        # four drafted tokens and the last accepted one of 16 sequences, with
        # the weight of every cached token for a later eviction
        {"name": "decode_draft_scores", "kind": "decode", "B": 16, "Q": 5, "heads": 32, "kv": 8, "D": 128, "page": 32,
         "len": 5001, "window": 0, "sinks": 0, "weights": True, "type": "f16"},
        # a short prompt, whole
        {"name": "prefill_short", "kind": "prefill", "B": 1, "new": 100, "heads": 8, "kv": 2, "D": 256, "page": 16,
         "ctx": 0, "window": 0, "sinks": 0, "type": "bf16"},
        # prompts of mixed lengths with earlier context, sliding window and sinks
        {"name": "prefill_window", "kind": "prefill", "B": 8, "new": 1000, "heads": 32, "kv": 8, "D": 128, "page": 32,
         "ctx": 1500, "window": 512, "sinks": 4, "type": "f16"},
        # a chunk of a long document: the largest
        {"name": "prefill_long", "kind": "prefill", "B": 1, "new": 2048, "heads": 8, "kv": 2, "D": 256, "page": 64,
         "ctx": 14336, "window": 0, "sinks": 0, "type": "bf16"},
        # the keys and values of one new token of 32 sequences
        {"name": "append_decode", "kind": "append", "B": 32, "new": 1, "kv": 2, "D": 256, "page": 16, "ctx": 2000,
         "weights": False, "type": "bf16"},
        # those of eight prompts
        {"name": "append_prompts", "kind": "append", "B": 8, "new": 2001, "kv": 8, "D": 128, "page": 32, "ctx": 333,
         "weights": True, "type": "f16"},
        # a few chats cut to a quarter
        {"name": "evict_chats", "kind": "evict", "B": 4, "kv": 2, "D": 256, "page": 16, "len": 4096, "keep": 1024,
         "sinks": 4, "recent": 64, "type": "bf16"},
        # long documents cut to fit
        {"name": "evict_long", "kind": "evict", "B": 12, "kv": 8, "D": 128, "page": 64, "len": 30000, "keep": 8000,
         "sinks": 4, "recent": 256, "type": "f16"},
        # four drafted tokens of one chat
        {"name": "verify_one", "kind": "verify", "B": 1, "draft": 4, "V": VOCAB, "greedy": False, "type": "f32"},
        # seven drafted tokens of 64 sequences
        {"name": "verify_batch", "kind": "verify", "B": 64, "draft": 7, "V": VOCAB, "greedy": False, "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    hi = max(lo, int(hi))
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


HEADS = [(8, 2), (8, 2), (32, 8), (8, 8), (16, 1), (12, 4), (40, 8)]


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "prefill", "prefill", "append", "evict", "verify"])
    heads, kv = rng.choice(HEADS)
    D = rng.choice([64, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "f16"])
    # now and then a sliding window with a few sinks
    window, sinks = (_log_int(rng, 16, 4096), rng.choice([0, 1, 4, 16, 40])) if rng.random() < 0.4 else (0, 0)
    if kind == "decode":
        B, Q = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5, 8])
        # at most half of the values that the largest listed batch caches
        top = 2 ** 27 // (B * kv * D)
        return {"kind": kind, "B": B, "Q": Q, "heads": heads, "kv": kv, "D": D, "page": page,
                "len": _log_int(rng, Q, min(32768, top)), "window": window, "sinks": sinks,
                "weights": rng.random() < 0.25, "type": dtype}
    if kind == "prefill":
        B = _log_int(rng, 1, 8)
        new = _log_int(rng, 9, 2048 // B)
        ctx = rng.choice([0, _log_int(rng, 1, 12288 // B)])
        # at most two thirds of the scores of the longest listed chunk
        ctx = max(0, min(ctx, int(1.8e8 / (B * heads * new)) - new))
        return {"kind": kind, "B": B, "new": new, "heads": heads, "kv": kv, "D": D, "page": page, "ctx": ctx,
                "window": window, "sinks": sinks, "type": dtype}
    if kind == "append":
        B = _log_int(rng, 1, 64)
        return {"kind": kind, "B": B, "new": _log_int(rng, 1, 8192 // B), "kv": kv, "D": D, "page": page,
                "ctx": _log_int(rng, 1, 4096), "weights": rng.random() < 0.5, "type": dtype}
    if kind == "evict":
        B = _log_int(rng, 1, 16)
        top = _log_int(rng, 64, min(32768, 2 ** 27 // (B * kv * D)))
        return {"kind": kind, "B": B, "kv": kv, "D": D, "page": page, "len": top, "keep": _log_int(rng, 16, top),
                "sinks": rng.choice([0, 4, 16]), "recent": rng.choice([0, 1, 32, 128]), "type": dtype}
    return {"kind": kind, "B": _log_int(rng, 1, 32), "draft": rng.randint(1, 8),
            "V": rng.choice([VOCAB, _log_int(rng, 1000, VOCAB)]), "greedy": rng.random() < 0.25,
            "type": rng.choice(["f32", "f32", "bf16", "f16"])}


# --- sizes that follow from a case ------------------------------------------------

def _ragged(n, top, least=1):
    """n whole numbers from `top` down to about a quarter of it, in mixed order."""
    return [max(least, top - (i * 7 % n) * 3 * top // (4 * n)) for i in range(n)]


def _lens(case):
    """(tokens in the cache, new ones among them) of every sequence."""
    B = case["B"]
    if case["kind"] == "decode":
        return _ragged(B, case["len"], case["Q"]), [case["Q"]] * B
    if case["kind"] == "evict":
        return _ragged(B, case["len"]), [0] * B
    new = [case["new"]] * B if case["new"] == 1 else _ragged(B, case["new"])
    ctx = _ragged(B, case["ctx"], 0)
    return [c + n for c, n in zip(ctx, new)], new


def _seen(length, new, window, sinks):
    """(tokens that at least one new token sees, sum over the new ones of those each sees)."""
    first, total = length - new, 0
    if window <= 0:
        return length, sum(range(first + 1, length + 1))
    for p in range(first, length):
        total += min(window, p + 1) + min(sinks, max(0, p + 1 - window))
    return min(length, new + window - 1) + min(sinks, max(0, length - new - window + 1)), total


def work(case):
    """Visible keys and values read once, queries read and outputs written
    once; copied tokens read and written once; the probabilities of the row
    that gives the next token and of the drafted tokens."""
    kind = case["kind"]
    if kind == "verify":
        size = 4 if case["type"] == "f32" else 2
        rows = 1 if case["greedy"] else 2  # the target's row, and the draft's
        n = case["B"] * (rows * case["V"] + 2 * case["draft"])
        return {"bytes": n * size + case["B"] * (case["draft"] * 12 + 12), "flops": 2 * case["B"] * case["V"]}
    lens, new = _lens(case)
    token = 4 * case["kv"] * case["D"]  # bytes of a token's key and value
    slot = 4 * case["kv"]  # of its weights
    if kind == "append":
        n = sum(new)
        return {"bytes": 2 * n * token + (n * slot if case["weights"] else 0), "flops": 0}
    if kind == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        return {"bytes": sum(lens) * slot + kept * (2 * token + 2 * slot), "flops": 0}
    seen = [_seen(n, m, case["window"], case["sinks"]) for n, m in zip(lens, new)]
    w = sum(lens) * slot if kind == "decode" and case["weights"] else 0
    return {"bytes": sum(s for s, _ in seen) * token + 4 * sum(new) * case["heads"] * case["D"] + w,
            "flops": 4 * sum(t for _, t in seen) * case["heads"] * case["D"]}


# --- inputs -----------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(gen, lens, page, skip=0):
    """Page numbers of every sequence, in random order, -1 past its end."""
    need = _int32([-(-n // page) for n in lens])
    width = max(-(-n // page) for n in lens)
    total = int(sum(-(-n // page) for n in lens))
    at = torch.arange(width, device="cuda")[None, :] < need[:, None]
    t = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    t[at] = torch.randperm(total, generator=gen, device="cuda").to(torch.int32) + skip
    return t, total


def prepare(case, seed):
    gen, kind = _gen(seed), case["kind"]
    if kind == "verify":
        return _prepare_verify(case, gen)
    dtype, page, kv, D = DTYPES[case["type"]], case["page"], case["kv"], case["D"]
    lens, new = _lens(case)
    tables, total = _tables(gen, lens, page)
    st = {**case, "tables": tables, "lens": _int32(lens), "max_len": max(lens), "max_new": max(new)}
    pages = total + 3  # a pool has free pages
    if kind == "evict":
        kept = [min(n, case["keep"]) for n in lens]
        st["dst"], more = _tables(gen, kept, page, skip=total)
        pages = total + more
    st["k"] = _randn(gen, pages, kv, page, D, dtype=dtype)
    st["v"] = _randn(gen, pages, kv, page // 8, D, 8, dtype=dtype)
    st["w"] = None
    if kind == "evict":  # a heavy tail: few tokens draw most of the attention
        st["w"] = _randn(gen, pages, kv, page, dtype=torch.float32).mul_(2).exp_()
    elif case.get("weights"):
        st["w"] = torch.zeros(pages, kv, page, device="cuda")
    if kind == "decode":
        st["q"] = _randn(gen, case["B"], case["Q"], case["heads"], D, dtype=dtype)
        st["out"] = torch.empty_like(st["q"])
    else:
        st["cu"] = _int32([sum(new[:i]) for i in range(len(new) + 1)])
    if kind == "prefill":
        st["q"] = _randn(gen, sum(new), case["heads"], D, dtype=dtype)
        st["out"] = torch.empty_like(st["q"])
    if kind == "append":
        st["nk"] = _randn(gen, sum(new), kv, D, dtype=dtype)
        st["nv"] = _randn(gen, sum(new), kv, D, dtype=dtype)
    return st


def _prepare_verify(case, gen):
    """Probabilities of a model and of a smaller one that mostly agrees, and
    tokens drawn from the latter."""
    B, G, V, dtype = case["B"], case["draft"], case["V"], DTYPES[case["type"]]
    logits = torch.empty(B, G + 1, V, device="cuda").normal_(0, 2.5, generator=gen)
    target = torch.softmax(logits, dim=2).to(dtype)
    noise = torch.empty(B, G, V, device="cuda").normal_(0, 0.5, generator=gen)
    logits = logits[:, :G] + noise
    noise.exponential_(generator=gen)
    # drawn from softmax(logits): the largest of logits + Gumbel noise
    tokens = (logits - noise.log_()).argmax(dim=2).to(torch.int32)
    draft = None if case["greedy"] else torch.softmax(logits, dim=2).to(dtype)
    return {**case, "target": target, "draft_p": draft, "tokens": tokens,
            "u": torch.rand(B, G, device="cuda", generator=gen), "u_next": torch.rand(B, device="cuda", generator=gen)}


# --- the plain forms ----------------------------------------------------------------

def _dense(st, cache, keys):
    """[B, kv heads, width * page, D] of a cache through the tables, in fp32."""
    x = cache[st["tables"].clamp(min=0).long()]  # [B, width, kv, ...]
    x = x.permute(0, 2, 1, 3, 4) if keys else x.permute(0, 2, 1, 3, 5, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, st["D"]).float()


def _plain_attention(st, q, pos):
    """q [B, n, heads, D] at positions pos [B, n] (negative: no such token):
    (outputs like q in fp32, weights [B, kv heads, width * page])."""
    B, n, H, D = q.shape
    kv = st["kv"]
    k, v = _dense(st, st["k"], True), _dense(st, st["v"], False)
    L = k.shape[2]
    s = q.float().view(B, n, kv, H // kv, D).permute(0, 2, 3, 1, 4).reshape(B, kv, -1, D)
    s = torch.matmul(s * D ** -0.5, k.transpose(2, 3)).view(B, kv, H // kv, n, L)
    del k
    t = torch.arange(L, device="cuda")
    see = t[None, None, :] <= pos[:, :, None]
    if st["window"] > 0:
        see &= (t[None, None, :] > pos[:, :, None] - st["window"]) | (t < st["sinks"])
    see = see[:, None, None]
    s.masked_fill_(~see, float("-inf"))
    s -= s.amax(dim=4, keepdim=True).clamp_(min=-3e38)
    s.exp_()
    s /= s.sum(dim=4, keepdim=True).clamp_(min=1e-30)
    o = torch.matmul(s.view(B, kv, -1, L), v).view(B, kv, H // kv, n, D)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, H, D), s


def _slots(st, mask):
    """(page, place in it) of the tokens of mask [B, width * page]."""
    b, t = mask.nonzero(as_tuple=True)
    return st["tables"][b, t // st["page"]].long(), t % st["page"]


def _plain_decode(st):
    n, Q = st["lens"].long(), st["Q"]
    pos = n[:, None] - Q + torch.arange(Q, device="cuda")
    o, s = _plain_attention(st, st["q"], pos)
    out = o.to(st["q"].dtype)
    if st["w"] is None:
        return out
    w = s.sum(dim=(2, 3))  # [B, kv, L]
    has = torch.arange(w.shape[2], device="cuda") < n[:, None]
    at, off = _slots(st, has)
    st["w"][at, :, off] = w.transpose(1, 2)[has]
    return [out, st["w"]]


def _plain_prefill(st):
    cu = st["cu"].long()
    new = cu[1:] - cu[:-1]
    i = torch.arange(st["max_new"], device="cuda")
    real = i < new[:, None]
    q = st["q"][(cu[:-1, None] + i).clamp(max=st["q"].shape[0] - 1)]
    pos = torch.where(real, st["lens"].long()[:, None] - new[:, None] + i, -1)
    o, _ = _plain_attention(st, q, pos)
    return o[real].to(st["q"].dtype)


def _plain_append(st):
    cu = st["cu"].long()
    new = cu[1:] - cu[:-1]
    b = torch.repeat_interleave(torch.arange(st["B"], device="cuda"), new, output_size=st["nk"].shape[0])
    t = st["lens"].long()[b] - new[b] + torch.arange(b.shape[0], device="cuda") - cu[b]
    at, off = st["tables"][b, t // st["page"]].long(), t % st["page"]
    st["k"][at, :, off] = st["nk"]
    st["v"][at, :, off // 8, :, off % 8] = st["nv"]
    if st["w"] is None:
        return [st["k"], st["v"]]
    st["w"][at, :, off] = 0.0
    return [st["k"], st["v"], st["w"]]


def _plain_evict(st):
    B, kv, page, keep = st["B"], st["kv"], st["page"], st["keep"]
    n = st["lens"].long()[:, None, None]
    w = st["w"][st["tables"].clamp(min=0).long()].permute(0, 2, 1, 3).reshape(B, kv, -1)
    t = torch.arange(w.shape[2], device="cuda")
    s = min(st["sinks"], keep)
    held = (t < s) | (t >= n - min(st["recent"], keep - s))
    w = torch.where(held, float("inf"), w).masked_fill(t >= n, float("-inf"))
    # equal weights: the earlier token first
    order = torch.sort(w, dim=2, descending=True, stable=True).indices[:, :, :keep]
    many = n.clamp(max=keep)
    i = torch.arange(order.shape[2], device="cuda")
    kept = torch.sort(torch.where(i < many, order, t.shape[0]), dim=2).values
    kept = torch.where(i < many, kept, -1)
    b, h, j = (kept >= 0).nonzero(as_tuple=True)
    src = kept[b, h, j]
    at, off = st["tables"][b, src // page].long(), src % page
    to, place = st["dst"][b, j // page].long(), j % page
    st["k"][to, h, place] = st["k"][at, h, off]
    st["v"][to, h, place // 8, :, place % 8] = st["v"][at, h, off // 8, :, off % 8]
    st["w"][to, h, place] = st["w"][at, h, off]
    wide = torch.full((B, kv, keep), -1, dtype=torch.int32, device="cuda")
    wide[:, :, :kept.shape[2]] = kept
    return [wide, many.view(-1).to(torch.int32), st["k"], st["v"], st["w"]]


def _plain_verify(st):
    B, G, V = st["B"], st["draft"], st["V"]
    x = st["tokens"].long()
    b = torch.arange(B, device="cuda")
    p = torch.gather(st["target"][:, :G], 2, x[:, :, None])[:, :, 0].float()
    q = torch.ones_like(p) if st["draft_p"] is None else torch.gather(st["draft_p"], 2, x[:, :, None])[:, :, 0].float()
    n = torch.cumprod((st["u"] * q < p).long(), dim=1).sum(dim=1)
    # probabilities in units of 2^-40: whole numbers, whose sums have no order
    unit = 2.0 ** 40
    row = st["target"][b, n].float()
    whole = (row.clamp(0.0, 1.0) * unit).long()
    at = n.clamp(max=G - 1)
    if st["draft_p"] is None:
        less = torch.zeros_like(row)
        less[b, x[b, at]] = 1.0
    else:
        less = st["draft_p"][b, at].float()
    rest = ((row - less).clamp(0.0, 1.0) * unit).long()
    rest = torch.where(((n < G) & (rest.sum(dim=1) > 0))[:, None], rest, whole)
    below = rest.cumsum(dim=1)
    total = below[:, -1]
    U = (st["u_next"] * 2.0 ** 24).long().clamp(0, 2 ** 24 - 1)
    mark = (total >> 24) * U + (((total & (2 ** 24 - 1)) * U) >> 24)
    token = (below <= mark[:, None]).sum(dim=1)
    i = torch.arange(G + 1, device="cuda")
    out = torch.full((B, G + 1), -1, dtype=torch.int64, device="cuda")
    out[:, :G] = torch.where(i[:G] < n[:, None], x, -1)
    out[b, n] = torch.where(total > 0, token, -1)
    return [out.to(torch.int32), n.to(torch.int32)]


PLAIN = {"decode": _plain_decode, "prefill": _plain_prefill, "append": _plain_append, "evict": _plain_evict,
         "verify": _plain_verify}


# --- the package's operators ----------------------------------------------------------

def _modules():
    pkg = os.path.join(os.getcwd(), "cudalm-agent_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from cudalm_w4a16 import draft, paged_kv
    return paged_kv, draft


def _own(st):
    paged_kv, draft = _modules()
    kind = st["kind"]
    if kind == "verify":
        return list(draft.verify(st["target"], st["draft_p"], st["tokens"], st["u"], st["u_next"]))
    pages = (st["k"], st["v"], st["tables"], st["lens"])
    if kind == "append":
        paged_kv.append(st["nk"], st["nv"], *pages, cu_new=st["cu"], weights=st["w"])
        return [st["k"], st["v"]] + ([] if st["w"] is None else [st["w"]])
    if kind == "evict":
        kept, lens = paged_kv.evict(*pages, st["w"], st["dst"], st["keep"], sinks=st["sinks"], recent=st["recent"],
                                    max_len=st["max_len"])
        return [kept, lens, st["k"], st["v"], st["w"]]
    if kind == "decode":
        paged_kv.decode(st["q"], *pages, window=st["window"], sinks=st["sinks"], weights=st["w"], accumulate=False,
                        max_len=st["max_len"], out=st["out"])
        return st["out"] if st["w"] is None else [st["out"], st["w"]]
    return paged_kv.prefill(st["q"], st["cu"], *pages, window=st["window"], sinks=st["sinks"],
                            max_len=st["max_len"], out=st["out"])


def run(state):
    return _own(state) if own else PLAIN[state["kind"]](state)


# --- 64-bit results -------------------------------------------------------------------

def exact(case, seed):
    """Attention by its definition, a sequence and a key-value head at a time.
    Copied values and whole numbers have none."""
    if case["kind"] not in ("decode", "prefill"):
        return None
    st = prepare(case, seed)
    decode = case["kind"] == "decode"
    lens, new = _lens(case)
    H, kv, D, page = case["heads"], case["kv"], case["D"], case["page"]
    q = st["q"].reshape(-1, H, D)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    w = None if st["w"] is None else st["w"].double()
    at = 0
    for b, (length, m) in enumerate(zip(lens, new)):
        ids = st["tables"][b, :-(-length // page)].long()
        p = torch.arange(length - m, length, device="cuda")[:, None]
        t = torch.arange(length, device="cuda")[None, :]
        hidden = t > p
        if case["window"] > 0:
            hidden = hidden | ((p - t >= case["window"]) & (t >= case["sinks"]))
        for h in range(kv):
            keys = st["k"][ids, h].double().reshape(-1, D)[:length]
            values = st["v"][ids, h].double().transpose(2, 3).reshape(-1, D)[:length]
            received = torch.zeros(length, dtype=torch.float64, device="cuda")
            for g in range(h * (H // kv), (h + 1) * (H // kv)):
                s = q[at:at + m, g].double() @ keys.t() / D ** 0.5
                e = torch.exp(s - s.masked_fill(hidden, -1e300).max(dim=1, keepdim=True).values).masked_fill(hidden, 0.0)
                e = e / e.sum(dim=1, keepdim=True)
                out[at:at + m, g] = e @ values
                received += e.sum(dim=0)
            if w is not None:
                full = torch.zeros(ids.numel() * page, dtype=torch.float64, device="cuda")
                full[:length] = received
                spots = (torch.arange(ids.numel() * page, device="cuda") < length).view(-1, page)
                block = w[ids, h]
                block[spots] = full.view(-1, page)[spots]
                w[ids, h] = block
        at += m
    out = out.view(st["q"].shape)
    return out if not decode or w is None else [out, w]
