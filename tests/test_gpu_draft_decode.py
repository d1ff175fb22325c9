"""The example's generation loop: append, prefill, decode, evict and verify
together with the projections and the head. Drafted tokens must not change
the greedy continuation beyond the rounding of logits."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cudalm-agent_amd", "examples",
                    "draft_decode.py")


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("draft_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("window", [0, 40])
def test_drafts_keep_the_greedy_text(ex, dev, window):
    model = ex.Decoder(seed=3)
    prompt = torch.randint(0, model.vocab, (70,), generator=torch.Generator().manual_seed(2)).tolist()
    tokens, steps, _ = ex.generate(model, prompt, 60, drafts=4, window=window)
    assert len(tokens) == 60 and steps <= 60
    # all logits again, in one prefill: every token is the best one up to the rounding of
    # bf16 logits and hidden states (a few units of 2^-8 of the largest logit)
    logits = ex.Chat(model, window=window).prompt(prompt + tokens).float()
    at = logits[len(prompt) - 1:-1]
    best = at.max(dim=1).values
    got = at.gather(1, torch.tensor(tokens, device=dev)[:, None])[:, 0]
    assert bool((best - got <= 8 * 2.0 ** -8 * at.abs().max()).all())


def test_budget(ex, dev):
    model = ex.Decoder(layers=1, seed=4)
    prompt = torch.randint(0, model.vocab, (100,), generator=torch.Generator().manual_seed(2)).tolist()
    tokens, _, chat = ex.generate(model, prompt, 150, drafts=3, temperature=1.0, budget=128, capacity=512)
    assert all(0 <= t < model.vocab for t in tokens)
    assert chat.length <= 128 + 4 and len(chat.free) + len(chat.pages) == 2 * 512 // 16
