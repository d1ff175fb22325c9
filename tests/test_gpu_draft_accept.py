"""The example's generation loop on a model whose text repeats: drafted tokens are accepted, and
leave the text as it is."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cudalm-agent_amd", "examples",
                    "draft_decode.py")
WORDS = 64


@pytest.fixture(scope="module")
def model(dev):
    spec = importlib.util.spec_from_file_location("draft_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    m = mod.Decoder(vocab=WORDS, seed=5)
    # the head likes the word after the one that came in: next to embeddings of size 16 the
    # layers' outputs, of size 1, do not change the best
    m.head = m.embed.roll(1, 0).contiguous()
    m.embed = m.embed * 16
    m.generate = lambda *a, **k: mod.generate(m, *a, **k)
    return m


@pytest.mark.parametrize("window", [0, 40])
def test_accepted_drafts_save_steps(model, window):
    prompt = [t % WORDS for t in range(130)]
    text = [t % WORDS for t in range(130, 190)]
    tokens, steps, _ = model.generate(prompt, 60, drafts=0, window=window)
    assert tokens == text and steps == 59  # the first one comes from the prompt
    tokens, steps, chat = model.generate(prompt, 60, drafts=4, window=window)
    assert tokens == text and steps == 12 and chat.length >= 130 + 59


def test_refused_drafts_leave_the_text(model):
    """A prompt that names other words after each: what it suggests is refused."""
    prompt = [0, 2, 0, 5, 1, 7, 1, 9, 2, 4, 2, 8, 3, 1, 3, 3, 0]
    tokens, steps, chat = model.generate(prompt, 30, drafts=4)
    assert tokens == [t % WORDS for t in range(1, 31)]
    assert steps == 29
    assert chat.length == len(prompt) + 29
