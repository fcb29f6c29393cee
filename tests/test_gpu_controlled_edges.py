"""Generation with controls where it ends early or its callbacks keep what they were given."""

import numpy as np
import pytest

import llm_b200
from llm_b200 import synth


@pytest.fixture(scope="module")
def gpu_model():
    g = llm_b200.GPU(synth.ensure("tiny-qwen2"), ctx=256)
    yield g
    g.close()


@pytest.mark.gpu
def test_times_of_a_generation_without_tokens(gpu_model):
    """The prompt's time is the prefill's, not the decoding's, also where nothing is generated."""
    g = gpu_model
    prompt = synth.prompt_ids(g.cfg.vocab, 200, seed=2)
    g.generate_controlled(prompt, 1)
    for kw in (dict(n=0), dict(n=5, mask=lambda tokens, words: False)):
        got, tm = g.generate_controlled(prompt, **kw)
        assert len(got) == 0 and tm.generated == 0 and tm.prompt_tokens == 200
        assert tm.prefill_ms > 0 and tm.prefill_ms >= tm.gpu_prefill_ms * 0.9 and tm.decode_ms < tm.prefill_ms


@pytest.mark.gpu
def test_a_mask_that_is_kept_is_the_callbacks_own():
    """The words a mask callback fills are its own memory: they outlive the model."""
    g = llm_b200.GPU(synth.ensure("tiny-qwen2"), ctx=64)
    kept = []

    def mask(tokens, words):
        words[:] = 0
        words[1] = 1 << 5  # token 37
        kept.append(words)
        return True

    got, _ = g.generate_controlled(synth.prompt_ids(g.cfg.vocab, 10, seed=1), 3, mask=mask)
    g.close()
    assert got.tolist() == [37] * 3
    assert all(w.flags.owndata and w.dtype == np.uint32 for w in kept)
    kept[0][:] = 7
