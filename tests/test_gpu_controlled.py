"""Generation with llmb_logits_control between the logits and the token (llmb_generate_controlled).

Each token is checked against the plain restatement of the controls (test_logits_control.py) on the very logits that
the model had for it (llmb_peek "logits"), which are in turn those of the prompt and the tokens so far.
"""

import ctypes as C

import numpy as np
import pytest

import llm_b200
from llm_b200 import LlmError, synth
from tests.test_logits_control import plain


def test_no_model_is_refused():
    c = llm_b200._Controls(1, 0, 0, 0, None, None, llm_b200.MASK_FN(), None)
    assert llm_b200.lib().llmb_generate_controlled(None, None, 0, 1, -1, C.byref(c), llm_b200.EMIT_FN(), None, None, None,
                                                   None) == llm_b200.ERR_ARG


@pytest.fixture(scope="module")
def gpu_model():
    g = llm_b200.GPU(synth.ensure("tiny-qwen2"), ctx=256)
    yield g
    g.close()


def _bits(words, vocab):
    return np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 1])
def test_without_controls_it_is_generate(gpu_model, mode):
    g = gpu_model
    prompt = synth.prompt_ids(g.cfg.vocab, 21, seed=3)
    old = llm_b200.get_knob("decode_mode")
    try:
        llm_b200.set_knob("decode_mode", mode)
        want, _ = g.generate(prompt, 40)
        got, tm = g.generate_controlled(prompt, 40)
        assert np.array_equal(got, want) and tm.generated == 40 and tm.prompt_tokens == 21
        eos = int(want[17])
        short, _ = g.generate(prompt, 40, eos=eos)
        assert np.array_equal(g.generate_controlled(prompt, 40, eos=eos)[0], short)
        seen = []
        g.generate_controlled(prompt, 40, emit=lambda t: seen.append(t) or len(seen) < 5)
        assert seen == want[:5].tolist()
        assert len(g.generate_controlled(prompt, 0)[0]) == 0
        again, _ = g.generate(prompt, 40)  # and the model is as it was
        assert np.array_equal(again, want)
    finally:
        llm_b200.set_knob("decode_mode", old)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [0, 1])
def test_every_token_is_the_controls_choice(gpu_model, mode):
    g = gpu_model
    V, n = g.cfg.vocab, 30
    rng = np.random.default_rng(4)
    prompt = synth.prompt_ids(V, 70, seed=9)
    biases = {int(v): float(b) for v, b in zip(rng.integers(0, V, 20), rng.normal(0, 2, 20))}
    biases[int(g.generate(prompt, 1)[0][0])] = -np.inf
    pen = np.array([[1.3, 0.4, 0.2]], np.float32)
    steps, masks = [], []

    def mask(tokens, words):
        words[:] = rng.integers(0, 1 << 32, len(words), dtype=np.uint64).astype(np.uint32)
        masks.append((tokens, words.copy()))
        return True

    def emit(t):
        steps.append((t, g.peek("logits", V)))
        return True

    old = llm_b200.get_knob("decode_mode")
    try:
        llm_b200.set_knob("decode_mode", mode)
        got, _ = g.generate_controlled(prompt, n, repetition=1.3, presence=0.4, frequency=0.2, biases=biases, mask=mask,
                                       emit=emit)
    finally:
        llm_b200.set_knob("decode_mode", old)
    assert len(got) == n == len(steps) == len(masks)
    ids, values = np.array(list(biases), np.int32), np.array(list(biases.values()), np.float32)
    for i, (tok, logits) in enumerate(steps):
        so_far, words = masks[i]
        assert np.array_equal(so_far, got[:i])
        history = np.concatenate([prompt, got[:i]]).astype(np.int32)[None]
        _, want = plain(logits[None], history, None, np.array([len(prompt)]), pen, ids, values, None, words.view(np.int32)[None])
        assert tok == got[i] == want[0], i
        assert _bits(words, V)[tok] and tok != ids[-1]
    # the logits were those of the controlled sequence: a prompt of it gives them again (within the parity tests' 1e-5)
    for i in (0, 1, 13, n - 1):
        again = g.prefill_logits(np.concatenate([prompt, got[:i]]))
        assert np.max(np.abs(again - steps[i][1])) <= 1e-5 * np.max(np.abs(again)), i


@pytest.mark.gpu
def test_stops(gpu_model):
    g = gpu_model
    V = g.cfg.vocab
    prompt = synth.prompt_ids(V, 10, seed=1)
    allowed = [7, 11, 200]

    def script(tokens, words):  # tokens 7, 11, 200 in turn, then nothing
        words[:] = 0
        if len(tokens) < 3:
            v = allowed[len(tokens)]
            words[v // 32] = 1 << (v % 32)
        return True

    got, _ = g.generate_controlled(prompt, 20, mask=script)
    assert got.tolist() == allowed
    got, _ = g.generate_controlled(prompt, 20, mask=lambda t, w: script(t, w) and len(t) < 2)
    assert got.tolist() == allowed[:2]
    got, _ = g.generate_controlled(prompt, 20, eos=11, mask=script)
    assert got.tolist() == [7]

    def broken(tokens, words):
        raise ValueError("no grammar")

    with pytest.raises(ValueError, match="no grammar"):
        g.generate_controlled(prompt, 20, mask=broken)
    with pytest.raises(ZeroDivisionError):
        g.generate_controlled(prompt, 20, emit=lambda t: 1 // 0)
    want, _ = g.generate(prompt, 8)
    assert np.array_equal(g.generate_controlled(prompt, 8)[0], want)


@pytest.mark.gpu
def test_refusals(gpu_model):
    g = gpu_model
    prompt = synth.prompt_ids(g.cfg.vocab, 10, seed=1)
    for kw in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=np.inf), dict(repetition=np.nan),
               dict(presence=np.nan), dict(frequency=np.inf), dict(biases={-1: 0.0}), dict(biases={g.cfg.vocab: 1.0}),
               dict(biases={0: np.nan})):
        with pytest.raises(LlmError) as e:
            g.generate_controlled(prompt, 4, **kw)
        assert e.value.code == llm_b200.ERR_ARG
    for bad, code in (((prompt, -1), llm_b200.ERR_ARG), (([], 4), llm_b200.ERR_ARG), (([g.cfg.vocab], 4), llm_b200.ERR_ARG),
                      ((prompt, 250), llm_b200.ERR_CONTEXT)):
        with pytest.raises(LlmError) as e:
            g.generate_controlled(*bad)
        assert e.value.code == code
    many = np.zeros(4096, np.int32)
    c = llm_b200._Controls(1, 0, 0, 4096, many.ctypes.data, many.ctypes.data, llm_b200.MASK_FN(), None)
    p = np.ascontiguousarray(prompt, np.int32)
    args = (p.ctypes.data, len(p), 4, -1)
    L = llm_b200.lib()
    assert L.llmb_generate_controlled(g._h, *args, C.byref(c), llm_b200.EMIT_FN(), None, None, None, None) == llm_b200.ERR_ARG
    assert L.llmb_generate_controlled(g._h, *args, None, llm_b200.EMIT_FN(), None, None, None, None) == llm_b200.ERR_ARG
