"""Penalties, biases and masks on logits (llmb_logits_control) against a plain restatement.

Every operation is one float32 rounding, and the restatement makes the same ones in numpy, so results are compared
exactly; a float64 evaluation beside it bounds both (four operations: 4 half steps of the largest intermediate).
"""

import ctypes as C

import numpy as np
import pytest

import llm_b200
from llm_b200 import LlmError, logits_control

gpu = pytest.mark.gpu


def _types():
    import torch

    return torch, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def plain(x, history=None, lens=None, prompts=None, penalties=None, ids=None, values=None, starts=None, mask=None,
          dtype=np.float32):
    """x [rows, vocab] in `dtype` arithmetic, the formula token by token: (result, tokens)."""
    f = dtype
    x = x.astype(f).copy()
    rows, vocab = x.shape
    tokens = np.empty(rows, np.int32)
    for b in range(rows):
        if history is not None:
            n = history.shape[1] if lens is None else int(np.clip(lens[b], 0, history.shape[1]))
            p = 0 if prompts is None else int(prompts[b])
            h = history[b, :n]
            rep, pres, freq = (f(1), f(0), f(0)) if penalties is None else penalties[b].astype(f)
            for v in set(h.tolist()):
                if not 0 <= v < vocab:
                    continue
                c = int((h[max(p, 0):] == v).sum())
                with np.errstate(all="ignore"):
                    x[b, v] = x[b, v] / rep if x[b, v] > 0 else x[b, v] * rep
                    if c:
                        x[b, v] = f(f(x[b, v] - pres) - f(freq * f(c)))
        if ids is not None:
            lo, hi = (0, len(ids)) if starts is None else (int(starts[b]), min(int(starts[b + 1]), int(starts[b]) + 4095))
            for v, value in dict(zip(ids[lo:hi].tolist(), values[lo:hi])).items():  # the last of a token's
                if 0 <= v < vocab:
                    x[b, v] = f(x[b, v] + f(value))
        if mask is not None:
            bits = np.unpackbits(mask[b].view(np.uint8), bitorder="little")[:vocab]
            x[b, bits == 0] = -np.inf
        y = np.where(np.isnan(x[b]), -np.inf, x[b])
        tokens[b] = int(np.argmax(y)) if y.max() > -np.inf else -1
    return x, tokens


def _run(x, dtype="f32", pad=0, out="new", tokens=True, **kw):
    torch, types = _types()
    rows, vocab = x.shape
    wide = torch.full((rows, vocab + pad), 77.0, dtype=types[dtype], device="cuda")
    wide[:, :vocab] = torch.from_numpy(x).cuda().to(types[dtype])
    d = wide[:, :vocab]
    seen = d.float().cpu().numpy()
    args = {k: torch.from_numpy(np.ascontiguousarray(v)).cuda() for k, v in kw.items()}
    o = {"new": torch.full((rows, vocab), 55.0, dtype=types[dtype], device="cuda"), "same": d, None: None}[out]
    t = torch.full((rows,), -7, dtype=torch.int32, device="cuda") if tokens else None
    logits_control(d, out=o, tokens=t, stream=torch.cuda.current_stream().cuda_stream, **args)
    torch.cuda.synchronize()
    if pad:
        assert (wide[:, vocab:] == 77).all()
    return seen, o, None if t is None else t.cpu().numpy()


def _mask(rng, rows, vocab, share):
    bits = rng.random((rows, -(-vocab // 32) * 32)) < share
    return np.packbits(bits, axis=1, bitorder="little").view(np.int32)


def _case(seed, rows, vocab, h, biases, share):
    rng = np.random.default_rng(seed)
    x = (3 * rng.normal(0, 1, (rows, vocab))).astype(np.float32)
    kw = dict(history=(rng.random((rows, h)) ** 4 * vocab).astype(np.int32), history_lens=rng.integers(0, h + 1, rows).astype(np.int32),
              penalties=np.stack([rng.uniform(0.7, 1.5, rows), rng.uniform(-0.5, 1, rows), rng.uniform(0, 0.5, rows)], 1).astype(np.float32),
              bias_ids=rng.integers(0, vocab, biases).astype(np.int32), bias_values=rng.normal(0, 3, biases).astype(np.float32),
              mask=_mask(rng, rows, vocab, share))
    kw["prompt_lens"] = (kw["history_lens"] // 2).astype(np.int32)
    return x, kw


def _want(seen, kw, dtype=np.float32):
    return plain(seen, kw.get("history"), kw.get("history_lens"), kw.get("prompt_lens"), kw.get("penalties"),
                 kw.get("bias_ids"), kw.get("bias_values"), kw.get("bias_starts"), kw.get("mask"), dtype)


def _check(x, kw, dtype="f32", pad=0, out="new"):
    torch, types = _types()
    seen, got, tokens = _run(x, dtype, pad, out, **kw)
    want, wt = _want(seen, kw)
    assert np.array_equal(tokens, wt)
    # numpy's float16 rounding is torch's; bfloat16 has torch's only
    w = torch.from_numpy(want).to(types[dtype])
    g = got.cpu()
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    assert torch.equal(g.nan_to_num(nan=1.0), w.nan_to_num(nan=1.0))
    exact, _ = _want(seen, kw, np.float64)
    fine = np.isfinite(exact)
    # (of the finite logits: a result made from one that is not is not finite either)
    size = 8.0 * np.abs(seen[np.isfinite(seen)], dtype=np.float64).max(initial=0) + 64
    # no intermediate is larger: penalties are below 1.5, 1, 0.5 c with c <= 64, biases below 16
    if kw.get("history") is None or kw["history"].shape[1] <= 64:
        assert (np.abs(want[fine] - exact[fine]) <= 4 * 2.0 ** -24 * size).all()
    return got, tokens


# ---------------------------------------------------------------- refusals, without a GPU


def test_bad_arguments_are_refused():
    L, arg = llm_b200.lib(), llm_b200.ERR_ARG

    def call(logits=4096, stride=100, type_=0, rows=2, vocab=100, out=4096, os_=100, tokens=256, **kw):
        c = llm_b200._LogitsCtl()
        for k, v in kw.items():
            setattr(c, k, v)
        return L.llmb_logits_control(logits, stride, type_, rows, vocab, C.byref(c), out, os_, tokens, None)

    for bad in (dict(type_=3), dict(rows=-1), dict(rows=70000), dict(vocab=0), dict(stride=99), dict(os_=99),
                dict(vocab=1 << 25, stride=1 << 25, os_=1 << 25), dict(out=None, tokens=None), dict(logits=None),
                dict(logits=4098), dict(out=4097, type_=1), dict(tokens=257), dict(history=256, history_stride=0),
                dict(history=256, history_stride=1 << 19), dict(history_lens=256), dict(prompt_lens=256), dict(n_bias=-1),
                dict(n_bias=3), dict(bias_ids=256, n_bias=3), dict(bias_values=256), dict(bias_ids=256, bias_values=256, n_bias=4096),
                dict(bias_starts=256), dict(mask=256, mask_stride=3), dict(mask=258, mask_stride=4), dict(penalties=255)):
        assert call(**bad) == arg, bad
        assert b"logits_control" in L.llmb_last_error(None)
    assert L.llmb_logits_control(4096, 100, 0, 2, 100, None, 4096, 100, 256, None) == arg


def test_python_checks_refuse_wrong_tensors():
    torch, _ = _types()
    x = torch.zeros(2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    for kw in (dict(out=x.half()), dict(out=x[:, :63]), dict(tokens=i.long()), dict(tokens=i[:1]), dict(history=i),
               dict(history=x), dict(history=torch.zeros(2, 4, dtype=torch.int32), history_lens=i[:1]), dict(penalties=x),
               dict(bias_ids=i), dict(bias_values=x[0]), dict(bias_ids=i, bias_values=x[0]), dict(mask=x), dict(mask=i)):
        with pytest.raises(LlmError):
            logits_control(x, **{"tokens": i, **kw})
    with pytest.raises(LlmError):
        logits_control(x.double(), tokens=i)
    with pytest.raises(LlmError):
        logits_control(x[0], tokens=i)
    with pytest.raises(LlmError):
        logits_control(x.t(), tokens=i)


# ---------------------------------------------------------------- on the GPU


@gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,h,pad", [(1, 1, 1, 0), (3, 31, 5, 0), (2, 32, 64, 1), (5, 257, 40, 3), (2, 2049, 64, 0),
                                              (4, 4097, 64, 7), (3, 49152, 64, 0), (2, 151936, 64, 8), (1, 180233, 33, 0),
                                              (1, 400001, 64, 0)])
def test_against_plain(rows, vocab, h, pad, dtype):
    """From one token to vocabularies of several rounds; rows that are and are not aligned to 16 bytes."""
    x, kw = _case(vocab + rows, rows, vocab, h, min(vocab, 50), 0.5)
    _check(x, kw, dtype, pad)
    _check(x, kw, dtype, pad, "same")


@gpu
@pytest.mark.parametrize("used", ["none", "history", "penalties", "bias", "mask", "prompt"])
def test_each_control_alone(used):
    x, kw = _case(5, 3, 5000, 60, 40, 0.1)
    keep = {"none": (), "history": ("history",), "penalties": ("history", "penalties"), "bias": ("bias_ids", "bias_values"),
            "mask": ("mask",), "prompt": ("history", "prompt_lens", "penalties")}[used]
    _check(x, {k: kw[k] for k in keep})


@gpu
def test_long_histories_and_many_biases():
    x, kw = _case(6, 2, 49152, 20000, 4095, 0.9)
    kw["history_lens"][:] = [20000, 13]
    _check(x, kw)
    x, kw = _case(7, 1, 500, 300000, 4095, 1.0)  # each token many times; of its biases the last
    kw["history_lens"][:] = 300000
    kw["prompt_lens"][:] = 100000
    _check(x, kw)


@gpu
def test_biases_of_each_row():
    x, kw = _case(8, 4, 3000, 10, 9000, 1.0)
    kw["bias_starts"] = np.array([0, 5000, 5000, 5003, 9000], np.int32)  # 5000: those past 4095 do not count
    _check(x, kw)


@gpu
@pytest.mark.parametrize("vocab", [100, 49152])
def test_rows_that_allow_nothing_or_one_token(vocab):
    rng = np.random.default_rng(1)
    x, kw = _case(9, 4, vocab, 20, 5, 0.0)
    one = rng.integers(0, vocab)
    kw["mask"][1, one // 32] = np.uint32(1 << (one % 32)).astype(np.int32)
    kw["mask"][2] = -1
    x[2] = -np.inf
    kw["mask"][3, (vocab - 1) // 32] = np.int64(1 << ((vocab - 1) % 32)).astype(np.uint32).view(np.int32)
    got, tokens = _check(x, kw)
    assert tokens.tolist() == [-1, one, -1, vocab - 1]


@gpu
def test_ties_zeros_infinities_and_nan():
    x = np.zeros((6, 5000), np.float32)
    x[0, [4999, 17, 300]] = 2.0            # the first of equal ones
    x[1, 10], x[1, 3] = 0.0, -0.0          # 0 and -0 are equal: the first
    x[1] -= 0.0
    x[2, 40], x[2, 41] = np.nan, 1.0       # a NaN is not taken
    x[3, 50], x[3, 60] = np.inf, 5.0
    x[4] = np.nan
    x[5] = -np.finfo(np.float32).max       # the lowest value is a value
    got, tokens = _check(x, {})
    assert tokens.tolist() == [17, 0, 41, 50, -1, 0]
    # an infinity that is not allowed, and NaN where it is not
    mask = np.full((6, -(-5000 // 32)), -1, np.int32)
    mask[3, 50 // 32] &= ~np.int32(1 << 50 % 32)
    mask[2, 40 // 32] &= ~np.int32(1 << 40 % 32)
    got, tokens = _check(x, {"mask": mask})
    assert tokens.tolist() == [17, 0, 41, 60, -1, 0] and not got[2].isnan().any()


@gpu
def test_ids_outside_the_vocabulary_and_lengths_outside_the_history():
    x, kw = _case(10, 3, 1000, 30, 20, 1.0)
    kw["history"][:, ::3] = [[-1] * 10, [1000] * 10, [np.iinfo(np.int32).min] * 10]
    kw["bias_ids"][:3] = [-5, 1000, np.iinfo(np.int32).max]
    kw["history_lens"] = np.array([-3, 31, 1 << 30], np.int32)
    kw["prompt_lens"] = np.array([5, -1, 12], np.int32)
    _check(x, kw)
    del kw["bias_ids"], kw["bias_values"]
    kw["prompt_lens"][:] = 1 << 30
    _check(x, kw)


@gpu
def test_tokens_alone_and_results_alone():
    x, kw = _case(11, 3, 7000, 30, 20, 0.5)
    seen, _, tokens = _run(x, out=None, **kw)
    want, wt = _want(seen, kw)
    assert np.array_equal(tokens, wt)
    _, got, none = _run(x, tokens=False, **kw)
    assert none is None and np.array_equal(got.cpu().numpy(), want)


@gpu
def test_captured_replayed_and_refused():
    torch, _ = _types()
    x, kw = _case(12, 2, 49152, 40, 20, 0.5)
    args = {k: torch.from_numpy(v).cuda() for k, v in kw.items()}
    d, t = torch.from_numpy(x).cuda(), torch.empty(2, dtype=torch.int32, device="cuda")
    out, graph = torch.empty_like(d), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        logits_control(d, out=out, tokens=t, stream=torch.cuda.current_stream().cuda_stream, **args)
    for n in (0, 7, 40):
        kw["history_lens"][:] = n
        args["history_lens"].fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        want, wt = _want(x, kw)
        assert np.array_equal(out.cpu().numpy(), want) and np.array_equal(t.cpu().numpy(), wt)
    with pytest.raises(LlmError, match="not device memory"):
        logits_control(d, tokens=torch.empty(2, dtype=torch.int32))
    logits_control(d[:0], tokens=t[:0])  # no rows
