"""The operators as a program uses them together: prompts into the 8-bit cache and their attention in one chunk, then
decoding steps of a batch (append, attention, logits, controls), captured once and replayed."""

import numpy as np
import pytest

from llm_b200 import KV8Batch, logits_control
from tests.test_kv8 import Device, _reference, _tolerance, _workspace
from tests.test_logits_control import _mask, plain

pytestmark = pytest.mark.gpu

HEADS, KV, HD, VOCAB = 14, 2, 64, 1000


@pytest.mark.parametrize("cache,block", [("int8", 32), ("e4m3", 64)])
def test_a_batch_from_prompts_to_answers(cache, block):
    import torch

    rng = np.random.default_rng(block)
    width = HEADS * HD

    def weight(rows, cols):
        return torch.from_numpy((rng.normal(0, 1, (rows, cols)) / np.sqrt(rows)).astype(np.float32)).cuda()

    embed, wq, wk, wv = weight(VOCAB, 128) * np.sqrt(VOCAB), weight(128, width), weight(128, KV * HD), weight(128, KV * HD)
    head = weight(width, VOCAB) * 4
    prompts, steps = [200, 1, 77], 12
    n_seq, top = len(prompts), max(prompts) + steps
    d = Device(KV, block, HD, cache, [n + steps for n in prompts], rng)
    history = torch.zeros(n_seq, top, dtype=torch.int32, device="cuda")
    for i, n in enumerate(prompts):
        history[i, :n] = torch.from_numpy(rng.integers(0, VOCAB, n).astype(np.int32)).cuda()

    # the prompts: all rows in one append and one attention
    ids = torch.cat([history[i, :n] for i, n in enumerate(prompts)]).long()
    x = embed[ids]
    q, k, v = (x @ w for w in (wq, wk, wv))
    d.append(prompts, prompts, k.view(-1, KV, HD), v.view(-1, KV, HD), max_new=max(prompts))
    d.same_as_plain(prompts)
    q, out = q.view(-1, HEADS, HD), torch.empty(len(ids), HEADS, HD, device="cuda")
    batch = d.batch(prompts, prompts, max_new=max(prompts))
    d.cache.attention(batch, q, out, workspace=_workspace(d, batch, HEADS))
    want, size = _reference(d, prompts, prompts, q.cpu(), HD ** -0.5, 0)
    assert ((out.cpu().double() - want).abs() <= _tolerance(size, max(prompts), HD, "f32", want)).all()
    last = torch.tensor(np.cumsum(prompts) - 1).cuda()
    logits = out.reshape(-1, width)[last] @ head

    # the first answers, then the steps
    penalties = torch.tensor([[1.2, 0.5, 0.3]] * n_seq, device="cuda")
    mask = torch.from_numpy(_mask(rng, n_seq, VOCAB, 0.6)).cuda()
    prompt_lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    lens = prompt_lens.clone()
    tokens = torch.empty(n_seq, dtype=torch.int32, device="cuda")
    controls = dict(history=history, history_lens=lens, prompt_lens=prompt_lens, penalties=penalties, mask=mask)

    def check(logits, tokens):
        _, want = plain(logits.cpu().numpy(), history.cpu().numpy(), lens.cpu().numpy(), np.array(prompts),
                        penalties.cpu().numpy(), mask=mask.cpu().numpy())
        assert np.array_equal(tokens.cpu().numpy(), want) and (want >= 0).all()

    logits_control(logits, tokens=tokens, stream=torch.cuda.current_stream().cuda_stream, **controls)
    check(logits, tokens)

    step = KV8Batch(lens, d.dtables, rows=n_seq, max_len=top)
    work = _workspace(d, step, HEADS)
    q, k, v, out = (torch.empty(n_seq, h, HD, device="cuda") for h in (HEADS, KV, KV, HEADS))
    rows = torch.arange(n_seq, device="cuda")

    def one():
        s = torch.cuda.current_stream().cuda_stream
        history[rows, lens.long()] = tokens  # the token goes to the end of its sequence
        lens.add_(1)
        x = embed[tokens.long()]
        for w, to in ((wq, q), (wk, k), (wv, v)):
            torch.matmul(x, w, out=to.view(n_seq, -1))
        d.cache.append(step, k, v, stream=s)
        d.cache.attention(step, q, out, workspace=work, stream=s)
        torch.matmul(out.view(n_seq, width), head, out=logits)
        logits_control(logits, tokens=tokens, stream=s, **controls)

    saved = history.clone(), lens.clone(), tokens.clone()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # libraries set themselves up outside the capture
        one()
    torch.cuda.synchronize()
    for i in range(n_seq):  # that step was a step
        d.plain.append(d.tables[i], prompts[i] + 1, torch.stack([k[i:i + 1], v[i:i + 1]]).cpu())
    with torch.cuda.graph(graph, stream=side):
        one()
    for to, was in zip((history, lens, tokens), saved):
        to.copy_(was)
    for n in range(1, steps + 1):
        graph.replay()
        torch.cuda.synchronize()
        now = [m + n for m in prompts]
        if n > 1:
            for i in range(n_seq):
                d.plain.append(d.tables[i], now[i], torch.stack([k[i:i + 1], v[i:i + 1]]).cpu())
        d.same_as_plain(now)
        want, size = _reference(d, now, [1] * n_seq, q.cpu(), HD ** -0.5, 0)
        assert ((out.cpu().double() - want).abs() <= _tolerance(size, max(now), HD, "f32", want)).all(), n
        check(logits, tokens)
