"""The cache of 8-bit keys and values (append, read, attention) and the control of logits, as cases to measure.

`run` computes an operator in its plain form (elementary torch operations in float32), or, with `own` set, by the
framework's entry points (`llm_b200.KV8Cache`, `llm_b200.logits_control`). Sizes are those of the model shapes the
framework's benchmark runs (9 query heads on 3 key/value heads and 14 on 2, head size 64, vocabularies of 49152 and
151936, 64 sequences, chunks of 64 tokens) and generic ones with head size 128.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
CACHE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest 8-bit value
FIT = 2.0 ** -12  # a block's scale still fits values of up to top + FIT steps: they saturate at top
TINY = 2.0 ** -100  # rows whose largest value is below this are held as zeros
GOLDEN = 0.6180339887498949


def listed():
    return [
        # one new token of one sequence of the 14-on-2-heads model: the write of every decoding step
        _kv("append step", "append", 1, 300, 1, 14, 2, 64, 64, "int8", "f32", 0.0),
        # prompts of 64 requests of different lengths, written at once
        _kv("append prompts", "append", 64, 1000, 1000, 32, 8, 128, 64, "int8", "bf16", 0.9),
        # one sequence's rows brought back to float32, as for the framework's float32 attention
        _kv("read one sequence", "read", 1, 4096, 4096, 14, 2, 64, 64, "int8", "f32", 0.0),
        # the prefixes of a batch moved out of the cache
        _kv("read batch", "read", 48, 2011, 2011, 32, 8, 128, 32, "e4m3", "bf16", 0.8),
        # a decoding step of one short chat
        _kv("decode short", "attend", 1, 300, 1, 14, 2, 64, 64, "int8", "f32", 0.0),
        # a decoding step of 64 sequences of different lengths, the framework's multi-stream workload
        _kv("decode 64 sequences", "attend", 64, 2048, 1, 9, 3, 64, 32, "int8", "f32", 0.7),
        # a decoding step over one very long document
        _kv("decode long", "attend", 1, 131071, 1, 32, 8, 128, 64, "e4m3", "bf16", 0.0),
        # a server's batch with long contexts, of which a window is seen
        _kv("decode window", "attend", 33, 8190, 1, 14, 2, 64, 16, "int8", "bf16", 0.5, window=4000),
        # a 64-token prompt chunk behind an earlier context, the framework's prefill
        _kv("chunk of 64", "attend", 1, 1984, 64, 14, 2, 64, 64, "int8", "f32", 0.0),
        # long prompts of several requests in one pass
        _kv("prompts", "attend", 3, 5000, 1023, 32, 8, 128, 64, "int8", "bf16", 0.3),
        # one row of logits with a grammar's mask, biases and a short history
        _logits("logits one row", 1, 49152, 256, 16, "f32", 0.02),
        # a batch of rows over the larger vocabulary with long histories
        _logits("logits batch", 64, 151936, 4096, 300, "f32", 0.5),
    ]


def _kv(name, op, seqs, length, new, heads, kv_heads, hd, block, cache, dtype, spread, window=0):
    return {"name": name, "op": op, "seqs": seqs, "length": length, "new": new, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "block": block, "cache": cache, "type": dtype, "spread": spread, "window": window}


def _logits(name, rows, vocab, history, biases, dtype, allowed, pad=0):
    return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "history": history, "biases": biases,
            "type": dtype, "allowed": allowed, "pad": pad}


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))

    op = rng.choice(["append", "read", "decode", "decode", "chunk", "logits"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "logits":
        c = _logits("", log(1, 64), log(300, 150000), log(1, 4000), log(1, 300), dtype,
                    rng.choice([0.001, 0.02, 0.5, 1.0]), rng.choice([0, 0, 1, 7]))
        del c["name"]
        return c
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    hd, block, cache = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice(["int8", "e4m3"])
    spread, window = rng.choice([0.0, 0.3, 0.9]), 0
    if op in ("append", "read"):
        seqs = log(1, 64)
        length = log(1, max(1, min(4000, 1_200_000 // (seqs * kv_heads * hd) * 16)))
        new = length if op == "read" else rng.choice([1, log(1, length), length])
    elif op == "decode":
        op, seqs, new = "attend", log(1, 64), 1
        length = log(1, max(1, min(100_000, 100_000_000 // (seqs * kv_heads * hd))))
        window = rng.choice([0, 0, log(1, length)])
    else:
        op, seqs, new = "attend", log(1, 4), log(2, 700)
        length = new + log(1, 3000)
        heads = min(heads, 4 * kv_heads) if kv_heads == 8 else heads
        window = rng.choice([0, 0, log(1, length)])
    c = _kv("", op, seqs, length, new, heads, kv_heads, hd, block, cache, dtype, spread, window)
    del c["name"]
    return c


def _shape(c):
    """The sequences' lengths and their numbers of rows in this pass, from the case alone."""
    lens, new = [], []
    for i in range(c["seqs"]):
        f = 1.0 - c["spread"] * ((i * GOLDEN) % 1.0)
        lens.append(max(1, round(c["length"] * f)))
        new.append(min(lens[-1], max(1, round(c["new"] * f))))
    if c["seqs"] >= 32:
        lens[-1] = 0  # a batch of that size has a slot without a sequence: nothing of it is seen
        new[-1] = 1 if c["new"] == 1 and c["op"] == "attend" else 0
    return lens, new


def _visible(c):
    """(row, position) pairs that the attention's masks leave."""
    total = 0
    for n, m in zip(*_shape(c)):
        for p in range(max(0, n - m), n):
            total += min(p + 1, c["window"]) if c["window"] else p + 1
    return total


def _back(c):
    """Rows from the start of the first block that an append touches to the end, for each sequence."""
    return [n - (n - m) // c["block"] * c["block"] if m else 0 for n, m in zip(*_shape(c))]


def work(c):
    if c["op"] == "logits":
        cells = c["rows"] * c["vocab"]
        return {"bytes": cells * 2 * SIZE[c["type"]] + cells / 8 + 4 * c["rows"] * c["history"] + 8 * c["biases"],
                "flops": 4 * cells}
    lens, new = _shape(c)
    width, e = 2 * c["kv_heads"] * c["hd"], SIZE[c["type"]]  # K and V of one position
    if c["op"] == "append":
        return {"bytes": width * (sum(new) * (e + 1) + sum(_back(c)) * (e + 1)), "flops": 4 * width * sum(new)}
    if c["op"] == "read":
        return {"bytes": width * sum(new) * (e + 1), "flops": width * sum(new)}
    held = 0
    for n, m in zip(lens, new):
        held += min(n, c["window"] + m - 1) if c["window"] else n
    return {"bytes": width * held + 2 * sum(new) * c["heads"] * c["hd"] * e,
            "flops": 4 * c["heads"] * c["hd"] * _visible(c)}


def prepare(c, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    if c["op"] == "logits":
        return _prepare_logits(c, g)
    lens, new = _shape(c)
    rows, per = sum(new), [-(-n // c["block"]) for n in lens]
    stride = max(1, -(-max(lens) // c["block"]))
    blocks = sum(per) + 1  # block 0 belongs to no sequence
    order = 1 + torch.randperm(blocks - 1, generator=g, device=DEV).to(torch.int32)
    tables = torch.zeros(len(lens), stride, dtype=torch.int32, device=DEV)
    used = torch.arange(stride, device=DEV)[None, :] < torch.tensor(per, device=DEV)[:, None]
    tables[used] = order
    s = {"case": c, "tables": tables, "lens": torch.tensor(lens, dtype=torch.int32, device=DEV),
         "starts": _starts(new), "rows": rows, "max_new": max(new), "max_len": max(max(lens), 1)}
    one = c["new"] == 1 and all(m == 1 for m in new)
    if one:
        s["starts"] = None  # one row each: the sequences' rows follow one another
    shape = (blocks, c["kv_heads"], c["block"], c["hd"])
    for name in ("k", "v"):
        # keys have channels that are larger than the others, blocks differ in size
        x = torch.randn(shape, generator=g, device=DEV)
        x *= torch.exp(0.5 * torch.randn(1, c["kv_heads"], 1, c["hd"], generator=g, device=DEV))
        x *= torch.exp(0.3 * torch.randn(blocks, c["kv_heads"], 1, 1, generator=g, device=DEV))
        scale = x.abs().amax(dim=(2, 3)) / TOP[c["cache"]]
        x = x / scale[:, :, None, None]
        s[name + "_scale"] = scale.contiguous()
        s[name] = x.round().to(torch.int8) if c["cache"] == "int8" else x.to(torch.float8_e4m3fn)
        del x
    t = TYPES[c["type"]]
    if c["op"] == "append":
        s["k_new"], s["v_new"] = (
            (torch.randn(rows, c["kv_heads"], c["hd"], generator=g, device=DEV)
             * torch.exp(0.5 * torch.randn(rows, 1, 1, generator=g, device=DEV))).to(t) for _ in range(2))
        back = _back(c)
        s["back_starts"], s["back_rows"], s["back_max"] = _starts(back), sum(back), max(back)
    if c["op"] == "attend":
        s["q"] = (1.5 * torch.randn(rows, c["heads"], c["hd"], generator=g, device=DEV)).to(t)
    return s


def _starts(new):
    at = [0]
    for m in new:
        at.append(at[-1] + m)
    return torch.tensor(at, dtype=torch.int32, device=DEV)


def _prepare_logits(c, g):
    rows, vocab, h = c["rows"], c["vocab"], c["history"]
    t = TYPES[c["type"]]
    full = (3 * torch.randn(rows, vocab + c["pad"], generator=g, device=DEV)).to(t)
    words = -(-vocab // 32)
    bits = torch.rand(rows, words, 32, generator=g, device=DEV) < c["allowed"]
    if rows > 2:
        bits[rows // 2] = False  # a grammar that allows nothing any more
    mask = (bits.to(torch.int64) << torch.arange(32, device=DEV)).sum(2)
    # few tokens make up most of a text
    history = (torch.rand(rows, h, generator=g, device=DEV) ** 4 * vocab).long().clamp_(max=vocab - 1).to(torch.int32)
    lens = torch.randint(0, h + 1, (rows,), generator=g, device=DEV, dtype=torch.int32)
    if rows == 1:
        lens.fill_(h)
    penalties = torch.tensor([1.0, 0.0, 0.0], device=DEV) + torch.tensor([0.3, 0.5, 0.4], device=DEV) * torch.rand(
        rows, 3, generator=g, device=DEV)
    return {"case": c, "logits": full[:, :vocab], "mask": torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32),
            "history": history, "history_lens": lens, "prompt_lens": lens // 3, "penalties": penalties.contiguous(),
            "bias_ids": torch.randint(0, vocab, (c["biases"],), generator=g, device=DEV, dtype=torch.int32),
            "bias_values": 2 * torch.randn(c["biases"], generator=g, device=DEV)}


def run(s):
    c = s["case"]
    if own:
        return _own(s)
    if c["op"] == "append":
        return _plain_append(s)
    if c["op"] == "read":
        return _plain_read(s, _starts_of(s), s["rows"])
    if c["op"] == "attend":
        return _plain_attend(s)
    return _plain_logits(s)


# ---- the framework's calls

def _own(s):
    import llm_b200

    c, stream = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "logits":
        out = torch.empty(c["rows"], c["vocab"], dtype=s["logits"].dtype, device=DEV)
        tokens = torch.empty(c["rows"], dtype=torch.int32, device=DEV)
        llm_b200.logits_control(s["logits"], out=out, tokens=tokens, history=s["history"],
                                history_lens=s["history_lens"], prompt_lens=s["prompt_lens"],
                                penalties=s["penalties"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
                                mask=s["mask"], stream=stream)
        return {"logits": out, "tokens": tokens}
    if "cache" not in s:  # what a program keeps for as long as it has the cache and the batch
        s["cache"] = llm_b200.KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = llm_b200.KV8Batch(s["lens"], s["tables"], s["starts"], rows=s["rows"], max_new=s["max_new"],
                                       max_len=s["max_len"])
        if c["op"] == "append":
            s["back"] = llm_b200.KV8Batch(s["lens"], s["tables"], s["back_starts"], rows=s["back_rows"],
                                          max_new=s["back_max"], max_len=s["max_len"])
        if c["op"] == "attend":
            n = s["cache"].attention_workspace(s["batch"], c["heads"])
            s["workspace"] = torch.empty(n, dtype=torch.uint8, device=DEV)
    cache, t = s["cache"], TYPES[c["type"]]
    if c["op"] == "attend":
        out = torch.empty_like(s["q"])
        cache.attention(s["batch"], s["q"], out, window=c["window"], workspace=s["workspace"], stream=stream)
        return out
    if c["op"] == "append":
        cache.append(s["batch"], s["k_new"], s["v_new"], stream=stream)
    batch, rows = (s["back"], s["back_rows"]) if c["op"] == "append" else (s["batch"], s["rows"])
    k, v = (torch.empty(rows, c["kv_heads"], c["hd"], dtype=t, device=DEV) for _ in range(2))
    cache.read(batch, k, v, stream=stream)
    return {"k": k, "v": v}


# ---- the plain forms

def _starts_of(s):
    if s["starts"] is not None:
        return s["starts"].long()
    return torch.arange(s["rows"] + 1, device=DEV)


def _places(s, starts, rows):
    """The sequence and the position of each row."""
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), r, right=True)
    return seq, s["lens"].long()[seq] - starts[seq + 1] + r


def _plain_read(s, starts, rows):
    c = s["case"]
    seq, pos = _places(s, starts, rows)
    page = s["tables"].long()[seq, pos // c["block"]]
    out = {}
    for name in ("k", "v"):
        q = s[name].view(torch.uint8)[page, :, pos % c["block"]].view(CACHE[c["cache"]]).float()
        out[name] = (q * s[name + "_scale"][page][:, :, None]).to(TYPES[c["type"]])
    return out


def _plain_append(s):
    c = s["case"]
    block, top, starts, lens = c["block"], TOP[c["cache"]], _starts_of(s), s["lens"].long()
    new = starts[1:] - starts[:-1]
    first = (lens - new) // block
    touched = (s["max_new"] + block - 2) // block + 1
    j = first[:, None] + torch.arange(touched, device=DEV)  # [seq, touched]: the blocks' places in their sequences
    fresh = (j * block < lens[:, None]) & (new[:, None] > 0)
    page = torch.where(fresh, s["tables"].long().gather(1, j.clamp(max=s["tables"].shape[1] - 1)), 0)
    pos = j[:, :, None] * block + torch.arange(block, device=DEV)
    is_new = (pos >= (lens - new)[:, None, None]) & (pos < lens[:, None, None])
    row = torch.where(is_new, starts[:-1][:, None, None] + pos - (lens - new)[:, None, None], 0)
    older = fresh & (j * block < (lens - new)[:, None])
    for name in ("k", "v"):
        x = s[name + "_new"].float()[row].transpose(2, 3)  # [seq, touched, head, block, hd]
        keep = is_new[:, :, None, :, None]
        a = torch.where(keep & torch.isfinite(x), x.abs(), 0.0).amax(dim=(3, 4))
        s0 = torch.where(older[:, :, None], s[name + "_scale"][page], 0.0)
        s0 = torch.where((s0 > 0) & torch.isfinite(s0), s0, 0.0)
        r = a / ((top + FIT) * s0)
        m, e = torch.frexp(torch.where((r > 1) & (r <= 2.0 ** 20), r, 1.0))
        k = e - (m == 0.5).int()
        grown = torch.where(r <= 1, s0, torch.where(r <= 2.0 ** 20, torch.ldexp(s0, k), a / top))
        scale = torch.where(a < TINY, s0, torch.where(s0 == 0, a / top, grown))
        down = torch.where((a >= TINY) & (s0 > 0) & (r > 1), torch.where(r <= 2.0 ** 20, torch.ldexp(torch.ones_like(a), -k), 0.0), 1.0)
        inverse = torch.where(scale > 0, 1.0 / scale, 0.0)[:, :, :, None, None]
        y = torch.where(torch.isnan(x), 0.0, x * inverse).clamp(-top, top)
        y = torch.where(torch.isnan(y), 0.0, y)
        old = s[name].view(torch.uint8)[page].view(CACHE[c["cache"]]).float() * down[:, :, :, None, None]
        y = torch.where(keep, y, torch.where(s0[:, :, :, None, None] > 0, old, 0.0))
        q = y.round().to(torch.int8) if c["cache"] == "int8" else y.to(torch.float8_e4m3fn)
        # rows past the end of a sequence stay as they were
        held = (pos < lens[:, None, None])[:, :, None, :, None]
        q = torch.where(held, q.view(torch.uint8), s[name].view(torch.uint8)[page])
        s[name].view(torch.uint8)[page] = q
        s[name + "_scale"][page] = scale
    return _plain_read(s, s["back_starts"].long(), s["back_rows"])


def _plain_attend(s):
    c = s["case"]
    seqs, heads, kv, hd, block = c["seqs"], c["heads"], c["kv_heads"], c["hd"], c["block"]
    lens, starts, t, group = s["lens"].long(), _starts_of(s), s["max_new"], heads // kv
    new = starts[1:] - starts[:-1]
    at = starts[:-1][:, None] + torch.arange(t, device=DEV)  # [seq, t]: padded rows
    q = s["q"].float()[at.clamp(max=s["rows"] - 1)].view(seqs, t, kv, group, hd).permute(0, 2, 1, 3, 4)
    page = s["tables"].long()
    held = {}
    for name in ("k", "v"):
        x = s[name].view(torch.uint8)[page].view(CACHE[c["cache"]]).float() * s[name + "_scale"][page][..., None, None]
        held[name] = x.permute(0, 2, 1, 3, 4).reshape(seqs, kv, -1, hd)
    score = q.reshape(seqs, kv, t * group, hd) @ held["k"].transpose(2, 3) / math.sqrt(hd)
    j = torch.arange(held["k"].shape[2], device=DEV)
    p = (lens - new)[:, None] + torch.arange(t, device=DEV)
    seen = (j <= p[:, :, None]) & (j < lens[:, None, None])
    if c["window"]:
        seen &= j > p[:, :, None] - c["window"]
    hidden = ~seen[:, None, :, None, :]
    score = score.view(seqs, kv, t, group, -1).masked_fill_(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = w.sum(-1, keepdim=True)
    out = w.view(seqs, kv, t * group, -1) @ held["v"]
    out = out.view(seqs, kv, t, group, hd) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(seqs, t, heads, hd)
    seq, _ = _places(s, starts, s["rows"])
    return out[seq, torch.arange(s["rows"], device=DEV) - starts[seq]].to(s["q"].dtype)


def _plain_logits(s):
    c = s["case"]
    rows, vocab, h = c["rows"], c["vocab"], c["history"]
    x = s["logits"].float()
    i = torch.arange(h, device=DEV)
    said = (i < s["history_lens"][:, None]).int()
    answered = said * (i >= s["prompt_lens"][:, None]).int()
    ids = s["history"].long()
    zero = torch.zeros(rows, vocab, dtype=torch.int32, device=DEV)
    any_, count = zero.scatter_add(1, ids, said) > 0, zero.scatter_add(1, ids, answered)
    rep, presence, frequency = (s["penalties"][:, k:k + 1] for k in range(3))
    x = torch.where(any_, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, (x - presence) - frequency * count.float(), x)
    # of a token's biases the last in the list counts
    n = torch.arange(1, c["biases"] + 1, device=DEV)
    last = torch.zeros(vocab, dtype=torch.int64, device=DEV).scatter_reduce(0, s["bias_ids"].long(), n, "amax")
    value = torch.where(last > 0, s["bias_values"][(last - 1).clamp(min=0)], 0.0)
    x = torch.where(last > 0, x + value, x)
    v = torch.arange(vocab, device=DEV)
    bit = s["mask"][:, v // 32] >> (v % 32).int() & 1
    x = torch.where(bit == 1, x, -math.inf)
    best = torch.where(torch.isnan(x), -math.inf, x).amax(1, keepdim=True)
    token = torch.where(x == best, v, vocab).amin(1)
    token = torch.where(best[:, 0] == -math.inf, -1, token).to(torch.int32)
    return {"logits": x.to(s["logits"].dtype), "tokens": token}


# ---- the definitions in 64 bits

def _f32(x):
    return x.float().double()  # what the definition itself rounds to float32


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "logits":
        return _exact_logits(s)
    lens, new = _shape(c)
    at = [0]
    for m in new:
        at.append(at[-1] + m)
    if c["op"] == "append":
        for i, (n, m) in enumerate(zip(lens, new)):
            if m:
                _exact_append(s, i, n, m, at[i])
        new = _back(c)
    if c["op"] in ("append", "read"):
        out = {"k": [], "v": []}
        for i, (n, m) in enumerate(zip(lens, new)):
            for name in out:
                out[name].append(_exact_rows(s, name, i, n)[n - m:n] if m else _exact_rows(s, name, i, 0))
        return {name: torch.cat(x) for name, x in out.items()}
    group, out = c["heads"] // c["kv_heads"], torch.zeros(s["rows"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
    for i, (n, m) in enumerate(zip(lens, new)):
        if n == 0 or m == 0:
            continue
        k, v = _exact_rows(s, "k", i, n), _exact_rows(s, "v", i, n)
        p, j = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None, :]
        seen = (j <= p) if not c["window"] else (j <= p) & (p - j < c["window"])
        for h in range(c["heads"]):
            z = s["q"][at[i]:at[i] + m, h].double() @ k[:, h // group].T * c["hd"] ** -0.5
            z = z.where(seen, torch.tensor(-math.inf, dtype=torch.float64, device=DEV))
            out[at[i]:at[i] + m, h] = torch.softmax(z, 1) @ v[:, h // group]
    return out


def _exact_rows(s, name, i, n):
    """The values that sequence i holds at positions 0..n-1."""
    c = s["case"]
    page = s["tables"][i].long()[:max(1, -(-n // c["block"]))]
    q = s[name].view(torch.uint8)[page].view(CACHE[c["cache"]]).double() * s[name + "_scale"][page].double()[:, :, None, None]
    return q.transpose(1, 2).reshape(-1, c["kv_heads"], c["hd"])[:n]


def _exact_append(s, i, n, m, row):
    """Sequence i's m new rows, the last of its n positions, into its blocks one after another."""
    c = s["case"]
    block, top, p = c["block"], TOP[c["cache"]], n - m

    def to8(y):
        y = y.clamp(-top, top)
        return y.round().to(torch.int8) if c["cache"] == "int8" else y.float().to(torch.float8_e4m3fn)

    while p < n:
        page, lo = int(s["tables"][i, p // block]), p % block
        hi = min(block, lo + n - p)
        for name in ("k", "v"):
            x = s[name + "_new"][row:row + hi - lo].double().transpose(0, 1)  # [head, row, hd]
            a = x.abs().amax(dim=(1, 2))
            pool, scales = s[name].view(torch.uint8)[page], s[name + "_scale"][page]
            if lo:
                s0 = scales.double()
                r = _f32(a / _f32((top + FIT) * s0))
                k = torch.ceil(torch.log2(r.clamp(1.0, 2.0 ** 20)))
                scale = torch.where(r > 2.0 ** 20, _f32(a / top), s0 * 2.0 ** k)
                down = torch.where(r > 2.0 ** 20, 0.0, 2.0 ** -k)
                q = pool[:, :lo].contiguous().view(CACHE[c["cache"]]).double() * down[:, None, None]
                pool[:, :lo] = to8(q).view(torch.uint8)
            else:
                scale = _f32(a / top)
            pool[:, lo:hi] = to8(_f32(x * _f32(1.0 / scale)[:, None, None])).view(torch.uint8)
            scales.copy_(scale.float())
        row, p = row + hi - lo, p + hi - lo


def _exact_logits(s):
    c = s["case"]
    x = s["logits"].double()
    for b in range(c["rows"]):
        n, p = int(s["history_lens"][b]), int(s["prompt_lens"][b])
        rep, presence, frequency = s["penalties"][b].double().tolist()
        said, times = torch.unique(s["history"][b, p:n].long(), return_counts=True)
        every = torch.unique(s["history"][b, :n].long())
        z = x[b, every]
        x[b, every] = torch.where(z > 0, z / rep, z * rep)
        x[b, said] -= presence + frequency * times.double()
    biases = dict(zip(s["bias_ids"].tolist(), s["bias_values"].double().tolist()))  # the last of a token's
    if biases:
        x[:, list(biases)] += torch.tensor(list(biases.values()), dtype=torch.float64, device=DEV)
    bits = torch.stack([s["mask"] >> k & 1 for k in range(32)], 2).reshape(c["rows"], -1)[:, :c["vocab"]]
    x[bits == 0] = -math.inf
    return {"logits": x, "tokens": None}
