"""The 8-bit key/value cache: llmb_kv8_append, llmb_kv8_read, llmb_kv8_attention.

Append and read are compared bit for bit with a plain float32 restatement of their definition, attention with a
float64 softmax over the values that the cache stands for. Tolerances are derived where they are computed.
"""

import ctypes as C
import math

import numpy as np
import pytest

import llm_b200
from llm_b200 import KV8Batch, KV8Cache, LlmError

gpu = pytest.mark.gpu
TOP = {"int8": 127.0, "e4m3": 448.0}
DTYPES = ("f32", "f16", "bf16")


def _t():
    import torch

    return torch, {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}, \
        {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------- refusals, without a GPU


def _structs(**kw):
    c = llm_b200._KV8Cache(4096, 8192, 256, 512, 2 * 64 * 64, 8, 64, 2, 64, 0)
    b = llm_b200._KV8Batch(256, 512, 1024, 2, 4, 3, 0, 0)
    for k, v in kw.items():
        setattr(c if hasattr(c, k) else b, k, v)
    return C.byref(c), C.byref(b)


def _append(L, c, b, k=4096, v=4096, type_=0, stride=128):
    return L.llmb_kv8_append(c, b, k, v, type_, stride, None)


def _attend(L, c, b, q=4096, qs=896, out=4096, os_=896, type_=0, heads=14, scale=0.0, window=0, ws=4096, n=1 << 30):
    return L.llmb_kv8_attention(c, b, q, qs, out, os_, type_, heads, scale, window, ws, n, None)


@pytest.mark.parametrize("bad", [
    dict(block=48), dict(block=0), dict(head_dim=96), dict(head_dim=0), dict(type=2), dict(kv_heads=0), dict(n_blocks=0),
    dict(block_stride=2 * 64 * 64 - 16), dict(block_stride=2 * 64 * 64 + 8), dict(block_stride=-16), dict(n_seq=0),
    dict(n_seq=70000), dict(table_stride=0), dict(table_stride=1 << 30), dict(n_rows=-1), dict(max_new=-1),
    dict(max_len=-1), dict(k=0), dict(v=4100), dict(k_scale=None), dict(v_scale=258), dict(lens=None), dict(tables=None),
    dict(starts=1026), dict(starts=None)])
def test_bad_caches_and_batches_are_refused(bad):
    """Each call, before any CUDA call (this runs without a GPU); starts=None: 3 rows do not divide among 2 sequences."""
    L = llm_b200.lib()
    c, b = _structs(**bad)
    for rc in (_append(L, c, b), L.llmb_kv8_read(c, b, 4096, 4096, 0, 128, None), _attend(L, c, b)):
        assert rc == llm_b200.ERR_ARG
        assert L.llmb_last_error(None)


def test_bad_rows_are_refused():
    L = llm_b200.lib()
    c, b = _structs()
    arg = llm_b200.ERR_ARG
    assert _append(L, None, b) == arg and _append(L, c, None) == arg
    assert _append(L, c, b, k=None) == arg and _append(L, c, b, v=4104) == arg
    assert _append(L, c, b, type_=3) == arg and _append(L, c, b, stride=124) == arg and _append(L, c, b, stride=130) == arg
    assert _append(L, c, b, type_=2, stride=132) == arg  # 264 bytes
    assert L.llmb_kv8_read(c, b, 4097, None, 0, 128, None) == arg
    for bad in (dict(heads=13), dict(heads=0), dict(heads=2 * 65), dict(window=-1), dict(scale=math.inf), dict(scale=-0.5),
                dict(scale=math.nan), dict(qs=892), dict(os_=894), dict(q=None), dict(out=4104), dict(type_=-1)):
        assert _attend(L, c, b, **bad) == arg, bad
    assert b"attention" in L.llmb_last_error(None)
    for heads, want in ((13, -1), (0, -1), (130, -1), (14, 0)):
        c, b = _structs(max_len=256)
        assert L.llmb_kv8_attention_workspace(c, b, heads) == want
    c, b = _structs(block=7)
    assert L.llmb_kv8_attention_workspace(c, b, 14) == -1


def test_python_checks_refuse_wrong_tensors():
    torch, types, caches = _t()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.ones(4, 2)
    for args in ((k, k.to(torch.float8_e4m3fn), s, s), (k.float(), k.float(), s, s), (k, k[:3], s, s), (k, k, s[:3], s),
                 (k, k, s.double(), s), (k.transpose(1, 2), k.transpose(1, 2), s, s), (k[0], k[0], s, s)):
        with pytest.raises(LlmError):
            KV8Cache(*args)
    lens, tables = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    for args in ((lens.long(), tables), (lens, tables[:1]), (lens, tables.t()), (lens, tables, lens), (lens, tables[0])):
        with pytest.raises(LlmError):
            KV8Batch(*args, rows=2)
    cache, batch = KV8Cache(k, k, s, s), KV8Batch(lens, tables, rows=2)
    x = torch.zeros(2, 2, 64)
    for a in ((x[:1], x), (x.double(), x.double()), (x, x.half()), (x, None), (x[:, :, :32], x), (x[:, :1], x)):
        with pytest.raises(LlmError):
            cache.append(batch, *a)
    with pytest.raises(LlmError):
        cache.read(batch)
    for a in ((1, 2), ("k", x), (x, object())):  # no tensors at all
        with pytest.raises((AttributeError, TypeError)):
            cache.append(batch, *a)
    with pytest.raises(TypeError):
        cache.append(batch, x, x, stream="0")
    q = torch.zeros(2, 4, 64)
    with pytest.raises(LlmError, match="window"):
        cache.attention(batch, q, q, window=1 << 40)
    for a in ((q, q.half()), (q, q[:1]), (q[0], q[0]), (q.transpose(0, 1), q)):
        with pytest.raises(LlmError):
            cache.attention(batch, *a)


# ---------------------------------------------------------------- a plain restatement


class Plain:
    """The cache in the clear: 8-bit values as float32 numbers, on the CPU."""

    def __init__(self, blocks, kv, block, hd, cache):
        import torch

        self.block, self.cache, self.top = block, cache, np.float32(TOP[cache])
        self.q = torch.zeros(2, blocks, kv, block, hd)
        self.scale = np.zeros((2, blocks, kv), np.float32)

    def to8(self, y):
        import torch

        y = torch.nan_to_num(y, nan=0.0).clamp(-float(self.top), float(self.top))
        return y.round() if self.cache == "int8" else y.to(torch.float8_e4m3fn).float()

    def append(self, table, length, rows):
        """rows [2 (k, v), n, kv, hd] float32: the last n of the sequence's positions; per block, head and kind."""
        import torch

        f = np.float32
        n, p = rows.shape[1], max(length - rows.shape[1], 0)
        first = length - n
        while p < length:
            b, lo = int(table[p // self.block]), p % self.block
            hi = min(self.block, lo + length - p)
            for kind in range(2):
                for h in range(rows.shape[2]):
                    x = rows[kind, p - first:p - first + hi - lo, h]
                    a = f(torch.where(torch.isfinite(x), x.abs(), torch.zeros(())).max())
                    s0 = self.scale[kind, b, h] if lo else f(0)
                    s0 = s0 if np.isfinite(s0) and s0 > 0 else f(0)
                    fresh, old, s = f(a * (f(1) / self.top)), f(1), s0
                    if a >= f(2.0 ** -100):
                        if s0 == 0:
                            s = fresh
                        else:
                            r = float(f(a / f((self.top + f(2.0 ** -12)) * s0)))
                            if r > 2 ** 20:
                                s, old = fresh, f(0)
                            elif r > 1:
                                k = math.ceil(math.log2(r))
                                s, old = f(s0 * f(2.0 ** k)), f(2.0 ** -k)
                    inv = f(1) / s if s > 0 else f(0)
                    self.q[kind, b, h, :lo] = self.to8(self.q[kind, b, h, :lo] * float(old if s0 > 0 else 0))
                    y = x * torch.tensor(inv)
                    self.q[kind, b, h, lo:hi] = self.to8(torch.where(torch.isinf(x), x, y))
                    self.scale[kind, b, h] = s
            p += hi - lo

    def rows(self, table, length, n, dtype="f32"):
        """[2, n, kv, hd] of the positions length - n .. length - 1, in float32 rounded to the type."""
        _, types, _ = _t()
        p = np.arange(length - n, length)
        b = np.asarray(table)[p // self.block]
        import torch

        x = self.q[:, b, :, p % self.block].permute(1, 0, 2, 3)  # [2, n, kv, hd] (advanced indices come first)
        return (x * torch.from_numpy(self.scale[:, b])[..., None]).to(types[dtype])


class Device:
    """A cache on the GPU with a Plain one beside it; every block that belongs to no sequence holds garbage."""

    def __init__(self, kv, block, hd, cache, lens_max, rng, spare=2):
        torch, _, caches = _t()
        self.per = [-(-n // block) for n in lens_max]
        blocks = sum(self.per) + spare
        self.plain = Plain(blocks, kv, block, hd, cache)
        self.kv, self.hd, self.block, self.kind = kv, hd, block, cache
        self.k = torch.full((blocks, kv, block, hd), 0x7f, dtype=torch.uint8, device="cuda").view(caches[cache])
        self.v = self.k.clone()
        self.ks = torch.full((blocks, kv), math.nan, device="cuda")
        self.vs = self.ks.clone()
        order = rng.permutation(blocks)
        stride = max(max(self.per), 1)
        self.tables = np.full((len(lens_max), stride), -1, np.int32)
        at = 0
        for i, m in enumerate(self.per):
            self.tables[i, :m] = order[at:at + m]
            at += m
        self.dtables = torch.from_numpy(self.tables).cuda()
        self.cache = KV8Cache(self.k, self.v, self.ks, self.vs)

    def batch(self, lens, new=None, max_new=0, max_len=0, rows=None):
        torch, _, _ = _t()
        starts = None if new is None else torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32).cuda()
        rows = rows if rows is not None else len(lens) if new is None else int(sum(new))
        return KV8Batch(torch.tensor(lens, dtype=torch.int32).cuda(), self.dtables, starts, rows=rows, max_new=max_new,
                        max_len=max_len)

    def append(self, lens, new, k, v, **kw):
        torch, _, _ = _t()
        self.cache.append(self.batch(lens, new, **kw), k, v)
        at, new = 0, new if new is not None else [1] * len(lens)
        for i, (n, m) in enumerate(zip(lens, new)):
            if m:
                self.plain.append(self.tables[i], n, torch.stack([k[at:at + m], v[at:at + m]]).float().cpu())
            at += m

    def same_as_plain(self, lens):
        """Bytes and scales of everything the sequences hold."""
        torch, _, _ = _t()
        for kind, (x, s) in enumerate(((self.k, self.ks), (self.v, self.vs))):
            x, s = x.cpu().float(), s.cpu().numpy()
            for i, n in enumerate(lens):
                for j in range(-(-n // self.block)):
                    b, m = self.tables[i, j], min(self.block, n - j * self.block)
                    assert np.array_equal(s[b], self.plain.scale[kind, b]), (i, j, s[b], self.plain.scale[kind, b])
                    assert torch.equal(x[b, :, :m], self.plain.q[kind, b, :, :m]), (kind, i, j)


def _rows(torch, rng, n, heads, hd, dtype, spread=1.0):
    _, types, _ = _t()
    x = rng.normal(0, 1, (n, heads, hd)) * np.exp(spread * rng.normal(0, 1, (n, 1, 1)))
    return torch.from_numpy(x.astype(np.float32)).to(types[dtype]).cuda()


# ---------------------------------------------------------------- append and read


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,block,hd,cache", [(2, 64, 64, "int8"), (3, 16, 64, "e4m3"), (1, 128, 128, "int8"),
                                               (8, 32, 128, "e4m3"), (1, 16, 64, "int8"), (2, 128, 128, "e4m3")])
def test_append_and_read(kv, block, hd, cache, dtype):
    """Prompts of ragged lengths (none and one among them), then single tokens whose growing size makes scales grow."""
    torch, types, _ = _t()
    rng = np.random.default_rng(block * hd + kv)
    new = [0, 1, block - 1, block, block + 1, 3 * block + 5]
    steps = 5
    d = Device(kv, block, hd, cache, [n + steps + 1 for n in new], rng)
    lens = list(new)
    d.append(lens, new, *(_rows(torch, rng, sum(new), kv, hd, dtype) for _ in range(2)), max_new=max(new))
    d.same_as_plain(lens)
    for step in range(steps):
        lens = [n + 1 for n in lens]
        d.append(lens, None, *(3.0 ** step * _rows(torch, rng, len(lens), kv, hd, dtype) for _ in range(2)))
        d.same_as_plain(lens)
    k, v = (torch.full((sum(lens) + 3, kv, hd), 7.0, dtype=types[dtype], device="cuda") for _ in range(2))
    d.cache.read(d.batch(lens, lens, rows=len(k)), k, v)
    at = 0
    for i, n in enumerate(lens):
        want = d.plain.rows(d.tables[i], n, n, dtype)
        assert torch.equal(k[at:at + n].cpu(), want[0]) and torch.equal(v[at:at + n].cpu(), want[1]), i
        at += n
    assert (k[at:] == 7).all() and (v[at:] == 7).all()  # rows behind the last sequence


@gpu
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_all_roundings_of_a_value_stay_within_one_step(cache):
    """Whatever the chunks the rows come in. int8's step is the final scale; e4m3's at a value x is 2^-3 of x's power
    of two (3 mantissa bits), at least 2^-9 of the scale (its subnormals); the factor that growing multiplies by is
    exact, and float32 roundings of x / s add 2^-22."""
    torch, _, _ = _t()
    rng = np.random.default_rng(5)
    kv, block, hd, n = 2, 64, 64, 150
    x = _rows(torch, rng, n, kv, hd, "f32", 1.5)
    for chunk in (1, 7, 64, n):
        d = Device(kv, block, hd, cache, [n], rng)
        for a in range(0, n, chunk):
            m = min(chunk, n - a)
            d.cache.append(d.batch([a + m], [m]), x[a:a + m].contiguous(), x[a:a + m].contiguous())
        k = torch.empty_like(x)
        d.cache.read(d.batch([n], [n]), k)
        page = torch.from_numpy(d.tables[0][np.arange(n) // block]).long()
        scale = d.ks.cpu()[page][:, :, None].double()
        xd = x.cpu().double()
        step = scale if cache == "int8" else torch.maximum(scale * 2.0 ** -9, 2.0 ** (torch.floor(torch.log2(xd.abs())) - 3))
        assert ((k.cpu().double() - xd).abs() <= step + 2.0 ** -22 * xd.abs()).all(), chunk


@gpu
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_append_of_zeros_tiny_huge_and_non_finite_rows(cache):
    torch, _, _ = _t()
    rng = np.random.default_rng(9)
    kv, block, hd = 2, 16, 64
    d = Device(kv, block, hd, cache, [40], rng)
    n = 0
    for value in (0.0, 1e-36, 2.0 ** -99, 1e-20, 1e-3, 1.0, 0.0, 1e30, 3.4e38, 1.0):
        x = value * (torch.rand(1, kv, hd, generator=torch.Generator().manual_seed(n)) + 0.5).clamp(max=1).cuda()
        n += 1
        d.append([n], [1], x, -x)
        d.same_as_plain([n])
    x = _rows(torch, rng, 20, kv, hd, "f32")
    x[3, 0, 5], x[4, 1, 6], x[5, 0, 7], x[17] = math.inf, -math.inf, math.nan, math.nan
    n += 20
    d.append([n], [20], x, x)
    d.same_as_plain([n])


@gpu
def test_append_again_changes_nothing():
    torch, _, _ = _t()
    rng = np.random.default_rng(2)
    d = Device(2, 32, 64, "int8", [77, 40], rng)
    d.append([70, 0], [70, 0], *(_rows(torch, rng, 70, 2, 64, "bf16") for _ in range(2)))
    k, v = (4 * _rows(torch, rng, 9, 2, 64, "bf16") for _ in range(2))
    d.append([77, 2], [7, 2], k, v)
    before = d.k.clone(), d.v.clone(), d.ks.clone(), d.vs.clone()
    d.cache.append(d.batch([77, 2], [7, 2]), k, v)
    for a, b in zip(before, (d.k, d.v, d.ks, d.vs)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@gpu
def test_lengths_tables_and_starts_that_are_wrong_touch_nothing_else():
    """Block numbers outside the pool, lengths past the table, more rows than positions, starts that go back: reads and
    writes stay inside the buffers, and what belongs to others stays as it was."""
    torch, _, _ = _t()
    rng = np.random.default_rng(3)
    kv, block, hd = 2, 16, 64
    d = Device(kv, block, hd, "int8", [64, 64], rng)
    good = d.tables.copy()
    d.append([64, 64], [64, 64], *(_rows(torch, rng, 128, kv, hd, "f32") for _ in range(2)))
    bad = good.copy()
    bad[0] = [good[0][0], -1, 1 << 30, len(d.k)]
    d.dtables.copy_(torch.from_numpy(bad))
    x = _rows(torch, rng, 300, kv, hd, "f32")
    before = d.k.clone()
    d.cache.append(d.batch([60, 0], [44, 0]), x[:44].contiguous(), x[:44].contiguous())  # positions 16..59: no block
    assert torch.equal(before, d.k)
    k, v = (torch.full((64, kv, hd), 5.0, device="cuda") for _ in range(2))
    d.cache.read(d.batch([64, 0], [64, 0]), k, v)
    assert torch.equal(k[:16].cpu(), d.plain.rows(good[0], 64, 64)[0][:16]) and (k[16:] == 0).all()
    # a row before position 0 reads as 0; it is not written
    d.dtables.copy_(torch.from_numpy(good))
    k.fill_(5)
    d.cache.read(d.batch([10, 0], [14, 0], rows=64), k, v)
    assert (k[:4] == 0).all() and torch.equal(k[4:14].cpu(), d.plain.rows(good[0], 10, 10)[0]) and (k[14:] == 5).all()
    q = _rows(torch, rng, 64, 4, hd, "f32")
    out = torch.full_like(q, 3.0)
    for lens, new in (([1 << 30, -5], [10, 3]), ([64, 64], [50, -20]), ([64, 64], [70, 100]), ([-1, 3], [-3, 5])):
        b = d.batch(lens, new, rows=64, max_len=64)
        d.cache.attention(b, q, out, workspace=_workspace(d, b, 4))
        d.cache.read(b, k, v)
        d.cache.append(b, x[:64].contiguous(), x[:64].contiguous())
    torch.cuda.synchronize()
    others = np.setdiff1d(np.arange(len(d.k)), good)
    assert torch.equal(d.k[others], before[others]) and torch.isnan(d.ks[others]).all()


# ---------------------------------------------------------------- attention


def _workspace(d, batch, heads):
    torch, _, _ = _t()
    n = d.cache.attention_workspace(batch, heads)
    return torch.full((max(n, 16),), 0xff, dtype=torch.uint8, device="cuda")  # NaN: nothing is read before it is written


def _reference(d, lens, new, q, scale, window):
    """float64 attention over the plain cache, and for each row what its tolerance is made of: the largest
    scale sum |q k| and the largest |v| it sees."""
    torch, _, _ = _t()
    heads = q.shape[1]
    grp = heads // d.kv
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape[0], 2, dtype=torch.float64)
    at = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        k, v = d.plain.rows(d.tables[i], n, n).double()
        for r in range(m):
            p = n - m + r
            lo = max(0, p + 1 - window) if window else 0
            if p < 0:
                continue
            kk, vv = k[lo:p + 1].repeat_interleave(grp, 1), v[lo:p + 1].repeat_interleave(grp, 1)
            z = scale * torch.einsum("hd,nhd->hn", q[at + r].double(), kk)
            out[at + r] = torch.einsum("hn,nhd->hd", torch.softmax(z, 1), vv)
            size[at + r, 0] = scale * torch.einsum("hd,nhd->hn", q[at + r].double().abs(), kk.abs()).max()
            size[at + r, 1] = vv.abs().max()
        at += m
    return out, size


def _tolerance(size, n, hd, dtype, want):
    """How far the kernels' arithmetic may be off, for each row.

    A score's operands: the query's pieces keep 22 bits (float32), 8-bit values are exact; the sum of hd products in
    float32 steps of 16 (two pieces each) that are each off by 2^-23 of the largest partial sum: together
    (2^-22 + hd / 8 * 2^-23 + 2^-22 for the factor, the block's scale and the shift) * S, S = scale sum |q k|.
    A weight exp(z): that much relative, 2^-21 for exp2 and the mantissa of V's scale, and its rounding: two float16
    pieces 2^-22, one (bfloat16 rows) 2^-11 (half a step is 2^-12, twice for subnormal ones near the bottom).
    The result is a mean of v: an error of w relative in the weights is off by at most 2 w max|v|; the sums over n
    positions in steps of 16, and over parts and warps, add (n / 16 + 32) 2^-23 max|v| twice (numerator and
    denominator). At last the rounding to the type, half a step."""
    torch, types, _ = _t()
    s, v = size[:, 0], size[:, 1]
    w = s * (2.0 ** -21 + hd / 8 * 2.0 ** -23) + 2.0 ** -21 + (2.0 ** -11 if dtype == "bf16" else 2.0 ** -22)
    tol = 2 * w * v + 2 * (n / 16 + 32) * 2.0 ** -23 * v
    return tol[:, None, None] + want.abs() * torch.finfo(types[dtype]).eps / 2


def _check_attention(d, lens, new, heads, dtype, window=0, scale=0.0, q=None, uniform=False, stride=0, **kw):
    torch, types, _ = _t()
    rng = np.random.default_rng(heads + sum(lens))
    rows = sum(new)
    q = q if q is not None else 1.5 * _rows(torch, rng, rows, heads, d.hd, dtype, 0.3)
    batch = d.batch(lens, None if uniform else new, rows=rows, **kw)
    if stride:  # rows inside wider ones, as the queries of a fused product are
        wide = torch.zeros(rows, heads * d.hd + stride, dtype=types[dtype], device="cuda")
        wide[:, :heads * d.hd] = q.reshape(rows, -1)
        q = wide[:, :heads * d.hd].unflatten(1, (heads, d.hd))
    out = torch.full((rows, heads, d.hd), math.nan, dtype=types[dtype], device="cuda")
    d.cache.attention(batch, q, out, scale=scale, window=window, workspace=_workspace(d, batch, heads))
    got = out.cpu().double()
    want, size = _reference(d, lens, new, q.cpu(), scale or 1 / math.sqrt(d.hd), window)
    err, tol = (got - want).abs(), _tolerance(size, max(lens), d.hd, dtype, want)
    assert (err <= tol).all(), (float((err / tol.clamp(min=1e-300)).nan_to_num(1e9).max()), float(err.max()))
    return out


def _filled(kv, block, hd, cache, lens, rng, dtype="f32"):
    torch, _, _ = _t()
    d = Device(kv, block, hd, cache, lens, rng)
    d.append(lens, lens, *(_rows(torch, rng, sum(lens), kv, hd, dtype, 0.5) for _ in range(2)))
    return d


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,group,block,hd,cache", [(2, 7, 64, 64, "int8"), (3, 3, 16, 64, "e4m3"), (1, 1, 32, 128, "int8"),
                                                     (2, 8, 128, 128, "e4m3"), (1, 17, 16, 64, "int8"),
                                                     (2, 4, 32, 128, "int8")])
def test_decode(kv, group, block, hd, cache, dtype):
    """One token of sequences from none and one position to several parts."""
    rng = np.random.default_rng(kv * group + block)
    lens = [1, 0, 2, 15, 16, 17, 127, 129, 700, 1500]
    d = _filled(kv, block, hd, cache, lens, rng)
    out = _check_attention(d, lens, [1] * len(lens), kv * group, dtype, uniform=True)
    assert (out[1] == 0).all()  # no position: 0
    one = _filled(kv, block, hd, cache, [2100], rng)
    _check_attention(one, [2100], [1], kv * group, dtype, uniform=True)  # one sequence: its parts are joined


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,new", [([5], [5]), ([64], [64]), ([200, 0, 77, 130], [100, 0, 77, 1]),
                                      ([1300, 1], [40, 1]), ([300], [129]), ([10, 3], [12, 5])])
def test_chunks(lens, new, dtype):
    """Prompt chunks: from the start, behind a context, of several sequences, and with more rows than positions."""
    rng = np.random.default_rng(sum(lens))
    d = _filled(2, 64, 64, "int8", lens, rng)
    _check_attention(d, lens, new, 14, dtype)
    d = _filled(1, 16, 128, "e4m3", lens, rng)
    _check_attention(d, lens, new, 4, dtype, stride=16)


def _reference_by_head(d, lens, new, q, scale, window):
    """_reference for many rows: a head's rows at once."""
    torch, _, _ = _t()
    grp = q.shape[1] // d.kv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size = torch.zeros(q.shape[0], 2, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        k, v = d.plain.rows(d.tables[i], n, n).double().cuda()
        p, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
        seen = (j <= p) & (j > p - window) if window else j <= p
        some = seen.any(1)
        for h in range(q.shape[1] if n and m else 0):
            qh, kh, vh = q[at:at + m, h].double().cuda(), k[:, h // grp], v[:, h // grp]
            z = (scale * qh @ kh.T).masked_fill(~seen, -math.inf)
            w = torch.where(some[:, None], torch.softmax(z, 1), 0.0)
            out[at:at + m, h] = w @ vh
            s = size[at:at + m]
            s[:, 0] = s[:, 0].maximum((scale * qh.abs() @ kh.abs().T).masked_fill(~seen, 0).amax(1))
            s[:, 1] = s[:, 1].maximum(vh.abs().amax())
        at += m
    return out.cpu(), size.cpu()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv,group,block,hd,cache", [(2, 4, 16, 64, "int8"), (1, 7, 128, 64, "e4m3"), (2, 3, 32, 128, "int8"),
                                                     (1, 5, 64, 128, "e4m3")])
def test_long_chunks(kv, group, block, hd, cache, dtype):
    """Enough rows for the tensor cores' tiles: ragged, whole prompts and chunks behind a context, a sequence without
    positions, one with more rows than positions, one of a single token; whole and in windows; one alone, in parts."""
    torch, types, _ = _t()
    rng = np.random.default_rng(kv * group + block)
    heads = kv * group
    for lens, new in (([1500, 0, 2, 900, 200], [400, 300, 1, 900, 260]), ([4000], [129])):
        d = _filled(kv, block, hd, cache, lens, rng)
        q = 1.5 * _rows(torch, rng, sum(new), heads, hd, dtype, 0.3)
        for window in (0, 1, 333):
            for bounds in (dict(), dict(max_new=max(new), max_len=max(lens))):
                batch = d.batch(lens, new, **bounds)
                out = torch.full_like(q, math.nan)
                d.cache.attention(batch, q, out, window=window, workspace=_workspace(d, batch, heads))
                want, size = _reference_by_head(d, lens, new, q.cpu(), 1 / math.sqrt(hd), window)
                err, tol = (out.cpu().double() - want).abs(), _tolerance(size, max(lens), hd, dtype, want)
                assert (err <= tol).all(), (lens, window, float(err.max()))
                at = 0
                for n, m in zip(lens, new):
                    assert (out[at:at + max(m - n, 0)] == 0).all()  # rows before position 0
                    at += m


def _near(out, want, tol, dtype):
    """Within the tolerance, or, where that reaches past the type's largest number, its infinity (float16 ends at 65504,
    and rounding to nearest takes what is beyond to infinity)."""
    torch, types, _ = _t()
    got = out.cpu().double()
    past = (want.abs() + tol >= torch.finfo(types[dtype]).max) & got.isinf() & (got.sign() == want.sign())
    return ((got - want).abs() <= tol) | past


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_chunks_of_all_sizes(dtype):
    """Scores that grow from step to step (the maximum has to follow), block scales that differ by 2^30, a query that is
    not finite, and blocks without a place in the pool."""
    torch, _, _ = _t()
    rng = np.random.default_rng(16)
    n, m, heads, hd = 2000, 300, 8, 64
    d = Device(2, 32, hd, "int8", [n], rng)
    k, v = (_rows(torch, rng, n, 2, hd, "f32", 0.3) for _ in range(2))
    k *= torch.linspace(0, 12, n, device="cuda")[:, None, None]
    v[320:640] *= 2.0 ** 30
    v[1000:1032] = 0
    d.append([n], [n], k, v)
    q = _rows(torch, rng, m, heads, hd, dtype, 0.3)
    q[7, 3, 5], q[250, 0, 0] = math.nan, math.inf
    batch = d.batch([n], [m])
    out = torch.empty_like(q)
    d.cache.attention(batch, q, out, workspace=_workspace(d, batch, heads))
    bad = torch.zeros(m, heads, dtype=torch.bool)
    bad[7, 3] = bad[250, 0] = True
    assert torch.isnan(out[bad.cuda()]).all()
    want, size = _reference_by_head(d, [n], [m], q.cpu().nan_to_num(0, 0, 0), 1 / 8, 0)
    assert _near(out, want, _tolerance(size, n, hd, dtype, want), dtype)[~bad].all()
    # without its first blocks a sequence is the rest of it (window: none of the rows sees what is left out)
    whole, cut = torch.empty_like(q), torch.empty_like(q)
    d.cache.attention(batch, q, whole, window=700, workspace=_workspace(d, batch, heads))
    tables = d.dtables.clone()
    tables[0, :20] = torch.tensor([-1, len(d.k)] * 10, dtype=torch.int32)
    gone = KV8Batch(torch.tensor([n], dtype=torch.int32).cuda(), tables, torch.tensor([0, m], dtype=torch.int32).cuda(), rows=m)
    d.cache.attention(gone, q, cut, window=700, workspace=_workspace(d, gone, heads))
    assert torch.equal(whole[~bad.cuda()], cut[~bad.cuda()])
    d.cache.attention(gone, q, cut, workspace=_workspace(d, gone, heads))
    d2 = Device(2, 32, hd, "int8", [n - 640], rng)
    d2.append([n - 640], [n - 640], k[640:].contiguous(), v[640:].contiguous())
    want, size = _reference_by_head(d2, [n - 640], [m], q.cpu().nan_to_num(0, 0, 0), 1 / 8, 0)
    assert _near(cut, want, _tolerance(size, n, hd, dtype, want), dtype)[~bad].all()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 15, 16, 64, 700, 5000])
def test_window(window, dtype):
    rng = np.random.default_rng(window)
    d = _filled(2, 32, 64, "int8", [1400, 9, 650], rng)
    _check_attention(d, [1400, 9, 650], [1, 1, 1], 6, dtype, window=window, uniform=True)
    _check_attention(d, [1400, 9, 650], [30, 9, 200], 6, dtype, window=window)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_of_all_sizes(dtype):
    """Large scores (one position takes all), equal ones, and block scales that differ by 2^60: V's scale is part of
    the weights' exponent."""
    torch, _, _ = _t()
    rng = np.random.default_rng(1)
    d = Device(2, 16, 64, "int8", [100], rng)
    k, v = (_rows(torch, rng, 100, 2, 64, "f32") for _ in range(2))
    size = torch.ones(100, device="cuda")
    size[16:32], size[32:48], size[48:64] = 2.0 ** 40, 2.0 ** -20, 0.0
    d.append([100], [100], k, v * size[:, None, None])
    q = _rows(torch, rng, 1, 4, 64, dtype)
    for scale in (1e-30, 0.01, 1.0, 300.0):
        _check_attention(d, [100], [1], 4, dtype, scale=scale, q=q)
    for f in (0.0, 1e-30, 1e30):
        _check_attention(d, [100], [1], 4, dtype, scale=1e-30 if f > 1 else 1.0, q=(q * f).to(q.dtype))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_that_are_not_finite_stay_in_their_rows(dtype):
    torch, types, _ = _t()
    rng = np.random.default_rng(8)
    d = _filled(2, 16, 64, "int8", [50, 0], rng)
    q = _rows(torch, rng, 6, 6, 64, dtype)
    batch = d.batch([50, 0], [4, 2])
    clean, out = torch.empty_like(q), torch.empty_like(q)
    d.cache.attention(batch, q, clean, workspace=_workspace(d, batch, 6))
    q[1, 2, 3], q[2, 5, 0], q[4, 0, 0] = math.nan, -math.inf, math.nan
    d.cache.attention(batch, q, out, workspace=_workspace(d, batch, 6))
    hit = torch.zeros(6, 6, dtype=torch.bool)
    hit[1, 2] = hit[2, 5] = True
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])
    assert (out[4:] == 0).all()  # rows that see nothing are 0 whatever the query


@gpu
def test_rows_behind_the_last_sequence_and_in_place():
    torch, _, _ = _t()
    rng = np.random.default_rng(4)
    d = _filled(2, 64, 64, "int8", [90, 600], rng)
    q = _rows(torch, rng, 20, 6, 64, "f32")
    batch = d.batch([90, 600], [3, 9], rows=20)
    out = torch.full_like(q, 9.0)
    d.cache.attention(batch, q, out, workspace=_workspace(d, batch, 6))
    assert (out[12:] == 9).all() and torch.isfinite(out[:12]).all()
    d.cache.attention(batch, q, q, workspace=_workspace(d, batch, 6))
    assert torch.equal(q[:12], out[:12])


@gpu
def test_two_sequences_share_a_prefix():
    torch, _, _ = _t()
    rng = np.random.default_rng(6)
    d = _filled(2, 32, 64, "int8", [64, 70], rng)
    d.tables[1, :2] = d.tables[0, :2]
    d.dtables.copy_(torch.from_numpy(d.tables))
    _check_attention(d, [64, 70], [1, 1], 4, "f32")


@gpu
def test_pools_beyond_32_bits_of_bytes():
    """Blocks 160 MiB apart, the last above 5 GiB."""
    torch, _, _ = _t()
    rng = np.random.default_rng(7)
    d = Device(2, 64, 64, "int8", [34 * 64 - 5], rng, spare=0)
    far = 160 << 20
    pools = [torch.empty(34 * far, dtype=torch.uint8, device="cuda") for _ in range(2)]
    d.k, d.v = (p.view(torch.int8).as_strided((34, 2, 64, 64), (far, 64 * 64, 64, 1)) for p in pools)
    d.cache = KV8Cache(d.k, d.v, d.ks, d.vs)
    n = 34 * 64 - 5
    d.append([n], [n], *(_rows(torch, rng, n, 2, 64, "bf16", 0.5) for _ in range(2)))
    _check_attention(d, [n], [1], 6, "f32")
    _check_attention(d, [n], [70], 6, "bf16")
    k = torch.empty(n, 2, 64, device="cuda")
    d.cache.read(d.batch([n], [n]), k)
    assert torch.equal(k.cpu(), d.plain.rows(d.tables[0], n, n)[0])


@gpu
def test_captured_steps_on_another_stream():
    """A decoding step (append, attention) captured once and replayed while the lengths grow; the workspace is the
    graph's own."""
    torch, _, _ = _t()
    rng = np.random.default_rng(11)
    n0, steps, heads = 1000, 4, 14
    d = Device(2, 64, 64, "int8", [n0 + steps, 30 + steps], rng)
    d.append([n0, 30], [n0, 30], *(_rows(torch, rng, n0 + 30, 2, 64, "f32", 0.5) for _ in range(2)))
    lens = torch.tensor([n0, 30], dtype=torch.int32, device="cuda")
    batch = KV8Batch(lens, d.dtables, rows=2, max_len=n0 + steps)
    k, v = (torch.empty(2, 2, 64, device="cuda") for _ in range(2))
    q, out = torch.empty(2, heads, 64, device="cuda"), torch.empty(2, heads, 64, device="cuda")
    w = _workspace(d, batch, heads)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        lens.add_(1)
        st = torch.cuda.current_stream().cuda_stream
        d.cache.append(batch, k, v, stream=st)
        d.cache.attention(batch, q, out, workspace=w, stream=st)
    for step in range(1, steps + 1):
        k.copy_(_rows(torch, rng, 2, 2, 64, "f32"))
        v.copy_(_rows(torch, rng, 2, 2, 64, "f32"))
        q.copy_(_rows(torch, rng, 2, heads, 64, "f32"))
        graph.replay()
        torch.cuda.synchronize()
        now = [n0 + step, 30 + step]
        for i in range(2):
            d.plain.append(d.tables[i], now[i], torch.stack([k[i:i + 1], v[i:i + 1]]).cpu())
        d.same_as_plain(now)
        want, size = _reference(d, now, [1, 1], q.cpu(), 0.125, 0)
        assert ((out.cpu().double() - want).abs() <= _tolerance(size, n0, 64, "f32", want)).all()


@gpu
def test_bounds_that_are_too_small_shift_nothing():
    """max_new and max_len below what a sequence has: its first rows are taken, at their own positions, and positions
    past max_len are not seen."""
    torch, _, _ = _t()
    rng = np.random.default_rng(14)
    d = _filled(2, 16, 64, "int8", [100], rng)
    k, v = (_rows(torch, rng, 20, 2, 64, "f32") for _ in range(2))
    batch = KV8Batch(torch.tensor([100], dtype=torch.int32).cuda(), d.dtables, torch.tensor([0, 20], dtype=torch.int32).cuda(),
                     rows=20, max_new=7, max_len=60)
    d.cache.append(batch, k, v)  # positions 80..86
    d.plain.append(d.tables[0], 87, torch.stack([k[:7], v[:7]]).cpu())
    d.same_as_plain([87])
    out = torch.full((20, 2, 64), 5.0, device="cuda")
    d.cache.read(batch, out)
    assert torch.equal(out[:7].cpu(), d.plain.rows(d.tables[0], 87, 7)[0]) and (out[7:] == 5).all()
    q = _rows(torch, rng, 20, 4, 64, "f32")
    got, want = torch.full_like(q, 5.0), torch.full((7, 4, 64), 5.0, device="cuda")
    d.cache.attention(batch, q, got, workspace=_workspace(d, batch, 4))
    one = KV8Batch(torch.tensor([60], dtype=torch.int32).cuda(), d.dtables, rows=1)
    for r in range(7):  # each of the rows sees positions 0..59
        d.cache.attention(one, q[r:r + 1], want[r:r + 1], workspace=_workspace(d, one, 4))
    # (the two batches may cut the positions into parts differently: two results within their tolerance)
    _, size = _reference(d, [60], [1], q[:1].cpu(), 0.125, 0)
    tol = 2 * _tolerance(size.expand(7, 2).clone(), 60, 64, "f32", want.cpu().double())
    s = torch.einsum("rhd,rhd->rh", q[:7].cpu().double().abs(), torch.ones(7, 4, 64, dtype=torch.float64)).max()
    big = 0.125 * s * d.plain.rows(d.tables[0], 60, 60).abs().max().double()  # scale sum |q| max |k| bounds every row's S
    tol = tol.maximum(2 * _tolerance(torch.stack([big, size[0, 1]]).expand(7, 2).clone(), 60, 64, "f32", want.cpu().double()))
    assert ((got[:7] - want).abs().cpu().double() <= tol).all() and (got[7:] == 5).all()


@gpu
def test_calls_at_once_on_two_streams():
    """Decoding, a chunk and reads of two caches on two streams, each with its own workspace, as one after the other."""
    torch, _, _ = _t()
    rng = np.random.default_rng(15)
    jobs = []
    for lens, new, dtype in (([3000, 500], [1, 1], "f32"), ([900, 1500], [200, 300], "bf16")):
        d = _filled(2, 64, 64, "int8", lens, rng)
        q = _rows(torch, rng, sum(new), 14, 64, dtype)
        batch, every = d.batch(lens, new, max_new=max(new)), d.batch(lens, lens)
        out, k = torch.empty_like(q), torch.empty(sum(lens), 2, 64, device="cuda")
        w = _workspace(d, batch, 14)

        def job(d=d, q=q, batch=batch, every=every, out=out, k=k, w=w):
            s = torch.cuda.current_stream().cuda_stream
            d.cache.attention(batch, q, out, workspace=w, stream=s)
            d.cache.read(every, k, stream=s)

        job()
        torch.cuda.synchronize()
        jobs.append((job, out, out.clone(), k, k.clone()))
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(20):
        for (job, out, _, k, _), s in zip(jobs, streams):
            with torch.cuda.stream(s):
                out.fill_(7)
                k.fill_(7)
                job()
        torch.cuda.synchronize()
        for _, out, want, k, want_k in jobs:
            assert torch.equal(out, want) and torch.equal(k, want_k)


@gpu
def test_refusals_on_the_device():
    """Host memory, a missing workspace, and no rows."""
    torch, _, _ = _t()
    rng = np.random.default_rng(12)
    d = _filled(2, 64, 64, "int8", [3000], rng)
    q = _rows(torch, rng, 1, 14, 64, "f32")
    batch = d.batch([3000])
    n = d.cache.attention_workspace(batch, 14)
    assert n > 0
    out = torch.empty_like(q)
    with pytest.raises(LlmError, match="workspace"):
        d.cache.attention(batch, q, out)
    with pytest.raises(LlmError, match="workspace"):
        d.cache.attention(batch, q, out, workspace=torch.empty(n // 2, dtype=torch.uint8, device="cuda"))
    with pytest.raises(LlmError, match="not device memory"):
        d.cache.attention(batch, q.cpu(), out, workspace=_workspace(d, batch, 14))
    with pytest.raises(LlmError, match="not device memory"):
        d.cache.append(d.batch([3000]), torch.zeros(1, 2, 64), torch.zeros(1, 2, 64))
    none = d.batch([3000], [0])
    e = torch.empty(0, 14, 64, device="cuda")
    d.cache.attention(none, e, e, workspace=_workspace(d, none, 14))
    d.cache.read(none, torch.empty(0, 2, 64, device="cuda"))
    d.cache.append(none, *(torch.empty(0, 2, 64, device="cuda") for _ in range(2)))
    torch.cuda.synchronize()


@gpu
def test_the_rows_read_back_are_the_float32_attentions_cache():
    """llmb_kv8_read gives llmb_attention_noalloc its rows, and both attentions agree."""
    torch, _, _ = _t()
    rng = np.random.default_rng(13)
    n, kv, heads, hd = 777, 3, 9, 64
    d = _filled(kv, 32, hd, "e4m3", [n], rng)
    k, v = (torch.empty(n, kv, hd, device="cuda") for _ in range(2))
    d.cache.read(d.batch([n], [n]), k, v)
    q = _rows(torch, rng, 1, heads, hd, "f32")
    out = torch.empty_like(q)
    st = torch.cuda.current_stream().cuda_stream
    assert llm_b200.lib().llmb_attention_noalloc(q.data_ptr(), k.data_ptr(), v.data_ptr(), n, heads, kv, hd, kv * hd,
                                                 out.data_ptr(), st) == llm_b200.OK
    got = _check_attention(d, [n], [1], heads, "f32", q=q)
    want, size = _reference(d, [n], [1], q.cpu(), 1 / 8, 0)
    tol = _tolerance(size, n, hd, "f32", want)
    assert ((out.cpu().double() - want).abs() <= tol).all() and ((out - got).abs().cpu() <= 2 * tol).all()
