"""The 8-bit key/value cache where callers' own scales, windows and bounds reach its limits.

Helpers, the plain restatement and the tolerances are test_kv8.py's.
"""

import ctypes as C
import math
import random

import numpy as np
import pytest

import llm_b200
from llm_b200 import LlmError
from tests.test_kv8 import DTYPES, Device, _filled, _reference_by_head, _rows, _t, _tolerance, _workspace

gpu = pytest.mark.gpu


def _scale(d, kind, table, values):
    """Gives the blocks of a sequence other scales over the bytes they have: values for its first blocks."""
    torch, _, _ = _t()
    for b, s in zip(table, values):
        (d.ks, d.vs)[kind][b] = s
        d.plain.scale[kind, b] = s


def _attention(d, lens, new, heads, dtype, q, window=0):
    """(result, float64 reference, tolerance)"""
    torch, _, _ = _t()
    batch = d.batch(lens, new)
    out = torch.full_like(q, math.nan)
    d.cache.attention(batch, q, out, window=window, workspace=_workspace(d, batch, heads))
    want, size = _reference_by_head(d, lens, new, q.cpu(), 1 / math.sqrt(d.hd), window)
    return out.cpu().double(), want, _tolerance(size, max(lens), d.hd, dtype, want)


# Rows of the call: one token (the kernel for few rows) and enough for the tensor cores' tiles.
ROWS = (1, 400)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("cache,hd", [("int8", 64), ("e4m3", 128)])
def test_a_scale_of_0_makes_values_0_whatever_the_bytes(cache, hd, rows, dtype):
    """Blocks whose V scale a caller cleared, or made smaller than float32's normal numbers, are as read gives them in
    the attention too, and their positions count in the softmax."""
    torch, _, _ = _t()
    rng = np.random.default_rng(21)
    n, kv, heads = 1500, 2, 8
    d = _filled(kv, 32, hd, cache, [n], rng)
    _scale(d, 1, d.tables[0][3::5], [0.0, 2.0 ** -130, 0.0, 2.0 ** -149, 2.0 ** -115, 0.0])
    k, v = (torch.empty(n, kv, hd, device="cuda") for _ in range(2))
    d.cache.read(d.batch([n], [n]), k, v)
    assert torch.equal(v.cpu(), d.plain.rows(d.tables[0], n, n)[1]) and (v[96:128] == 0).all()
    q = _rows(torch, rng, rows, heads, hd, dtype, 0.3)
    got, want, tol = _attention(d, [n], [rows], heads, dtype, q)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
    # and where no block has a scale, the result is 0
    _scale(d, 1, d.tables[0], [0.0] * len(d.tables[0]))
    got, _, _ = _attention(d, [n], [rows], heads, dtype, q)
    assert (got == 0).all()


@gpu
@pytest.mark.parametrize("dtype,size", [("f32", 2.0 ** -40), ("f32", 2.0 ** 20), ("f16", 2.0 ** -9), ("bf16", 2.0 ** -40),
                                        ("bf16", 2.0 ** 30)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("zeros", ["between", "before"])
def test_blocks_of_zeros_beside_values_of_any_size(zeros, rows, dtype, size):
    """Positions whose values are all 0 take their part of the softmax and nothing of the others' precision: between
    blocks of small or large values, and where a part of the positions starts with thousands of them."""
    torch, _, _ = _t()
    rng = np.random.default_rng(22)
    n, kv, heads, hd = 6000, 1, 4, 64
    d = Device(kv, 16, hd, "int8", [n], rng)
    k, v = (_rows(torch, rng, n, kv, hd, "f32", 0.3) for _ in range(2))
    v *= size
    if zeros == "between":
        for at in (0, 320, 1024, 4000):
            v[at:at + 32] = 0
    else:
        v[:4096] = 0
    d.append([n], [n], k, v)
    q = _rows(torch, rng, rows, heads, hd, dtype, 0.3)
    got, want, tol = _attention(d, [n], [rows], heads, dtype, q)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", ROWS)
def test_many_of_the_smallest_values(rows, dtype):
    """20000 positions of values just above 2^-100, the least that append keeps: the sum of the weights, in which the
    scale's inverse stands, stays finite."""
    torch, _, _ = _t()
    rng = np.random.default_rng(23)
    n, kv, heads, hd = 20000, 1, 2, 64
    d = Device(kv, 128, hd, "e4m3", [n], rng)
    k = 0.01 * _rows(torch, rng, n, kv, hd, "f32", 0.0)
    v = 2.0 ** -100 * (1 + 0.01 * torch.rand(n, kv, hd, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    d.append([n], [n], k, v)
    assert float(d.vs[torch.from_numpy(d.tables[0]).long()].min()) >= 2.0 ** -109
    q = _rows(torch, rng, rows, heads, hd, dtype, 0.0)
    got, want, tol = _attention(d, [n], [rows], heads, dtype, q)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cache", ["int8", "e4m3"])
def test_append_behind_scales_of_the_callers(cache, dtype):
    """Rows below 2^-100 leave a block's scale as it is; where that is smaller than they need they saturate, and no byte
    is a NaN or has another sign, down to scales whose inverse is not finite."""
    torch, types, caches = _t()
    rng = np.random.default_rng(24)
    kv, block, hd = 2, 16, 64
    scales = [2.0 ** -107, 2.0 ** -112, 2.0 ** -126, 2.0 ** -130, 2.0 ** -149, 2.0 ** -90, 1.0]
    for size in (0.0, 2.0 ** -101, 2.0 ** -105, 2.0 ** -125):
        d = Device(kv, block, hd, cache, [9] * len(scales), rng)
        n = len(scales)
        d.append([5] * n, [5] * n, *(_rows(torch, rng, 5 * n, kv, hd, "f32") for _ in range(2)))
        for i, s in enumerate(scales):
            for kind in range(2):
                _scale(d, kind, d.tables[i], [s])
        x = torch.from_numpy(rng.uniform(0.3, 0.9, (4 * n, kv, hd)).astype(np.float32))
        x[1::3] *= -1
        x = (x * size).to(types[dtype]).cuda()
        with np.errstate(over="ignore"):  # (the restatement's inverse)
            d.append([9] * n, [4] * n, x, -x)
        d.same_as_plain([9] * n)
        bytes_ = d.k.view(torch.uint8)[torch.from_numpy(d.tables[:, 0]).long(), :, :9]
        if cache == "e4m3":
            assert not ((bytes_ & 0x7f) == 0x7f).any()


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new,heads", [([10, 700], [14, 3], 2), ([900, 40], [1000, 300], 8)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 16385, 5])
def test_windows_up_to_the_largest_integer(window, lens, new, heads, dtype):
    """The largest window is none, also for sequences with more rows than positions, whose first rows see nothing."""
    torch, _, _ = _t()
    rng = np.random.default_rng(25)
    d = _filled(2, 16, 64, "int8", lens, rng)
    q = _rows(torch, rng, sum(new), heads, 64, dtype, 0.3)
    got, want, tol = _attention(d, lens, new, heads, dtype, q, window=window)
    assert ((got - want).abs() <= tol).all()
    if window > 5:
        whole, _, _ = _attention(d, lens, new, heads, dtype, q)
        # (another window may cut the positions into other parts: two results within their tolerance)
        assert ((got - whole).abs() <= 2 * tol).all() and (got[:new[0] - lens[0]] == 0).all()


# ---------------------------------------------------------------- the workspace's size, without a GPU


def _need(c, b, heads, type_, window, said):
    """Whether the call accepts a workspace of that many bytes (what comes after that check fails here: no memory of a
    GPU)."""
    L = llm_b200.lib()
    cache = C.cast(c, C.POINTER(llm_b200._KV8Cache)).contents
    width = heads * cache.head_dim
    assert L.llmb_kv8_attention(c, b, 4096, width, 4096, width, type_, heads, 0.0, window, 4096, said, None) != llm_b200.OK
    return b"a workspace of" not in L.llmb_last_error(None)


def _sizes(seqs, rows, max_new, max_len, kv, hd, block=64):
    c = llm_b200._KV8Cache(4096, 8192, 256, 512, kv * block * hd, 8, block, kv, hd, 0)
    return C.byref(c), C.byref(llm_b200._KV8Batch(256, 512, 1024, seqs, -(-max_len // block), rows, max_new, max_len))


@pytest.mark.parametrize("seqs,rows,max_new,max_len,at_most", [(3, 2563, 1023, 5000, 200 << 20), (1, 8192, 8192, 8192, 300 << 20),
                                                               (16, 16 * 4096, 4096, 4096, 0), (64, 64 * 4096, 4096, 4096, 0)])
def test_the_workspace_of_prompts_is_what_their_cut_can_need(seqs, rows, max_new, max_len, at_most):
    """32 heads on 8 of size 128.  (An attention's own output for 64 prompts of 4096 is 2 GiB in bfloat16.)"""
    c, b = _sizes(seqs, rows, max_new, max_len, 8, 128)
    said = llm_b200.lib().llmb_kv8_attention_workspace(c, b, 32)
    assert 0 <= said <= at_most


def test_no_call_needs_more_workspace_than_is_said():
    rng = random.Random(1)
    split = 0
    for _ in range(1500):
        kv, group, hd = rng.choice([1, 2, 3, 8]), rng.choice([1, 3, 4, 7, 64]), rng.choice([64, 128])
        seqs, max_new = int(2 ** rng.uniform(0, 8)), int(2 ** rng.uniform(0, 13))
        rows = rng.randint(max_new, max_new * seqs)
        max_len = int(2 ** rng.uniform(0, 20))
        c, b = _sizes(seqs, rows, max_new, max_len, kv, hd)
        said = llm_b200.lib().llmb_kv8_attention_workspace(c, b, kv * group)
        assert said >= 0
        for window in [0] + [int(2 ** rng.uniform(0, 20)) for _ in range(6)]:
            for type_ in range(3):
                assert _need(c, b, kv * group, type_, window, said), (seqs, rows, max_new, max_len, kv, group, hd, window, type_)
                split += not _need(c, b, kv * group, type_, window, 0)
    assert split > 5000  # (many of the calls are cut)


# ---------------------------------------------------------------- the Python objects, without a GPU


def _objects():
    torch, _, _ = _t()
    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.ones(4, 2)
    lens, tables = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    return llm_b200.KV8Cache(k, k, s, s), lens, tables


def test_sizes_that_the_kernels_go_by_cannot_be_changed():
    """What the tensors are checked against is what the C structures hold."""
    torch, _, _ = _t()
    cache, lens, tables = _objects()
    batch = llm_b200.KV8Batch(lens, tables, rows=2)
    assert (batch.rows, cache.kv_heads, cache.head_dim) == (2, 2, 64)
    for o, name in ((batch, "rows"), (cache, "kv_heads"), (cache, "head_dim")):
        with pytest.raises(AttributeError):
            setattr(o, name, 1)
    x = torch.zeros(1, 2, 64)
    with pytest.raises(LlmError):
        cache.append(batch, x, x)


def test_sizes_past_32_bits_are_refused():
    cache, lens, tables = _objects()
    for kw in (dict(rows=1 << 32), dict(rows=2, max_new=(1 << 32) + 1), dict(rows=2, max_len=1 << 31), dict(rows=-(1 << 40))):
        with pytest.raises(LlmError, match="out of range"):
            llm_b200.KV8Batch(lens, tables, **kw)
    with pytest.raises(LlmError, match="out of range"):
        cache.attention_workspace(llm_b200.KV8Batch(lens, tables, rows=2), (1 << 32) + 14)


@gpu
def test_the_largest_length_beside_a_long_sequence():
    """A length of 2^31 - 1 in a batch with a sequence of many rows: its rows are 0 (no table reaches there), and no other
    row is written, nor any byte of the cache."""
    torch, _, _ = _t()
    rng = np.random.default_rng(26)
    d = _filled(2, 16, 64, "int8", [100, 100], rng)
    before = d.k.clone(), d.v.clone(), d.ks.clone(), d.vs.clone()
    m = 40000
    batch = d.batch([2 ** 31 - 1, -1], [3, m], rows=m + 5)
    k = torch.full((m + 5, 2, 64), 5.0, device="cuda")
    d.cache.append(batch, k, k)
    d.cache.read(batch, k)
    assert (k[:m + 3] == 0).all() and (k[m + 3:] == 5).all()
    for a, b in zip(before, (d.k, d.v, d.ks, d.vs)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_in_place_with_another_stride_is_refused():
    """Rows would be overwritten before others have read them."""
    L, arg = llm_b200.lib(), llm_b200.ERR_ARG
    c, b = _sizes(2, 4, 2, 100, 2, 64)
    for q_stride, out_stride, refused in ((512, 256, True), (256, 512, True), (256, 256, False)):
        rc = L.llmb_kv8_attention(c, b, 4096, q_stride, 4096, out_stride, 0, 4, 0.0, 0, 4096, 1 << 30, None)
        assert rc != llm_b200.OK and (b"another stride" in L.llmb_last_error(None)) == refused
        ctl = llm_b200._LogitsCtl()
        rc = L.llmb_logits_control(4096, q_stride, 0, 2, 200, C.byref(ctl), 4096, out_stride, 256, None)
        assert rc != llm_b200.OK and (b"another stride" in L.llmb_last_error(None)) == refused
        assert not refused or rc == arg
