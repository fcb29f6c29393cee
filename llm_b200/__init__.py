"""B200 forward pass for go-wasmcontainers/llm: the host-side mirror of ``llm.GPU``.

The compute path is libllmb200.so (hand-written sm_100a CUDA behind the C ABI
of include/llm_b200.h). This module binds that ABI with ctypes and mirrors the
reference's Go API (gpu.go): ``NewGPU`` opens a GGUF model onto a device,
``GPU.generate`` decodes greedily (``Generate``, gpu.go:946),
``GPU.prefill_logits`` returns the last prompt token's logits
(``PrefillLogits``, gpu.go:904), ``GPU.peek`` reads a named buffer (``Peek``,
gpu.go:1018), ``GPU.memory_used`` (gpu.go:767), ``GPU.stats`` (gpu.go:56),
``GPU.layers`` (gpu.go:143-146) and the package knobs ``DecodeBatch`` and
``PrefillBatch`` (gpu.go:1052,165). Errors raise ``LlmError`` with the
library's status code, as the Go functions return ``error``.

There is no CPU fallback: importing this package fails when the library has
not been built (``python -m llm_b200.build``).
"""

from __future__ import annotations

import ctypes as C
import importlib
import os
from dataclasses import dataclass

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libllmb200.so")

OK, ERR_ARG, ERR_IO, ERR_FORMAT, ERR_BOUND, ERR_CONFIG, ERR_TENSOR, ERR_MEMORY, ERR_CONTEXT, ERR_CUDA, ERR_DEVICE = range(11)

# Every function include/llm_b200.h declares.
EXPORTS = ("llmb_open", "llmb_open_reader", "llmb_close", "llmb_last_error", "llmb_get_config", "llmb_memory_used",
           "llmb_get_stats", "llmb_generate", "llmb_generate_batch", "llmb_prefill_logits", "llmb_generate_logits",
           "llmb_peek",
           "llmb_set_layers", "llmb_set_knob", "llmb_get_knob", "llmb_attention_noalloc", "llmb_kv8_append",
           "llmb_kv8_read", "llmb_kv8_attention", "llmb_kv8_attention_workspace", "llmb_logits_control",
           "llmb_generate_controlled")

F32, F16, BF16 = range(3)            # types of rows and logits
KV8_INT8, KV8_E4M3 = range(2)        # types of the 8-bit cache


class LlmError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{msg} (status {code})")
        self.code = code


class _Config(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("layers", "embd", "ff", "heads", "kv_heads", "head_dim", "vocab", "ctx")] + \
               [("rope_base", C.c_float), ("eps", C.c_float)] + \
               [(n, C.c_int32) for n in ("rope_neox", "bias", "tied_output")] + [("arch", C.c_char * 16)]


class _Stats(C.Structure):
    _fields_ = [("submits", C.c_int64), ("dispatches", C.c_int64), ("tokens", C.c_int64)]


class _Timing(C.Structure):
    _fields_ = [("prefill_ms", C.c_double), ("decode_ms", C.c_double), ("prompt_tokens", C.c_int32),
                ("generated", C.c_int32), ("submits", C.c_int64), ("dispatches", C.c_int64),
                ("record_ms", C.c_double), ("submit_ms", C.c_double), ("gpu_prefill_ms", C.c_double),
                ("gpu_decode_ms", C.c_double), ("decode_kernel_ms", C.c_double), ("decode_launches", C.c_int64)]


class _KV8Cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [("block_stride", C.c_int64)] + \
               [(n, C.c_int32) for n in ("n_blocks", "block", "kv_heads", "head_dim", "type")]


class _KV8Batch(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("lens", "tables", "starts")] + \
               [(n, C.c_int32) for n in ("n_seq", "table_stride", "n_rows", "max_new", "max_len")]


class _LogitsCtl(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("history", "history_lens", "prompt_lens")] + \
               [(n, C.c_int32) for n in ("history_stride", "n_bias")] + \
               [(n, C.c_void_p) for n in ("penalties", "bias_ids", "bias_values", "bias_starts", "mask")] + \
               [("mask_stride", C.c_int32)]


MASK_FN = C.CFUNCTYPE(C.c_int, C.c_void_p, C.POINTER(C.c_int32), C.c_int, C.POINTER(C.c_uint32))


class _Controls(C.Structure):
    _fields_ = [(n, C.c_float) for n in ("repetition", "presence", "frequency")] + \
               [("n_bias", C.c_int32), ("bias_ids", C.c_void_p), ("bias_values", C.c_void_p), ("mask", MASK_FN),
                ("mask_user", C.c_void_p)]


READ_FN = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_uint64, C.c_void_p, C.c_uint64)
EMIT_FN = C.CFUNCTYPE(C.c_int, C.c_void_p, C.c_int32)

_lib = None


def lib() -> C.CDLL:
    """The loaded C-ABI library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python -m llm_b200.build` (no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        P, I = C.c_void_p, C.c_int
        L.llmb_open.argtypes, L.llmb_open.restype = [C.c_char_p, I, I, C.POINTER(P)], I
        L.llmb_open_reader.argtypes, L.llmb_open_reader.restype = [READ_FN, P, C.c_uint64, I, I, C.POINTER(P)], I
        L.llmb_close.argtypes, L.llmb_close.restype = [P], None
        L.llmb_last_error.argtypes, L.llmb_last_error.restype = [P], C.c_char_p
        L.llmb_get_config.argtypes, L.llmb_get_config.restype = [P, C.POINTER(_Config)], I
        L.llmb_memory_used.argtypes, L.llmb_memory_used.restype = [P], C.c_uint64
        L.llmb_get_stats.argtypes, L.llmb_get_stats.restype = [P, C.POINTER(_Stats)], I
        L.llmb_generate.argtypes = [P, P, I, I, C.c_int32, EMIT_FN, P, P, C.POINTER(I), C.POINTER(_Timing)]
        L.llmb_generate.restype = I
        L.llmb_generate_batch.argtypes = [P, P, P, I, I, C.c_int32, P, P, C.POINTER(_Timing)]
        L.llmb_generate_batch.restype = I
        L.llmb_generate_controlled.argtypes = [P, P, I, I, C.c_int32, C.POINTER(_Controls), EMIT_FN, P, P, C.POINTER(I),
                                               C.POINTER(_Timing)]
        L.llmb_generate_controlled.restype = I
        L.llmb_prefill_logits.argtypes, L.llmb_prefill_logits.restype = [P, P, I, P], I
        L.llmb_generate_logits.argtypes, L.llmb_generate_logits.restype = [P, P, I, I, P, P], I
        L.llmb_peek.argtypes, L.llmb_peek.restype = [P, C.c_char_p, P, I], I
        L.llmb_set_layers.argtypes, L.llmb_set_layers.restype = [P, I], I
        L.llmb_set_knob.argtypes, L.llmb_set_knob.restype = [C.c_char_p, C.c_int64], I
        L.llmb_get_knob.argtypes, L.llmb_get_knob.restype = [C.c_char_p], C.c_int64
        L.llmb_attention_noalloc.argtypes = [P, P, P, I, I, I, I, I, P, P]
        L.llmb_attention_noalloc.restype = I
        Q, F = C.c_int64, C.c_float
        kv8 = [C.POINTER(_KV8Cache), C.POINTER(_KV8Batch)]
        L.llmb_kv8_append.argtypes, L.llmb_kv8_append.restype = kv8 + [P, P, I, Q, P], I
        L.llmb_kv8_read.argtypes, L.llmb_kv8_read.restype = kv8 + [P, P, I, Q, P], I
        L.llmb_kv8_attention.argtypes = kv8 + [P, Q, P, Q, I, I, F, I, P, Q, P]
        L.llmb_kv8_attention.restype = I
        L.llmb_kv8_attention_workspace.argtypes, L.llmb_kv8_attention_workspace.restype = kv8 + [I], Q
        L.llmb_logits_control.argtypes = [P, Q, I, I, I, C.POINTER(_LogitsCtl), P, Q, P, P]
        L.llmb_logits_control.restype = I
        _lib = L
    return _lib


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def set_knob(name: str, value: int) -> None:
    """Sets a package knob: decode_batch, prefill_batch, memory_budget, decode_mode, prefill_mode, tag_reset,
    attn_positions, decode_trace, wait_limit_us or drop_publish (include/llm_b200.h describes each)."""
    if lib().llmb_set_knob(name.encode(), int(value)) != OK:
        raise LlmError(ERR_ARG, f"llm: no knob {name!r}")


def get_knob(name: str) -> int:
    return lib().llmb_get_knob(name.encode())


@dataclass
class Config:
    """llm.Config (config.go:11-23)."""

    layers: int
    embd: int
    ff: int
    heads: int
    kv_heads: int
    head_dim: int
    vocab: int
    ctx: int
    rope_base: float
    eps: float
    rope_neox: bool
    bias: bool
    tied_output: bool
    arch: str


@dataclass
class Timing:
    """llm.Timing (gpu.go:929-939) plus device time from CUDA events."""

    prefill_ms: float
    decode_ms: float
    prompt_tokens: int
    generated: int
    submits: int
    dispatches: int
    record_ms: float
    submit_ms: float
    gpu_prefill_ms: float
    gpu_decode_ms: float
    decode_kernel_ms: float
    decode_launches: int


class GPU:
    """The forward pass on one B200 (llm.GPU, gpu.go:115-159)."""

    def __init__(self, path: str | None = None, ctx: int = 0, device: int = 0, reader=None, size: int = 0):
        self._h = C.c_void_p()
        self._keep = None
        if reader is not None:
            def _read(_user, off, buf, n):
                try:
                    data = reader(off, n)
                    if len(data) < n:
                        return 1
                    C.memmove(buf, data, n)
                    return 0
                except Exception:
                    return 1

            self._keep = READ_FN(_read)
            rc = lib().llmb_open_reader(self._keep, None, size, ctx, device, C.byref(self._h))
        else:
            rc = lib().llmb_open(os.fsencode(path), ctx, device, C.byref(self._h))
        if rc != OK:
            raise LlmError(rc, lib().llmb_last_error(None).decode(errors="replace"))
        c = _Config()
        lib().llmb_get_config(self._h, C.byref(c))
        self.cfg = Config(c.layers, c.embd, c.ff, c.heads, c.kv_heads, c.head_dim, c.vocab, c.ctx, c.rope_base, c.eps,
                          bool(c.rope_neox), bool(c.bias), bool(c.tied_output), c.arch.decode())

    def _check(self, rc: int) -> None:
        if rc != OK:
            raise LlmError(rc, lib().llmb_last_error(self._h).decode(errors="replace"))

    def close(self) -> None:
        if self._h:
            lib().llmb_close(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.close()

    def memory_used(self) -> int:
        return lib().llmb_memory_used(self._h)

    @property
    def stats(self) -> dict:
        s = _Stats()
        self._check(lib().llmb_get_stats(self._h, C.byref(s)))
        return dict(submits=s.submits, dispatches=s.dispatches, tokens=s.tokens)

    @property
    def layers(self) -> int:
        return getattr(self, "_layers", 0)

    @layers.setter
    def layers(self, n: int) -> None:
        self._check(lib().llmb_set_layers(self._h, int(n)))
        self._layers = int(n)

    def generate(self, prompt, n: int, eos: int = -1, emit=None) -> tuple[np.ndarray, Timing]:
        """Greedy decoding (Generate, gpu.go:946): returns the emitted tokens and the timing."""
        p = np.ascontiguousarray(prompt, np.int32)
        out = np.zeros(max(n, 1), np.int32)
        n_out = C.c_int()
        tm = _Timing()
        cb = EMIT_FN()
        if emit is not None:
            cb = EMIT_FN(lambda _u, t: 1 if emit(int(t)) else 0)
        self._check(lib().llmb_generate(self._h, _ptr(p), len(p), n, eos, cb, None, _ptr(out), C.byref(n_out),
                                        C.byref(tm)))
        t = Timing(tm.prefill_ms, tm.decode_ms, tm.prompt_tokens, tm.generated, tm.submits, tm.dispatches,
                   tm.record_ms, tm.submit_ms, tm.gpu_prefill_ms, tm.gpu_decode_ms, tm.decode_kernel_ms,
                   tm.decode_launches)
        return out[: n_out.value].copy(), t

    def generate_batch(self, prompts, n: int, eos: int = -1) -> tuple[list[np.ndarray], Timing]:
        """Independent greedy sequences, one KV cache each (llmb_generate_batch): the tokens of each, and the timing."""
        ps = [np.ascontiguousarray(p, np.int32) for p in prompts]
        flat = np.concatenate(ps) if ps else np.zeros(0, np.int32)
        lens = np.array([len(p) for p in ps], np.int32)
        out = np.zeros((len(ps), max(n, 1)), np.int32)
        n_out = np.zeros(len(ps), np.int32)
        tm = _Timing()
        self._check(lib().llmb_generate_batch(self._h, _ptr(flat), _ptr(lens), len(ps), n, eos, _ptr(out),
                                              _ptr(n_out), C.byref(tm)))
        t = Timing(tm.prefill_ms, tm.decode_ms, tm.prompt_tokens, tm.generated, tm.submits, tm.dispatches,
                   tm.record_ms, tm.submit_ms, tm.gpu_prefill_ms, tm.gpu_decode_ms, tm.decode_kernel_ms,
                   tm.decode_launches)
        return [out[i, : n_out[i]].copy() for i in range(len(ps))], t

    def generate_controlled(self, prompt, n: int, eos: int = -1, repetition: float = 1.0, presence: float = 0.0,
                            frequency: float = 0.0, biases: dict | None = None, mask=None,
                            emit=None) -> tuple[np.ndarray, Timing]:
        """Greedy decoding with penalties for repeated tokens, biases {token: value} and a grammar
        (llmb_generate_controlled): mask(tokens, allowed) is given the tokens so far (int32) and the mask to fill
        (uint32, bit v % 32 of word v / 32 is token v) and returns whether to go on. An exception of mask or emit
        stops the generation and is raised."""
        p = np.ascontiguousarray(prompt, np.int32)
        out = np.zeros(max(n, 1), np.int32)
        ids = np.array(list(biases or {}), np.int32)
        values = np.array(list((biases or {}).values()), np.float32)
        raised = []
        words = (self.cfg.vocab + 31) // 32

        def guarded(f):
            def call(*a):
                try:
                    return 1 if f(*a) else 0
                except BaseException as e:
                    raised.append(e)
                    return 0
            return call

        mask_fn, emit_fn = MASK_FN(), EMIT_FN()
        if mask is not None:
            allowed = np.zeros(words, np.uint32)  # the callback's to keep: the library's own words end with the model

            def fill(_u, t, k, w):
                go = mask(np.ctypeslib.as_array(t, (k,)).copy() if k else np.zeros(0, np.int32), allowed)
                C.memmove(w, allowed.ctypes.data, allowed.nbytes)
                return go

            mask_fn = MASK_FN(guarded(fill))
        if emit is not None:
            emit_fn = EMIT_FN(guarded(lambda _u, t: emit(int(t))))
        c = _Controls(repetition, presence, frequency, len(ids), ids.ctypes.data, values.ctypes.data, mask_fn, None)
        n_out, tm = C.c_int(), _Timing()
        rc = lib().llmb_generate_controlled(self._h, _ptr(p), len(p), n, eos, c, emit_fn, None, _ptr(out),
                                            C.byref(n_out), C.byref(tm))
        if raised:
            raise raised[0]
        self._check(rc)
        t = Timing(tm.prefill_ms, tm.decode_ms, tm.prompt_tokens, tm.generated, tm.submits, tm.dispatches,
                   tm.record_ms, tm.submit_ms, tm.gpu_prefill_ms, tm.gpu_decode_ms, tm.decode_kernel_ms,
                   tm.decode_launches)
        return out[: n_out.value].copy(), t

    def prefill_logits(self, prompt) -> np.ndarray:
        """The logits of the prompt's last token (PrefillLogits, gpu.go:904)."""
        p = np.ascontiguousarray(prompt, np.int32)
        logits = np.zeros(self.cfg.vocab, np.float32)
        self._check(lib().llmb_prefill_logits(self._h, _ptr(p), len(p), _ptr(logits)))
        return logits

    def generate_logits(self, prompt, n: int) -> tuple[np.ndarray, np.ndarray]:
        """Greedy tokens and the logits that chose each (a test hook)."""
        p = np.ascontiguousarray(prompt, np.int32)
        toks = np.zeros(n, np.int32)
        logits = np.zeros((n, self.cfg.vocab), np.float32)
        self._check(lib().llmb_generate_logits(self._h, _ptr(p), len(p), n, _ptr(toks), _ptr(logits)))
        return toks, logits

    def peek(self, name: str, n: int) -> np.ndarray:
        """The first n words of a named device buffer, as float32 (Peek, gpu.go:1018)."""
        out = np.zeros(n, np.float32)
        self._check(lib().llmb_peek(self._h, name.encode(), _ptr(out), n))
        return out


# ---- operators over the caller's device tensors
#
# These take tensors of any library whose tensors have data_ptr(), shape,
# stride() and dtype (torch's do); the tensors must stay alive, and their
# device current, until the work is done. stream is a cudaStream_t handle
# (torch.cuda.current_stream().cuda_stream), 0 the default stream.
#
# Their checks and calls are in csrc/call.c.

_NAMES = {"float32": F32, "float16": F16, "bfloat16": BF16, "int8": 10, "float8_e4m3fn": 11, "int32": 20, "uint32": 20}


class _Types(dict):
    """dtype -> its entry in _NAMES, or -1."""

    def __missing__(self, dtype):
        self[dtype] = t = _NAMES.get(str(dtype).rsplit(".", 1)[-1], -1)
        return t


_TYPES = _Types()
_native_calls = None


def _refuse(msg: str):
    raise LlmError(ERR_ARG, "llm: " + msg)


def _op_check(rc: int) -> None:
    if rc != OK:
        raise LlmError(rc, lib().llmb_last_error(None).decode(errors="replace"))


def _calls():
    """The native calls, with the library they are linked to."""
    global _native_calls
    if _native_calls is None:
        lib()  # says how to build where it is missing
        try:
            module = importlib.import_module("._native", __name__)
        except ImportError as e:
            raise ImportError(f"{e}: build it with `python -m llm_b200.build` (a C compiler and Python 3.12 or later "
                              "with its headers)") from e
        module.setup(_TYPES, _refuse, _op_check)
        _native_calls = module
    return _native_calls


def _flat(t, what: str, name: str, shape: tuple) -> int:
    """The address of a contiguous tensor of that type and shape."""
    if _TYPES[t.dtype] != _NAMES[name] or tuple(t.shape) != shape or not t.is_contiguous():
        _refuse(f"{what} must be a contiguous {name} tensor of shape {shape}")
    return t.data_ptr()


def _int32(what: str, v: int) -> int:
    """v, which the C structures hold in 32 bits."""
    if not -1 << 31 <= v < 1 << 31:
        _refuse(f"{what} {v} out of range")
    return v


class KV8Batch:
    """The sequences of one call on a KV8Cache (llmb_kv8_batch): lens [n_seq] positions each holds once this call's
    rows are in, tables [n_seq, entries] its block numbers, starts [n_seq + 1] where its rows begin (None: rows / n_seq
    each), all int32 on the device. The tensors' contents may change between calls; max_new and max_len (0: not known)
    bound the rows and the positions of any one sequence. A batch of other sizes is another KV8Batch."""

    def __init__(self, lens, tables, starts=None, rows: int = 0, max_new: int = 0, max_len: int = 0):
        if len(tables.shape) != 2 or len(lens.shape) != 1 or tables.shape[0] != lens.shape[0]:
            _refuse("lens must be [n_seq], tables [n_seq, entries]")
        n, entries = lens.shape[0], tables.shape[1]
        self._keep = (lens, tables, starts)
        for what, x in (("rows", rows), ("max_new", max_new), ("max_len", max_len), ("table entries", entries)):
            _int32(what, x)
        self._c = _KV8Batch(_flat(lens, "lens", "int32", (n,)), _flat(tables, "tables", "int32", (n, entries)),
                            None if starts is None else _flat(starts, "starts", "int32", (n + 1,)),
                            n, entries, rows, max_new, max_len)
        self._at = C.addressof(self._c)
        self._n_rows = rows  # (kept beside the structure: a look into that costs more)

    @property
    def rows(self) -> int:
        """Rows of the calls' tensors; the kernels go by the same number."""
        return self._n_rows


class KV8Cache:
    """Keys and values held in 8 bits with a scale for each block of positions and kv head (llmb_kv8_cache): k, v
    [n_blocks, kv_heads, block, head_dim] of int8 or float8_e4m3fn (blocks may lie any multiple of 16 bytes apart),
    k_scale, v_scale [n_blocks, kv_heads] float32. The tensors are the caller's."""

    def __init__(self, k, v, k_scale, v_scale):
        if len(k.shape) != 4 or k.shape != v.shape:
            _refuse("k and v must be [n_blocks, kv_heads, block, head_dim]")
        n, heads, block, hd = k.shape
        t = _TYPES[k.dtype]
        if t not in (10, 11) or t != _TYPES[v.dtype]:
            _refuse("k and v must both be int8 or both float8_e4m3fn")
        for x in (k, v):
            if tuple(x.stride())[1:] != (block * hd, hd, 1) or x.stride(0) != k.stride(0):
                _refuse("k and v must be contiguous within a block and have one block stride")
        scales = [_flat(x, "a scale", "float32", (n, heads)) for x in (k_scale, v_scale)]
        self._keep = (k, v, k_scale, v_scale)
        self._kv_heads, self._head_dim = heads, hd
        self._c = _KV8Cache(k.data_ptr(), v.data_ptr(), *scales,
                            max(k.stride(0), heads * block * hd) if n == 1 else k.stride(0), n, block, heads, hd,
                            KV8_INT8 if t == 10 else KV8_E4M3)
        self._at = C.addressof(self._c)
        self._rows, self._attend = _calls().rows, _calls().attention

    @property
    def kv_heads(self) -> int:
        return self._kv_heads

    @property
    def head_dim(self) -> int:
        return self._head_dim

    def append(self, batch: KV8Batch, k, v, stream: int = 0) -> None:
        """Writes the rows k, v [rows, kv_heads, head_dim] (llmb_kv8_append)."""
        self._rows(0, self._at, batch._at, batch._n_rows, self._kv_heads, self._head_dim, k, v, stream)

    def read(self, batch: KV8Batch, k=None, v=None, stream: int = 0) -> None:
        """Reads what is held at the rows' positions into k, v [rows, kv_heads, head_dim] (llmb_kv8_read)."""
        self._rows(1, self._at, batch._at, batch._n_rows, self._kv_heads, self._head_dim, k, v, stream)

    def attention_workspace(self, batch: KV8Batch, heads: int) -> int:
        """Bytes of workspace for attention() with that many query heads (llmb_kv8_attention_workspace)."""
        n = lib().llmb_kv8_attention_workspace(C.byref(self._c), C.byref(batch._c), _int32("heads", heads))
        if n < 0:
            _op_check(ERR_ARG)
        return n

    def attention(self, batch: KV8Batch, q, out, scale: float = 0.0, window: int = 0, workspace=None,
                  stream: int = 0) -> None:
        """Attention of the queries q [rows, heads, head_dim] over the cache into out (llmb_kv8_attention); workspace:
        a contiguous tensor of attention_workspace() bytes."""
        self._attend(self._at, batch._at, batch._n_rows, self._head_dim, q, out, scale, window, workspace, stream)


def logits_control(logits, out=None, tokens=None, history=None, history_lens=None, prompt_lens=None, penalties=None,
                   bias_ids=None, bias_values=None, bias_starts=None, mask=None, stream: int = 0) -> None:
    """Penalties for repeated tokens, biases and a grammar's mask on logits [rows, vocab], and the largest that is
    left (llmb_logits_control): out [rows, vocab] (may be logits), tokens [rows] int32; history [rows, n] int32 with
    history_lens, prompt_lens [rows] int32; penalties [rows, 3] float32 (repetition, presence, frequency); bias_ids
    int32 and bias_values float32 [n], with bias_starts [rows + 1] int32 for biases of each row's own; mask
    [rows, ceil(vocab / 32)] int32, bit 1 where a token is allowed."""
    _calls().logits(logits, out, tokens, history, history_lens, prompt_lens, penalties, bias_ids, bias_values, bias_starts,
                   mask, stream)


def NewGPU(path: str, ctx: int = 0, device: int = 0) -> GPU:
    """NewGPU (gpu.go:465): parses the model, allocates its buffers and streams its weights to the device."""
    return GPU(path, ctx, device)
