/*
 * llm_b200.h -- the C ABI of the B200 forward pass for go-wasmcontainers/llm.
 *
 * A drop-in for the reference's GPU forward pass (gpu.go, fused.go,
 * kernels.go, kernels_fused.go): a Go host keeps its llm.GPU API and calls
 * these functions over cgo instead of recording WebGPU passes.  Each entry
 * point names the reference interface it replaces (file:line in the
 * reference repository).  Plain C types only; the library owns all device
 * memory, the caller owns every buffer it passes in.  No call aborts the
 * process: every failure is a status code with a message from
 * llmb_last_error.
 *
 * Threading (gpu.go:148,831): a model handle is used by one thread at a
 * time.  Several handles, one per device, may run concurrently from
 * separate threads; that is the multi-GPU mode (independent sequences).
 */
#ifndef LLM_B200_H
#define LLM_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define LLMB_API __attribute__((visibility("default")))
#else
#define LLMB_API
#endif

/* Status codes.  The reference returns Go error values; the classes below
 * follow its error sites. */
enum {
    LLMB_OK = 0,
    LLMB_ERR_ARG = 1,     /* a bad argument (empty prompt gpu.go:855, token id out of range) */
    LLMB_ERR_IO = 2,      /* reading the model file (gpu.go:365-367) */
    LLMB_ERR_FORMAT = 3,  /* GGUF header: gguf.ErrMagic, ErrVersion, ErrFormat (gguf/gguf.go:29-34) */
    LLMB_ERR_BOUND = 4,   /* GGUF header: gguf.ErrBound (gguf/gguf.go:32) */
    LLMB_ERR_CONFIG = 5,  /* ConfigFrom refusals (config.go:32-70) */
    LLMB_ERR_TENSOR = 6,  /* a missing tensor or a type without a kernel (gpu.go:300,326) */
    LLMB_ERR_MEMORY = 7,  /* the memory budget or a device allocation (gpu.go:175-177) */
    LLMB_ERR_CONTEXT = 8, /* prompt and new tokens exceed the context (gpu.go:948-950, 905-907) */
    LLMB_ERR_CUDA = 9,    /* a CUDA runtime error */
    LLMB_ERR_DEVICE = 10  /* a kernel reported an error (a bounded wait that gave up) */
};

typedef struct llmb_model llmb_model;

/* Config, config.go:11-23. */
typedef struct {
    int32_t layers, embd, ff, heads, kv_heads, head_dim, vocab, ctx;
    float rope_base, eps;
    int32_t rope_neox, bias, tied_output;
    char arch[16];
} llmb_config;

/* Stats, gpu.go:55-60.  A submit is one host->device launch group (one
 * CUDA graph launch or one prefill chunk); a dispatch is one kernel. */
typedef struct {
    int64_t submits, dispatches, tokens;
} llmb_stats;

/* Timing, gpu.go:929-939, plus device time from CUDA events on the model's
 * stream.  prefill_ms runs until the first sampled token is on the host;
 * decode_ms is the rest of the call.  gpu_decode_ms spans the first decode
 * launch to the end of the last; decode_kernel_ms sums the decode launches
 * alone (decode_launches of them). */
typedef struct {
    double prefill_ms, decode_ms;         /* wall clock, as time.Since in Generate */
    int32_t prompt_tokens, generated;
    int64_t submits, dispatches;
    double record_ms, submit_ms;          /* host time launching / waiting in decode */
    double gpu_prefill_ms, gpu_decode_ms; /* device time between CUDA events */
    double decode_kernel_ms;
    int64_t decode_launches;
} llmb_timing;

/* A reader of the model file: fill buf with len bytes at offset, return 0
 * on success.  Lets a Go host pass its io.ReaderAt (gpu.go:290,365). */
typedef int (*llmb_read_fn)(void *user, uint64_t offset, void *buf, uint64_t len);

/* Called with each generated token in order; return nonzero to go on, 0 to
 * stop (the emit callback of Generate, gpu.go:946,979). */
typedef int (*llmb_emit_fn)(void *user, int32_t token);

/* NewGPU, gpu.go:465-764.  Parses the GGUF header (gguf.Parse,
 * gguf/gguf.go:292), checks the configuration (ConfigFrom, config.go:29),
 * allocates every device buffer, builds the RoPE table in double precision
 * (gpu.go:524-541) and streams the weights through pinned host buffers into
 * their device layout.  ctx <= 0 or above the model's context_length means
 * context_length (gpu.go:470-472).  device is the CUDA ordinal. */
LLMB_API int llmb_open(const char *gguf_path, int ctx, int device, llmb_model **out);

/* NewGPU over a reader callback instead of a path; size is the file size. */
LLMB_API int llmb_open_reader(llmb_read_fn read, void *user, uint64_t size, int ctx, int device, llmb_model **out);

/* Releases every device and host resource of the model. */
LLMB_API void llmb_close(llmb_model *m);

/* The message of the last failure on this model; with m == NULL, the last
 * failure on the calling thread of a call that takes no model (llmb_open,
 * llmb_open_reader, llmb_kv8_*, llmb_logits_control).  Never NULL. */
LLMB_API const char *llmb_last_error(const llmb_model *m);

/* GPU.Cfg, gpu.go:119. */
LLMB_API int llmb_get_config(const llmb_model *m, llmb_config *out);

/* GPU.MemoryUsed, gpu.go:766-767: device bytes the model, its cache and its
 * scratch hold. */
LLMB_API uint64_t llmb_memory_used(const llmb_model *m);

/* GPU.Stats, gpu.go:138. */
LLMB_API int llmb_get_stats(const llmb_model *m, llmb_stats *out);

/* Generate, gpu.go:941-1014: greedy decoding.  The prompt goes through the
 * layers in chunks of up to PrefillBatch tokens, then tokens are decoded in
 * launches of DecodeBatch tokens, each sampled on the GPU (first index of the
 * largest logit) from the one before; only the sampled ids come back.
 * Stops after n tokens, at eos (not emitted) or when emit returns 0.  The
 * next launch is queued before the tokens of the one before are read back,
 * so up to 2*DecodeBatch-1 tokens may have been computed past the stop
 * (DecodeBatch-1 in the reference, gpu.go:1048-1051).  Each call starts at
 * position 0.  emit may be NULL.
 * out_tokens (may be NULL) receives the emitted tokens, n_out their count
 * (may be NULL), tm the timing (may be NULL). */
LLMB_API int llmb_generate(llmb_model *m, const int32_t *prompt, int n_prompt, int n, int32_t eos, llmb_emit_fn emit,
                  void *user, int32_t *out_tokens, int *n_out, llmb_timing *tm);

/* Multi-stream generation: n_seq independent greedy sequences on one model
 * (the reference runs one sequence per GPU object; this is the
 * llmb_generate_batch of its multi-stream workload).  Sequence s has the
 * prompt_lens[s] tokens that follow the earlier sequences' in prompts, its
 * own KV cache (the model keeps an arena of n_seq caches), and Generate's
 * semantics (gpu.go:946-1014): at most n tokens, eos stops it and is not
 * emitted.  Each call starts every sequence at position 0.  Prompt tokens
 * of all sequences go through the layers packed PrefillBatch-style in
 * batches of 64; then each step decodes one token of every unfinished
 * sequence, 64 per launch set.  out_tokens receives n_seq rows of n tokens
 * (row s at s * n), n_out (may be NULL) the count of each row, tm (may be
 * NULL) the summed timing. */
LLMB_API int llmb_generate_batch(llmb_model *m, const int32_t *prompts, const int *prompt_lens, int n_seq, int n,
                                 int32_t eos, int32_t *out_tokens, int *n_out, llmb_timing *tm);

/* PrefillLogits, gpu.go:902-927: runs the prompt and copies the vocab
 * logits of its last token into logits (a test hook: Generate never reads
 * logits back). */
LLMB_API int llmb_prefill_logits(llmb_model *m, const int32_t *prompt, int n_prompt, float *logits);

/* A test hook with no single counterpart in the reference: the greedy run
 * of Generate (prompt, then n tokens) that also copies the logits which
 * chose each token into step_logits (n rows of vocab floats), so that a
 * test checks every step against the CPU path, as examples/generate check
 * (main.go:141-181) does for step 1.  Decodes one token per launch. */
LLMB_API int llmb_generate_logits(llmb_model *m, const int32_t *prompt, int n_prompt, int n, int32_t *out_tokens,
                         float *step_logits);

/* Peek, gpu.go:1016-1043: the first n 32-bit words of a named device buffer,
 * as floats.  Names: "x" (residual stream), "q", "att", "gate" (the SwiGLU
 * output), "logits", "state" ({position, step} as raw bits), "tokens",
 * "kvblk.N." (layer N's cache: K then V) and, with the decode_trace knob,
 * "trace" (64-bit globaltimer stamps, see the knob). */
LLMB_API int llmb_peek(llmb_model *m, const char *name, float *out, int n);

/* GPU.Layers, gpu.go:143-146: run only that many layers (debugging: no
 * logits and no sampling are then produced).  0 restores all layers. */
LLMB_API int llmb_set_layers(llmb_model *m, int layers);

/* The package knobs of the reference: "decode_batch" (DecodeBatch,
 * gpu.go:1052, clamped to 1..16 as gpu.go:1046,1054), "prefill_batch"
 * (PrefillBatch, gpu.go:165; read by llmb_open, 1..64) and "memory_budget"
 * (Limits.MemoryBudget, gpu.go:35; bytes, 0 = the device's free memory;
 * read by llmb_open).  One more, with no counterpart in the reference:
 * "decode_mode" 0 (default) decodes with the persistent kernel, 1 with one
 * kernel per phase (an A/B and debugging aid); "prefill_mode" 0 (default)
 * runs prompt chunks and multi-stream batches through the chunked products
 * on the tensor cores (tcgen05, operands split exactly into bf16 pieces,
 * f32 accumulation), 1 through one matvec per token and phase, 2 through
 * chunked products on the FP32 CUDA cores (both A/B aids); "tag_reset" N > 0
 * clears the persistent kernel's tagged exchange buffers after every N
 * decoded tokens (a test aid: they are cleared anyway before the 32-bit tags
 * would wrap); "attn_positions" N (64..256, a multiple of 32; read by
 * llmb_open) sets the positions one attention item of the persistent kernel
 * covers, 0 (default) as many as its shared memory holds (an A/B and test
 * aid: longer contexts are split into items whose partials are merged);
 * "decode_trace" 1 makes models
 * opened afterwards record the persistent kernel's phase timeline, read with
 * llmb_peek(m, "trace", ...) (a profiling aid, the counterpart of GPU.Skip,
 * gpu.go:769-784); "wait_limit_us" N (0 = the default of 2 s) limits
 * every wait of the persistent kernel (a flag poll, a weight slot) to N
 * microseconds, past which the launch stops with LLMB_ERR_DEVICE; and
 * "drop_publish" S >= 0 (-1 = off) makes the persistent kernel skip one
 * publish at decode step S (the step counts prompt tokens too), so that the
 * next phase's wait runs out (a test aid for that error path, with
 * wait_limit_us).  Process-wide, like the Go package variables. */
LLMB_API int llmb_set_knob(const char *name, int64_t value);
LLMB_API int64_t llmb_get_knob(const char *name);

/* Decode attention that allocates no device memory.  It has no counterpart
 * in the reference; it exists for callers that cannot call cudaMalloc: a
 * host whose device memory is a fixed grant made by someone else (the
 * reference runs as a WebAssembly guest whose GPU memory its host grants up
 * front), or code that runs where allocation is not allowed.  Such a caller
 * passes device pointers it already owns:
 *   q        [heads * head_dim]               the query of one position
 *   k_cache  [n_pos rows of kv_stride floats] K, head g at g * head_dim
 *   v_cache  [n_pos rows of kv_stride floats] V, same layout
 *   out      [heads * head_dim]               softmax(q k / sqrt(head_dim)) v
 * (the attention of cpu.go:304-335; query head h reads kv head
 * h / (heads / kv_heads)).  The scratch, split-KV partials, is one
 * fixed array in device memory (about 1 MiB, held by every GPU that loads
 * this library until the process exits), so the sizes are limited: at most
 * 32 heads, head_dim 128 and 4096 positions; larger ones return LLMB_ERR_ARG
 * before any work.  Each call made outside stream capture looks up the
 * array's address on the current device (a host-side query that allocates
 * nothing), so the address always belongs to the current context; a call made
 * while `stream` is capturing a graph reuses the address its device's last
 * call outside capture found, so the first call on a device must come before
 * any capture.  An error already pending on the calling thread
 * (cudaPeekAtLastError) makes the call return LLMB_ERR_CUDA without
 * launching and without clearing it.  Every call shares the array: calls
 * that overlap on the GPU race, so serialise them (one stream).  No part of
 * the array needs clearing between calls: a call reads only what it wrote.
 * Asynchronous on `stream` (a cudaStream_t, NULL for the default stream); the
 * caller synchronises. */
LLMB_API int llmb_attention_noalloc(const float *q, const float *k_cache, const float *v_cache, int n_pos, int heads,
                                    int kv_heads, int head_dim, int kv_stride, float *out, void *stream);

/* ---- A key/value cache held in 8 bits -------------------------------------
 *
 * No counterpart in the reference, whose cache is float32 (gpu.go:509).  Like
 * llmb_attention_noalloc these calls work on device buffers the caller owns,
 * allocate nothing, are asynchronous on `stream` (a cudaStream_t of the
 * current device, NULL for the default stream) and may be captured into a
 * CUDA graph.  Arguments are checked before any work: NULL or misaligned
 * pointers, memory of another device, bad sizes are LLMB_ERR_ARG, with a
 * message from llmb_last_error(NULL); an error pending on the calling thread
 * is LLMB_ERR_CUDA and stays pending.  What only the GPU knows (lengths,
 * block numbers, row starts) is checked there: nothing outside the buffers
 * described here is read or written, whatever these hold.
 *
 * The cache is a pool of blocks.  A block holds `block` consecutive positions
 * of one sequence, for every kv head a tile [block][head_dim] of 8-bit
 * values, and one float scale for each head: element = value * scale.  Keys
 * and values are two pools of the same layout; both may lie in one
 * allocation (block_stride).  A sequence's blocks are listed in its row of a
 * table, so sequences grow block by block and may share the full blocks of a
 * common prefix. */
enum { LLMB_F32 = 0, LLMB_F16 = 1, LLMB_BF16 = 2 };   /* types of rows and logits */
enum { LLMB_KV8_INT8 = 0, LLMB_KV8_E4M3 = 1 };        /* types of the cache */

typedef struct {
    void *k, *v;             /* block b at b * block_stride bytes: [kv_heads][block][head_dim]; 16-byte aligned */
    float *k_scale, *v_scale;/* [n_blocks][kv_heads] */
    int64_t block_stride;    /* bytes; a multiple of 16, at least kv_heads * block * head_dim */
    int32_t n_blocks;
    int32_t block;           /* positions per block: 16, 32, 64 or 128 */
    int32_t kv_heads;
    int32_t head_dim;        /* 64 or 128 */
    int32_t type;            /* LLMB_KV8_INT8 or LLMB_KV8_E4M3 */
} llmb_kv8_cache;

/* The sequences of one call.  Sequence s has `lens[s]` positions once the
 * rows of this call are in, and the rows starts[s] .. starts[s+1]-1 (of q, k,
 * v and out) are its last positions, in order.  A sequence may have no rows
 * and no positions. */
typedef struct {
    const int32_t *lens;     /* device, [n_seq] */
    const int32_t *tables;   /* device, [n_seq] rows of table_stride block numbers */
    const int32_t *starts;   /* device, [n_seq + 1], not decreasing; NULL: n_rows / n_seq rows each */
    int32_t n_seq;           /* 1 .. 65535 */
    int32_t table_stride;    /* entries of a table row */
    int32_t n_rows;          /* rows of the call's buffers */
    int32_t max_new;         /* no sequence has more rows than this; 0: not known (n_rows) */
    int32_t max_len;         /* no sequence has more positions; 0: not known (table_stride * block).  The attention cuts
                              * its work by this bound, so a close one is faster */
} llmb_kv8_batch;

/* Writes the rows of k and v (n_rows rows of [kv_heads][head_dim] elements
 * of `type`, row_stride elements apart, 16-byte aligned) into the cache.  Per
 * block and head, with M = 127 (int8) or 448 (e4m3): a block's first rows
 * give it the scale a * (1 / M), a their largest magnitude.  Rows that come
 * later and do not fit grow the scale by the smallest power of two that fits,
 * and the values already there are rounded to the new step: all the roundings
 * of a value together stay within one step, however the rows came.  (a fits
 * where a <= (M + 2^-12) scale, so that it fits the scale made for it, however
 * that was rounded.  A scale that would grow more than 2^20-fold starts anew
 * at a * (1 / M); the earlier values are 0 then.)  Values round to nearest
 * even.  An infinity is stored as M steps and a NaN as 0, neither counts for
 * a.  Where a is below 2^-100 the scale stays as it is: rows of a block
 * without one are stored as 0, others are rounded to its step (and saturate at
 * M steps).  A sequence's blocks that receive rows must belong to it alone;
 * blocks outside the table's range or the pool are skipped. */
LLMB_API int llmb_kv8_append(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, const void *k, const void *v,
                             int type, int64_t row_stride, void *stream);

/* The reverse: the values held at the positions of each sequence's rows,
 * value * scale rounded once to `type`, into k and v (either may be NULL).
 * With lens and row counts of the caller's choice this reads any end of a
 * sequence, e.g. all of it for llmb_attention_noalloc, whose cache rows these
 * are.  Rows whose block is not in the pool are set to 0; rows of no sequence
 * stay as they were. */
LLMB_API int llmb_kv8_read(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, void *k, void *v, int type,
                           int64_t row_stride, void *stream);

/* Attention of the rows' queries over the cache, after the rows' own keys and
 * values were appended: out = softmax(scale q k) v over the positions up to
 * and including the row's own (and, with window > 0, among the last `window`
 * of those); query head h reads kv head h / (heads / kv_heads).  One row of a
 * sequence is a decoding step, more are a chunk of its prompt.  q and out:
 * n_rows rows of [heads][head_dim] elements of `type`, q_stride and
 * out_stride elements apart, 16-byte aligned; out must not overlap q unless
 * it is the same buffer with the same stride.  scale 0 means
 * 1 / sqrt(head_dim), negative ones are refused.  A row that sees no position
 * becomes 0, another whose query is not finite NaN; rows of no sequence stay
 * as they were.  Positions whose block is not in the pool are not seen.
 * Blocks' scales are finite and not negative; positions of a block whose
 * v_scale is 0 count in the softmax and add nothing to the result (a scale
 * below 2^-109, which append does not make, may be taken as 0).  A byte that
 * is a NaN of e4m3 (append writes none) is no value of the cache.  (A wait
 * inside the kernel that runs out after 1 s, which only a fault of the GPU can
 * cause, makes the rows NaN.)
 * Precision: 8-bit values enter the products exactly.  float32 queries have
 * 22 bits of their row's largest element, the weights of float32 and float16
 * rows 22 bits, those of bfloat16 rows 11 (off by 2^-12, a sixteenth of the
 * result's own rounding); sums are float32.
 * `workspace`: llmb_kv8_attention_workspace bytes of the caller's, 16-byte
 * aligned, not read before it is written; calls that may overlap on the GPU
 * need their own.  heads / kv_heads at most 64. */
LLMB_API int llmb_kv8_attention(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, const void *q,
                                int64_t q_stride, void *out, int64_t out_stride, int type, int heads, float scale,
                                int window, void *workspace, int64_t workspace_bytes, void *stream);

/* The bytes of workspace that llmb_kv8_attention needs for these sizes with
 * any type, scale and window (no pointer is looked at), or -1 where they are
 * not valid. */
LLMB_API int64_t llmb_kv8_attention_workspace(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, int heads);

/* ---- Logits between a model's head and the next token ---------------------
 *
 * No counterpart in the reference, which takes the largest logit as it is
 * (kernels_fused.go:271).  Device buffers of the caller's, any of the
 * controls NULL where it is not used; checks, stream and errors as for the
 * 8-bit cache. */
typedef struct {
    const int32_t *history;      /* [rows] rows of history_stride token ids: the prompt, then the answer so far */
    const int32_t *history_lens; /* [rows]; NULL: history_stride each */
    const int32_t *prompt_lens;  /* [rows] how many of them are the prompt; NULL: none */
    int32_t history_stride;      /* at most 524287 */
    int32_t n_bias;
    const float *penalties;      /* [rows][3]: repetition, presence, frequency; NULL: 1, 0, 0 */
    const int32_t *bias_ids;     /* [n_bias] token ids; of a token's biases the last counts */
    const float *bias_values;    /* [n_bias] */
    const int32_t *bias_starts;  /* [rows + 1], not decreasing: row r has the biases starts[r] .. starts[r+1]-1, at
                                  * most 4095 (later ones do not count); NULL: each row has all n_bias <= 4095 */
    const uint32_t *mask;        /* [rows] rows of mask_stride words: token v is allowed where bit v % 32 of word v / 32 is 1 */
    int32_t mask_stride;         /* at least (vocab + 31) / 32 */
} llmb_logits_ctl;

/* For each row of logits (rows rows of vocab elements of `type`, stride
 * elements apart) and each token: a token of the history has its logit
 * divided by `repetition` where it is above 0 and multiplied by it elsewhere;
 * one that the answer has c > 0 times loses presence and frequency * c; then
 * its bias is added, and it becomes -inf where the mask does not allow it.
 * In float32, each operation rounded once.  out (may be logits itself with
 * the same stride, or NULL) receives the result rounded to `type`; tokens
 * (may be NULL) per row the first index of the largest float32 result, or -1
 * where none is above -inf (a NaN is never taken).  Token ids outside the
 * vocabulary are passed over. */
LLMB_API int llmb_logits_control(const void *logits, int64_t stride, int type, int rows, int vocab,
                                 const llmb_logits_ctl *ctl, void *out, int64_t out_stride, int32_t *tokens,
                                 void *stream);

/* Called before each token is chosen, with the n tokens generated so far:
 * sets the bit of every token that may come next in mask ((vocab + 31) / 32
 * words; their contents are undefined before) and returns nonzero, or returns
 * 0 to stop. */
typedef int (*llmb_mask_fn)(void *user, const int32_t *tokens, int n, uint32_t *mask);

/* The controls of llmb_generate_controlled, in host memory. */
typedef struct {
    float repetition, presence, frequency; /* as llmb_logits_ctl's penalties (1, 0, 0: none); repetition above 0 */
    int32_t n_bias;                        /* at most 4095 */
    const int32_t *bias_ids;               /* in the vocabulary; of a token's biases the last counts */
    const float *bias_values;              /* -INFINITY forbids a token */
    llmb_mask_fn mask;                     /* NULL: every token is allowed */
    void *mask_user;
} llmb_controls;

/* llmb_generate with llmb_logits_control between the model's logits and each
 * token (the prompt and the answer so far are the history).  Stops as
 * Generate does, and where no token is allowed.  With penalties the prompt and
 * n are at most 524288 tokens together.  One token per launch, each read back
 * before the next. */
LLMB_API int llmb_generate_controlled(llmb_model *m, const int32_t *prompt, int n_prompt, int n, int32_t eos,
                                      const llmb_controls *controls, llmb_emit_fn emit, void *user,
                                      int32_t *out_tokens, int *n_out, llmb_timing *tm);

#ifdef __cplusplus
}
#endif

#endif /* LLM_B200_H */
