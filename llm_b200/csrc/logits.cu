// The control of logits between a model's head and its next token:
// llmb_logits_control (penalties for repeated tokens, biases, a grammar's
// mask, and the largest logit that is left).
//
// Per row and token id v, with c the times v is among the answer's tokens and
// any = v is anywhere in the history, in float32 with one rounding per
// operation:
//   any:    x = x > 0 ? x / repetition : x * repetition
//   c > 0:  x = (x - presence) - frequency c
//           x = x + bias(v)
//   mask:   x = -inf where v's bit is 0
//
// One pass over the vocabulary: the CTAs of a cluster share a row and hold a
// slice of it in registers.  While those loads are under way each CTA counts
// the history's tokens of its slice in a table in shared memory, a 32-bit
// word per token id: the count in bits 13..31, bit 12 for the prompt's tokens,
// in bits 0..11 the place of the token's bias (1..4095).  Counts are integers
// and of a token's biases the last counts, so the order of the atomics does
// not matter.  The cluster's first CTA takes the largest of the slices' maxima.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "kv8.hpp"
#include "ops.hpp"

namespace llmb {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 512;
constexpr int kMaxSlice = 11264;  // table words of a CTA: 44 KiB, so that four CTAs fit an SM
constexpr int kMaxBias = 4095, kMaxHistory = (1 << 19) - 1;

struct Ctl {
    const void *logits;
    void *out;
    int64_t stride, out_stride;
    int32_t *tokens;
    const int *history, *hist_lens, *prompt_lens;
    const float *penalties;
    const int *bias_ids, *bias_starts;
    const float *bias_values;
    const uint32_t *mask;
    int hist_stride, n_bias, mask_stride, vocab, slice, rounds;
};

// Orders like the values (-0 and 0 alike), a lower index above a higher one; 0 for NaN and -inf.
__device__ __forceinline__ uint64_t rank_of(float x, int v) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.f);
    const uint32_t key = u & 0x80000000u ? ~u : u | 0x80000000u;
    return (uint64_t)key << 32 | (uint32_t)~v;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) k_logits(const Ctl c) {
    constexpr int E = 16 / (int)sizeof(T), NV = (kMaxSlice / E + kThreads - 1) / kThreads;
    extern __shared__ uint32_t table[];
    __shared__ uint64_t best_w[kThreads / 32], best_c[16];
    cg::cluster_group cluster = cg::this_cluster();
    if (c.tokens) cluster_arrive();  // waited for before the first access to another CTA's shared memory
    const int nc = gridDim.x, rank = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const T *in = static_cast<const T *>(c.logits) + (int64_t)row * c.stride;
    T *out = c.out ? static_cast<T *>(c.out) + (int64_t)row * c.out_stride : nullptr;
    const uint32_t *mask = c.mask ? c.mask + (int64_t)row * c.mask_stride : nullptr;
    const int *hist = c.history ? c.history + (int64_t)row * c.hist_stride : nullptr;
    const int nh = hist ? min(max(c.hist_lens ? __ldg(c.hist_lens + row) : c.hist_stride, 0), c.hist_stride) : 0;
    const int np = c.prompt_lens ? __ldg(c.prompt_lens + row) : 0;
    float rep = 1.f, pres = 0.f, freq = 0.f;
    if (c.penalties)
        rep = __ldg(c.penalties + 3 * row), pres = __ldg(c.penalties + 3 * row + 1), freq = __ldg(c.penalties + 3 * row + 2);
    int bias0 = 0, bias1 = c.n_bias;
    if (c.bias_starts) {
        bias0 = min(max(__ldg(c.bias_starts + row), 0), c.n_bias);
        bias1 = min(min(max(__ldg(c.bias_starts + row + 1), bias0), c.n_bias), bias0 + kMaxBias);
    }
    uint64_t best = 0;
    for (int round = 0; round < c.rounds; ++round) {
        const int64_t first = (int64_t)(round * nc + rank) * c.slice;
        if (first >= c.vocab) break;
        const int v0 = (int)first, n = min(c.slice, c.vocab - v0);
        // the slice's logits, all on their way before the table is made
        uint4 raw[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = (tid + i * kThreads) * E;
            if (u >= n) continue;
            if (VEC && u + E <= n) {
                raw[i] = *reinterpret_cast<const uint4 *>(in + v0 + u);
            } else {
                T e[E];
#pragma unroll
                for (int k = 0; k < E; ++k) e[k] = u + k < n ? in[v0 + u + k] : kv8_from<T>(0.f);
                raw[i] = *reinterpret_cast<const uint4 *>(e);
            }
        }
        if (round > 0) __syncthreads();
        for (int i = tid; i < n; i += kThreads) table[i] = 0;
        __syncthreads();
        if (bias1 > bias0) {
            for (int i = bias0 + tid; i < bias1; i += kThreads) {
                const uint32_t off = (uint32_t)(__ldg(c.bias_ids + i) - v0);
                if (off < (uint32_t)n) atomicMax(table + off, (uint32_t)(i - bias0 + 1));
            }
            __syncthreads();
        }
        for (int i = tid; i < nh; i += kThreads) {
            const uint32_t off = (uint32_t)(__ldg(hist + i) - v0);
            if (off < (uint32_t)n) {
                if (i < np) atomicOr(table + off, 1u << 12);
                else atomicAdd(table + off, 1u << 13);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int u = (tid + i * kThreads) * E;
            if (u >= n) continue;
            const T *e = reinterpret_cast<const T *>(&raw[i]);
            T res[E];
            // E divides 32 and v0 + u is a multiple of E: one mask word
            const uint32_t bits = mask ? __ldg(mask + (v0 + u) / 32) >> ((v0 + u) % 32) : 0xffffffffu;
#pragma unroll
            for (int k = 0; k < E; ++k) {
                float x = kv8_float<T>(e[k]);
                const uint32_t w = u + k < n ? table[u + k] : 0;
                if (w >> 12) {
                    x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                    if (w >> 13) x = __fsub_rn(__fsub_rn(x, pres), __fmul_rn(freq, (float)(w >> 13)));
                }
                if (w & 0xfffu) x = __fadd_rn(x, __ldg(c.bias_values + bias0 + (w & 0xfffu) - 1));
                if (!(bits >> k & 1)) x = -INFINITY;
                res[k] = kv8_from<T>(x);
                if (u + k < n) {
                    const uint64_t r = rank_of(x, v0 + u + k);
                    best = r > best ? r : best;
                }
            }
            if (out) {
                if (VEC && u + E <= n) {
                    *reinterpret_cast<uint4 *>(out + v0 + u) = *reinterpret_cast<const uint4 *>(res);
                } else {
#pragma unroll
                    for (int k = 0; k < E; ++k)
                        if (u + k < n) out[v0 + u + k] = res[k];
                }
            }
        }
    }
    if (!c.tokens) return;
    for (int o = 16; o; o >>= 1) {
        const uint64_t r = __shfl_xor_sync(kFull, best, o);
        best = r > best ? r : best;
    }
    if ((tid & 31) == 0) best_w[tid >> 5] = best;
    cluster_wait();
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kThreads / 32; ++w) best = best_w[w] > best ? best_w[w] : best;
        *cluster.map_shared_rank(&best_c[rank], 0) = best;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (int w = 0; w < nc; ++w) best = best_c[w] > best ? best_c[w] : best;
        c.tokens[row] = best ? (int32_t)~(uint32_t)best : -1;
    }
}

// Clusters of 16 CTAs are above the portable size; each kernel is told so once per device.
template <class T, bool VEC>
cudaError_t allow_clusters(int device) noexcept {
    static std::atomic<bool> done[64];
    if (device < 64 && done[device].load(std::memory_order_relaxed)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(k_logits<T, VEC>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && device < 64) done[device].store(true, std::memory_order_relaxed);
    return e;
}

template <class T, bool VEC>
cudaError_t launch(const Ctl &c, int rows, int ctas, int device, cudaStream_t st) noexcept {
    const cudaError_t e = allow_clusters<T, VEC>(device);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas, attr.val.clusterDim.y = 1, attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(ctas, rows), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = (size_t)c.slice * 4;
    cfg.stream = st, cfg.attrs = &attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_logits<T, VEC>, c);
}

}  // namespace
}  // namespace llmb

using namespace llmb;

extern "C" int llmb_logits_control(const void *logits, int64_t stride, int type, int rows, int vocab,
                                   const llmb_logits_ctl *ctl, void *out, int64_t out_stride, int32_t *tokens,
                                   void *stream) {
    const char *what = "logits_control";
    if (!ctl) return op_error(LLMB_ERR_ARG, "llm: %s: no controls", what);
    if (type != LLMB_F32 && type != LLMB_F16 && type != LLMB_BF16)
        return op_error(LLMB_ERR_ARG, "llm: %s: no type %d", what, type);
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > 1 << 24 || stride < vocab || (out && out_stride < vocab))
        return op_error(LLMB_ERR_ARG, "llm: %s: %d rows of %d logits, %lld and %lld elements apart", what, rows, vocab,
                        (long long)stride, (long long)out_stride);
    if (!out && !tokens && rows > 0) return op_error(LLMB_ERR_ARG, "llm: %s: neither out nor tokens", what);
    if (ctl->history && (ctl->history_stride < 1 || ctl->history_stride > kMaxHistory))
        return op_error(LLMB_ERR_ARG, "llm: %s: histories of %d tokens (1 to %d)", what, ctl->history_stride, kMaxHistory);
    if (!ctl->history && (ctl->history_lens || ctl->prompt_lens))
        return op_error(LLMB_ERR_ARG, "llm: %s: lengths without a history", what);
    if (ctl->n_bias < 0 || (!ctl->bias_starts && ctl->n_bias > kMaxBias) || (!ctl->bias_ids != !ctl->bias_values) ||
        (!ctl->bias_ids && (ctl->n_bias > 0 || ctl->bias_starts)))
        return op_error(LLMB_ERR_ARG, "llm: %s: %d biases (at most %d a row, ids and values)", what, ctl->n_bias, kMaxBias);
    if (ctl->mask && ctl->mask_stride < (vocab + 31) / 32)
        return op_error(LLMB_ERR_ARG, "llm: %s: mask rows of %d words (at least %d)", what, ctl->mask_stride, (vocab + 31) / 32);
    const int es = type == LLMB_F32 ? 4 : 2;
    const std::initializer_list<OpPointer> ps = {
        {logits, "logits", es, rows == 0}, {out, "out", es, true}, {tokens, "tokens", 4, true},
        {ctl->history, "history", 4, true}, {ctl->history_lens, "history_lens", 4, true},
        {ctl->prompt_lens, "prompt_lens", 4, true}, {ctl->penalties, "penalties", 4, true},
        {ctl->bias_ids, "bias_ids", 4, true}, {ctl->bias_values, "bias_values", 4, true},
        {ctl->bias_starts, "bias_starts", 4, true}, {ctl->mask, "mask", 4, true}};
    int dev = 0, rc = op_alignment(what, ps);
    if (rc == LLMB_OK) rc = op_device(what, &dev);
    if (rc == LLMB_OK) rc = op_pointers(what, dev, ps);
    if (rc != LLMB_OK) return rc;
    if (rows == 0) return LLMB_OK;
    // one vector of a thread is the least that a CTA is worth launching for
    int ctas = 1;
    while (ctas < 16 && ctas * kThreads * 16 / es < vocab) ctas *= 2;
    Ctl c{};
    c.rounds = (int)((vocab + (int64_t)ctas * kMaxSlice - 1) / ((int64_t)ctas * kMaxSlice));
    c.slice = (vocab + ctas * c.rounds - 1) / (ctas * c.rounds);
    c.slice = (c.slice + 127) / 128 * 128;
    c.logits = logits, c.out = out, c.stride = stride, c.out_stride = out_stride, c.tokens = tokens;
    c.history = ctl->history, c.hist_lens = ctl->history_lens, c.prompt_lens = ctl->prompt_lens;
    c.hist_stride = ctl->history_stride, c.penalties = ctl->penalties;
    c.bias_ids = ctl->bias_ids, c.bias_values = ctl->bias_values, c.bias_starts = ctl->bias_starts;
    c.n_bias = ctl->n_bias, c.mask = ctl->mask, c.mask_stride = ctl->mask_stride, c.vocab = vocab;
    auto aligned = [es](const void *p, int64_t s) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s * es % 16 == 0; };
    const bool vec = aligned(logits, stride) && (!out || aligned(out, out_stride));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (type == LLMB_F32) e = vec ? launch<float, true>(c, rows, ctas, dev, st) : launch<float, false>(c, rows, ctas, dev, st);
    else if (type == LLMB_F16) e = vec ? launch<__half, true>(c, rows, ctas, dev, st) : launch<__half, false>(c, rows, ctas, dev, st);
    else e = vec ? launch<__nv_bfloat16, true>(c, rows, ctas, dev, st) : launch<__nv_bfloat16, false>(c, rows, ctas, dev, st);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return op_error(LLMB_ERR_CUDA, "llm: %s: %s", what, cudaGetErrorString(e));
    }
    return op_launched(what);
}
