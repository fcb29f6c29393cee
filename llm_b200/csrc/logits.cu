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
// One pass over the vocabulary: the CTAs of a cluster share a row; chunks of
// 32 tokens go round among them, so that the frequent tokens, which have low
// ids, do not all fall to one.  A CTA counts the history's tokens among its
// own in a table in shared memory, a 32-bit word per token: the count in bits
// 0..18, bit 19 for the prompt's tokens, in bits 20..31 the place of the
// token's bias (1..4095).  Counts are integers and of a token's biases the
// last counts, so the order of the atomics does not matter.  The pass looks a
// logit's word up and works out those that have one.
//
// Bound by instructions, and by latency at the start of a round, which has at
// most 11264 tokens of a CTA: what the round reads first (two vectors of logits
// a thread, and in the first round the history, biases and lengths) is asked
// for before the table is cleared, and there are two barriers in it and one
// between rounds.  64 rows of 151936 float32 logits with histories of up to
// 4096, in two rounds of 9504 tokens for each of 8 CTAs, so that the history is
// read and counted twice: 37 us, 2.2 TB/s, 33 % of the measured copy rate (22 us
// without a history; bfloat16 37 us too): 270 instructions for 128 logits, of
// which counting and the divisions of single lanes take 4 us each.  64 rows of
// 50256 take 19 us, of 50257, of which only every fourth is aligned to 16 bytes
// and all go element by element, 21 (bfloat16 20 and 31).  One row of 49152: 5.4
// us, latency.
//
// The cluster's first CTA takes the largest of the CTAs' maxima; the others do
// not wait for it.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "kv8.hpp"
#include "ops.hpp"
#include "ptx.hpp"

namespace llmb {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 384;
constexpr int kMaxSlice = 11264;  // tokens of a CTA and round: a table of 44 KiB
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

template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) k_logits(const Ctl c) {
    constexpr int E = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) uint32_t table[];  // c.slice words (a multiple of 32)
    __shared__ uint64_t best_w[kThreads / 32], best_c[16], bar;

    cg::cluster_group cluster = cg::this_cluster();
    const int nc = gridDim.x, rank = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int shift = 31 - __clz(nc);  // (a power of two)
    if (c.tokens) {  // the first CTA's barrier counts the others' maxima; they may come once the cluster has started
        if (tid == 0) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(&bar)), "r"(nc));
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    }
    const T *in = static_cast<const T *>(c.logits) + (int64_t)row * c.stride;
    T *out = c.out ? static_cast<T *>(c.out) + (int64_t)row * c.out_stride : nullptr;
    const uint32_t *mask = c.mask ? c.mask + (int64_t)row * c.mask_stride : nullptr;
    const int *hist = c.history ? c.history + (int64_t)row * c.hist_stride : nullptr;
    // the first ids of the thread, whether or not they will be wanted
    constexpr int G = 4;
    int ids[G], bias_id = -1;
#pragma unroll
    for (int k = 0; k < G; ++k) ids[k] = hist && tid + k * kThreads < c.hist_stride ? __ldg(hist + tid + k * kThreads) : -1;
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
    if (bias0 + tid < bias1) bias_id = __ldg(c.bias_ids + bias0 + tid);
    const bool controlled = nh > 0 || bias1 > bias0;
    float best_x = -INFINITY;
    int best_v = 0;
    for (int round = 0; round < c.rounds; ++round) {
        const int chunk0 = round * (c.slice / 32);  // this round's first chunk of the CTA's
        // the CTA's token u of the round, and back (-1: another's)
        auto token = [&](int u) { return (((chunk0 + (u >> 5)) << shift) + rank) * 32 + (u & 31); };
        auto place = [&](int v) {
            if (v < 0 || v >= c.vocab || ((v >> 5) & (nc - 1)) != rank) return -1;
            const int j = (v >> (5 + shift)) - chunk0;
            return j >= 0 && j < c.slice / 32 ? j * 32 + (v & 31) : -1;
        };
        auto load = [&](int u, uint4 &raw, uint32_t &bits) {
            const int v = token(u);
            // E divides 32 and u is a multiple of E: one word of the mask
            bits = mask && v < c.vocab ? __ldg(mask + (v >> 5)) >> (v & 31) : 0xffffffffu;
            if (VEC && v + E <= c.vocab) {
                raw = *reinterpret_cast<const uint4 *>(in + v);
            } else {
                T e[E];
#pragma unroll
                for (int k = 0; k < E; ++k) e[k] = v + k < c.vocab ? in[v + k] : kv8_from<T>(0.f);
                raw = *reinterpret_cast<const uint4 *>(e);
            }
        };
        constexpr int step = kThreads * E;
        // the first two vectors of the thread are on their way while the table is made
        uint4 r0, r1;
        uint32_t b0, b1;
        if (tid * E < c.slice) load(tid * E, r0, b0);
        if (tid * E + step < c.slice) load(tid * E + step, r1, b1);
        if (round > 0) __syncthreads();
        if (controlled) {
            for (int i = 4 * tid; i < c.slice; i += 4 * kThreads) *reinterpret_cast<uint4 *>(table + i) = make_uint4(0, 0, 0, 0);
            __syncthreads();
            auto bias = [&](int v, int i) {
                const int off = place(v);
                if (off < 0) return;
                const uint32_t n = (uint32_t)(i - bias0 + 1);
                for (uint32_t w = table[off], was; w >> 20 < n; w = was) {
                    was = atomicCAS(table + off, w, n << 20 | (w & 0xfffffu));
                    if (was == w) break;
                }
            };
            auto count = [&](int v, int i) {
                const int off = i < nh ? place(v) : -1;
                if (off < 0) return;
                if (i < np) atomicOr(table + off, 1u << 19);
                else atomicAdd(table + off, 1u);
            };
            if (bias0 + tid < bias1) bias(bias_id, bias0 + tid);
            for (int i = bias0 + tid + kThreads; i < bias1; i += kThreads) bias(__ldg(c.bias_ids + i), i);
#pragma unroll
            for (int k = 0; k < G; ++k) count(ids[k], tid + k * kThreads);
#pragma unroll 4
            for (int i = tid + G * kThreads; i < nh; i += kThreads) count(__ldg(hist + i), i);
            __syncthreads();
        }
        auto controls = [&](float y, uint32_t w) {
            if (w & 0xfffffu) {
                const uint32_t n = w & 0x7ffffu;
                y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                if (n) y = __fsub_rn(__fsub_rn(y, pres), __fmul_rn(freq, (float)n));
            }
            if (w >> 20) y = __fadd_rn(y, __ldg(c.bias_values + bias0 + (w >> 20) - 1));
            return y;
        };
        auto use = [&](int u, const uint4 &raw, uint32_t bits) {
            const T *e = reinterpret_cast<const T *>(&raw);
            const int v = token(u);
            if (v >= c.vocab) return;
            float x[E];
            if (v + E > c.vocab) bits &= (1u << (c.vocab - v)) - 1;
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] = kv8_float<T>(e[k]);
            if (controlled) {
#pragma unroll
                for (int k = 0; k < E; k += 4) {
                    const uint4 w4 = *reinterpret_cast<const uint4 *>(table + u + k);
                    if (w4.x) x[k] = controls(x[k], w4.x);
                    if (w4.y) x[k + 1] = controls(x[k + 1], w4.y);
                    if (w4.z) x[k + 2] = controls(x[k + 2], w4.z);
                    if (w4.w) x[k + 3] = controls(x[k + 3], w4.w);
                }
            }
            T res[E];
#pragma unroll
            for (int k = 0; k < E; ++k) {
                if (!(bits >> k & 1)) x[k] = -INFINITY;
                res[k] = kv8_from<T>(x[k]);
                if (x[k] > best_x) best_x = x[k], best_v = v + k;  // (the thread's tokens come in order)
            }
            if (out) {
                if (VEC && v + E <= c.vocab) {
                    *reinterpret_cast<uint4 *>(out + v) = *reinterpret_cast<const uint4 *>(res);
                } else {
#pragma unroll
                    for (int k = 0; k < E; ++k)
                        if (v + k < c.vocab) out[v + k] = res[k];
                }
            }
        };
        for (int u = tid * E; u < c.slice; u += 2 * step) {
            const uint4 now = r0;
            const uint32_t now_b = b0;
            if (u + 2 * step < c.slice) load(u + 2 * step, r0, b0);
            use(u, now, now_b);
            if (u + step >= c.slice) break;
            const uint4 next = r1;
            const uint32_t next_b = b1;
            if (u + 3 * step < c.slice) load(u + 3 * step, r1, b1);
            use(u + step, next, next_b);
        }
    }
    if (!c.tokens) return;
    uint64_t best = rank_of(best_x, best_v);
    for (int o = 16; o; o >>= 1) {
        const uint64_t r = __shfl_xor_sync(kFull, best, o);
        best = r > best ? r : best;
    }
    if (lane == 0) best_w[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
        best = tid < kThreads / 32 ? best_w[tid] : 0;
        for (int o = 16; o; o >>= 1) {
            const uint64_t r = __shfl_xor_sync(kFull, best, o);
            best = r > best ? r : best;
        }
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (tid != 0) return;
    *cluster.map_shared_rank(&best_c[rank], 0) = best;
    uint32_t first;  // the first CTA's barrier
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(first) : "r"(su32(&bar)));
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(first) : "memory");
    if (rank != 0) return;
    bool ok = false;
    for (int i = 0; i < 1 << 22 && !ok; ++i) {  // the others' work is a few microseconds; each try waits a while itself
        uint32_t p;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(p)
            : "r"(su32(&bar))
            : "memory");
        ok = p != 0;
    }
    for (int w = 0; w < nc; ++w) best = best_c[w] > best ? best_c[w] : best;
    c.tokens[row] = ok && best ? (int32_t)~(uint32_t)best : -1;
}

constexpr size_t slice_bytes(int slice) { return (size_t)slice * 4; }

// Clusters of 16 CTAs are above the portable size and the table above the default's; each kernel is told so once per device.
template <class T, bool VEC>
cudaError_t allow_clusters(int device) noexcept {
    static std::atomic<bool> done[64];
    if (device < 64 && done[device].load(std::memory_order_relaxed)) return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(k_logits<T, VEC>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k_logits<T, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)slice_bytes(kMaxSlice));
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
    cfg.gridDim = dim3(ctas, rows), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = slice_bytes(c.slice);
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
    if (out == logits && rows > 1 && out_stride != stride)
        return op_error(LLMB_ERR_ARG, "llm: %s: out is logits with another stride", what);
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
    // One vector of a thread is the least that a CTA is worth launching for.  Few rows take 16 CTAs each; with many, places
    // for 8 at once are free sooner (64 rows of 151936: 38 us, with 16: 45 us, although the history is then read twice).
    const int most = rows * 16 <= 2 * 148 ? 16 : 8;
    int ctas = 1;
    while (ctas < most && ctas * kThreads * 16 / es < vocab) ctas *= 2;
    Ctl c{};
    const int chunks = (vocab + 32 * ctas - 1) / (32 * ctas);  // of 32 tokens, for each CTA
    c.rounds = (chunks + kMaxSlice / 32 - 1) / (kMaxSlice / 32);
    c.slice = (chunks + c.rounds - 1) / c.rounds * 32;
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
