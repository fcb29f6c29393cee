// Attention of many rows over the 8-bit cache on the 5th-generation tensor
// cores (tcgen05): chunks of prompts (llmb_kv8_attention).
//
// A CTA owns two tiles A and B of 128 rows of one (sequence, kv head) (row r
// is query head r % group of token r / group) and one part of the positions,
// 128 at a time:
//
//   1 warp     looks up the blocks and copies the 8-bit K and V of 128
//              positions into shared memory (bulk copies of 16 positions,
//              a few steps ahead);
//   4 warps    store them as float16, which holds them exactly, in a ring of
//              slots (K, V, K, V, ...; rows of 64 elements with the 128-byte
//              swizzle, which is K's k-major layout and V's n-major one);
//   1 thread   issues S = Q K^T (A from shared memory) and O += P V (A from
//              tensor memory) for A and B in turn;
//   2 x 4 warps  own A's and B's rows, one a thread: read S from tensor
//              memory, take the softmax with a running maximum and write the
//              weights P over S as float16.
//
// While the softmax of one tile runs, the tensor cores work on the other.
// The accumulators are rescaled only when a weight would come out above 2^14,
// which is rare after the first positions (bfloat16 rows do not even look for
// a step's maximum otherwise).
//
// Three prompts of up to 1023 tokens behind 4000 positions (32 heads on 8, size
// 128, int8): bfloat16 rows 299 us, 635 TFLOP/s, 38 % of the measured bf16
// rate, float16 437, float32 707; 360 tiles are 2.4 waves.  The chain of one
// tile, softmax and then its two products, bounds a step, then shared memory's
// rate: 192 KB of operands, 64 KB of float16 stored and 64 KB of copies a step
// of two tiles.  Left out one at a time, when a step's maximum was still looked
// for in every step (332 us): the weights 222, the exponentials 289, the
// conversion 316.
//
// Precision is that of the kernel for few rows (kv8.cu): float32 queries and
// weights are two float16 pieces each, float16 queries one and their weights
// two, bfloat16 ones one and one; the scales of K's and V's blocks enter the
// scores and the weights.  The tensor cores' accumulators cut off what does
// not fit 24 bits, towards 0, at every 16 positions: a bias of about 1e-8 a
// step.  For float32 rows the products are therefore summed over 4 steps of
// 128 positions only and added to the result in float32; their space in
// tensor memory leaves room for one tile with head_dim 128.
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "kv8.hpp"
#include "kv8_chunk.hpp"
#include "ops.hpp"
#include "ptx.hpp"

namespace llmb {
namespace {

constexpr int kKeys = 128;                  // positions of a step
constexpr int kThreads = 16 * 32;           // warpgroups: A's softmax, B's softmax, the converters, the issuer and the copier
// Their registers a thread: as many together as the launch's 4 x 128.
constexpr int kRegSoft = 184, kRegCopy = 88, kRegIssue = 56;
static_assert(2 * kRegSoft + kRegCopy + kRegIssue <= 4 * 65536 / kThreads, "a split above the launch's registers waits forever");
constexpr uint64_t kWaitNs = 1000000000ull; // 1 s: the limit of a wait

template <class T> constexpr int kQPieces = 1;
template <> constexpr int kQPieces<float> = 2;
template <class T> constexpr int kPPieces = 2;
template <> constexpr int kPPieces<__nv_bfloat16> = 1;

// What 16 positions share: K's scale; V's scale = mv 2^lv, with 2^-lv in the unit of the weights' sums.  bfloat16 rows, whose
// precision leaves room for the rounding of a logarithm, have all of the scale in lv, and mv is not used; where a scale has
// no logarithm, or is below all that append makes, the group's values are 0 for them: zeros are stored in place of its copy.
struct Group {
    float ks, lv, mv, unlv;
};

template <class T> constexpr int kSumSteps = 0;  // steps between additions to the result; 0: the accumulator is the result
template <> constexpr int kSumSteps<float> = 4;

template <class T, int HD>
struct Layout {
    static constexpr int tiles = kv8_chunk_rows(sizeof(T) == 4, HD) / 128;
    static constexpr int slots = HD == 128 ? 3 : 4, copies = HD == 128 ? 4 : 8;  // ring slots; copies in flight
    static constexpr int panel = 128 * 128;                        // 128 rows of 64 float16
    static constexpr int slot = panel * (HD / 64);
    static constexpr int q_tile = panel * (HD / 64) * kQPieces<T>;
    static constexpr int ring = tiles * q_tile;
    static constexpr int raw = ring + slots * slot;                // [copies][128][HD] bytes
    static constexpr int group = raw + copies * 128 * HD;          // [8][8] Group
    static constexpr int fac = group + 8 * 8 * (int)sizeof(Group); // [256] float
    static constexpr int bars = fac + 256 * 4;
    static constexpr int total = bars + 384;
    // columns of tensor memory: S (and the weights) of each tile, the accumulators, and the results where they are apart
    static constexpr int tm_o = 128 * tiles, tm_r = kSumSteps<T> ? tm_o + HD * tiles : tm_o;
    static_assert(tm_r + HD * tiles <= 512, "tensor memory");
    static_assert(total <= 232448, "the shared memory exceeds the per-block maximum");
};

struct Bars {
    uint64_t full[4], empty[4], raw[8], free[8], group[8], s[2], p[2], q[2], o[2], done;
    uint32_t tmem, fail;
};
static_assert(sizeof(Bars) <= 384, "the barriers' space");

// Waits for a phase of a barrier, at most kWaitNs (counted from the first look at the clock, which is slow and so left
// until many tries were in vain); false after that, or once another wait has run out.
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, uint32_t *fail) {
    uint64_t t0 = 0;
    for (unsigned spins = 1; !bar_try(bar, parity); ++spins)
        if ((spins & 255) == 0) {
            if (*(volatile uint32_t *)fail) return false;
            const uint64_t t = gtime();
            if (t0 == 0) t0 = t;
            if (t - t0 > kWaitNs) {
                *(volatile uint32_t *)fail = 1;
                return false;
            }
        }
    return true;
}

__device__ __forceinline__ void bar_init(uint64_t *bar, int n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(n));
}
__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void commit(bool one, uint64_t *bar) {
    if (one)
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar)) : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle, version 1 (sm_100): 8 rows of 128 bytes are 1024 bytes apart
// from the next 8; lbo is the distance of an n-major operand's next 64 columns.
__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}

// Instruction descriptor: kind::f16, float16 A and B, float32 D, M = 128; bn: B is n-major.
__device__ __forceinline__ constexpr uint32_t idesc(int n, int bn) {
    return (1u << 4) | ((uint32_t)bn << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(bool one, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    if (one) asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
                 "l"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(bool one, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    if (one) asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(acc)
                 : "memory");
}

// 32 columns of the warp's 32 lanes; the values may be used after tm_wait on them.
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// (The values pass through, so that no use of them moves before the wait.)
__device__ __forceinline__ void tm_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
__device__ __forceinline__ void tm_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Bytes (a multiple of 16, both ends 16-byte aligned) to shared memory; their arrival is counted on the barrier.
__device__ __forceinline__ void bulk(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(su32(dst)),
                 "l"(src), "r"(bytes), "r"(su32(bar))
                 : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}

// The queries of tile w's 32 rows of this warp into shared memory, a row by 8 lanes.
template <class T, int HD>
__device__ __forceinline__ void load_queries(const Kv8Att &a, const Kv8Seq &sq, int head, int row0, int rows, int warp,
                                             int lane, uint8_t *q_smem, float *fac, float unit) {
    constexpr int PN = HD / 64, QP = kQPieces<T>, V4 = (int)sizeof(T) / 2, B = sizeof(T) == 4 && HD == 128 ? 4 : 8;
    const int sub = lane & 7;
    // row warp * 32 + lane / 8 and every fourth after it: token and head in its group, without more divisions
    int tok = (row0 + warp * 32 + (lane >> 3)) / a.group, in = row0 + warp * 32 + (lane >> 3) - tok * a.group;
    const int tok4 = 4 / a.group, in4 = 4 - tok4 * a.group;
    for (int it0 = 0; it0 < 8; it0 += B) {  // B rows' loads in flight
        uint4 raw[B][PN][V4];
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int r = row0 + warp * 32 + (it0 + i) * 4 + (lane >> 3);
            const T *src = static_cast<const T *>(a.q) + (int64_t)(sq.start + tok) * a.q_stride + (head * a.group + in) * HD + 8 * sub;
            tok += tok4, in += in4;
            if (in >= a.group) in -= a.group, ++tok;
#pragma unroll
            for (int p = 0; p < PN; ++p)
#pragma unroll
                for (int v = 0; v < V4; ++v)
                    raw[i][p][v] = r < rows ? *(reinterpret_cast<const uint4 *>(src + 64 * p) + v) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < B; ++i) {
            const int row = warp * 32 + (it0 + i) * 4 + (lane >> 3);
            float x[PN][8];
            uint32_t m = 0;  // the largest magnitude's bits, which order like it; infinity and NaN are above the finite ones
#pragma unroll
            for (int p = 0; p < PN; ++p) {
                const T *v = reinterpret_cast<const T *>(raw[i][p]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[p][e] = kv8_float<T>(v[e]);
                    m = max(m, __float_as_uint(x[p][e]) & 0x7fffffffu);
                }
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(kFull, m, o));
            float up, down;
            const bool fine = kv8_query_scale(m, up, down);
            if (sub == 0) fac[row] = fine ? a.scale * unit * down : NAN;
#pragma unroll
            for (int p = 0; p < PN; ++p) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float y0 = fine ? x[p][2 * e] * up : 0.f, y1 = fine ? x[p][2 * e + 1] * up : 0.f;
                    hi[e] = pack_half2(y0, y1);
                    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&hi[e]));
                    lo[e] = pack_half2(y0 - f.x, y1 - f.y);
                }
                uint8_t *dst = q_smem + p * Layout<T, HD>::panel + row * 128 + ((sub ^ (row & 7)) << 4);
                *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (QP == 2) *reinterpret_cast<uint4 *>(dst + PN * Layout<T, HD>::panel) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
}

// A row's largest score (in log2, with the exponent of V's scale) among positions [b0, b1) of a step; WHOLE: all 128.
template <bool WHOLE>
__device__ __forceinline__ float row_top(const uint32_t (&x)[4][32], const Group *gp, float fac, int b0, int b1) {
    float top = -FLT_MAX;
#pragma unroll
    for (int g = 0; g < 8; ++g) {
        const float ks = gp[g].ks, lv = gp[g].lv;
        float v = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int i = 16 * g + e;
            v = fmaxf(v, WHOLE || (i >= b0 && i < b1) ? __uint_as_float(x[i / 32][i % 32]) : -INFINITY);
        }
        // (no position of the group seen, and a factor 0: -inf * 0)
        if (WHOLE || v > -INFINITY) top = fmaxf(top, fmaf(v, fac * ks, lv));
    }
    return top;
}

// A row's weights 2^(score + shift) into tensor memory over its scores; returns their sum without V's scales. big becomes
// the largest sum of 16 of them: none of them is larger (NaN stays NaN).
template <int PP, bool WHOLE>
__device__ __forceinline__ float row_weights(const uint32_t (&x)[4][32], uint32_t sm, const Group *gp, float fac, float shift,
                                             int b0, int b1, float &big) {
    float l = 0.f;
    big = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        uint32_t ph[16], pl[16];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const Group gr = gp[2 * k + g];
            const float gf = fac * gr.ks, gd = gr.lv + shift;
            const uint64_t f2 = pack2(gf, gf), d2 = pack2(gd, gd);
            uint64_t sum2 = 0;
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const int i = 32 * k + 16 * g + e;
                const float2 z = unpack2(fma2(pack2(__uint_as_float(x[k][16 * g + e]), __uint_as_float(x[k][16 * g + e + 1])), f2, d2));
                float y0 = kv8_exp2(z.x), y1 = kv8_exp2(z.y);
                if (!WHOLE) {
                    if (!(i >= b0 && i < b1)) y0 = 0.f;
                    if (!(i + 1 >= b0 && i + 1 < b1)) y1 = 0.f;
                }
                sum2 = add2(sum2, pack2(y0, y1));
                if (PP == 2) y0 *= gr.mv, y1 *= gr.mv;
                const uint32_t p = pack_half2(y0, y1);
                ph[8 * g + e / 2] = p;
                if (PP == 2) {
                    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&p));
                    pl[8 * g + e / 2] = pack_half2(y0 - b.x, y1 - b.y);
                }
            }
            const float sum = unpack2(sum2).x + unpack2(sum2).y;
            big = sum <= big ? big : sum;
            l = fmaf(sum, gr.unlv, l);
        }
        // 32 columns for 32 positions: 16 of first pieces, 16 of second ones
        tm_st16(sm + 32 * k, ph);
        if (PP == 2) tm_st16(sm + 32 * k + 16, pl);
    }
    return l;
}

template <class T, bool E4M3, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_kv8_chunk(const Kv8 c, const Kv8Att a) {
    using L = Layout<T, HD>;
    constexpr int PN = HD / 64, QP = kQPieces<T>, PP = kPPieces<T>, NS = L::slots, SUM = kSumSteps<T>;
    constexpr int ROWS = 128 * L::tiles, SUM1 = SUM > 0 ? SUM : 1;
    constexpr float unit = E4M3 ? 256.f : 1.f;
    constexpr float SU = PP == 1 ? 1.f / 256.f : 1.f;  // the unit of the weights' sums: 1 / vs is up to 2^109, 2^-ex up to 2^101
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars &bar = *reinterpret_cast<Bars *>(smem + L::bars);
    Group *groups = reinterpret_cast<Group *>(smem + L::group);
    float *facs = reinterpret_cast<float *>(smem + L::fac);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int s = blockIdx.z, head = blockIdx.y % c.kvh, row0 = blockIdx.y / c.kvh * ROWS;
    cudaTriggerProgrammaticLaunchCompletion();  // the join waits for this kernel's end itself
    const Kv8Seq sq = kv8_seq(c, s);
    const int rows = sq.n * a.group;
    if (row0 >= rows) return;
    const int last = min(row0 + ROWS, rows) - 1;
    int lo, hi;
    kv8_span(sq, a.window, row0 / a.group, last / a.group, lo, hi);
    if (blockIdx.x > 0 && lo + (int64_t)blockIdx.x * a.part >= hi) return;
    lo += blockIdx.x * a.part;
    hi = min(hi, lo + a.part);
    const int steps = max(hi - lo + kKeys - 1, 0) / kKeys, tiles = last - row0 >= 128 ? 2 : 1;

    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&bar.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 4; ++i) bar_init(&bar.full[i], 4), bar_init(&bar.empty[i], 1);
        for (int i = 0; i < 8; ++i) bar_init(&bar.raw[i], 1), bar_init(&bar.free[i], 4), bar_init(&bar.group[i], 1);
        for (int i = 0; i < 2; ++i) bar_init(&bar.s[i], 1), bar_init(&bar.p[i], 4), bar_init(&bar.q[i], 4), bar_init(&bar.o[i], 1);
        bar_init(&bar.done, 1);
        bar.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = bar.tmem;
    uint32_t *fail = &bar.fail;
    bool ok = true;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegSoft));
        const int w = warp >> 2, wq = warp & 3;  // the tile; the warp's 32 lanes of tensor memory
        if (w < tiles) {
            load_queries<T, HD>(a, sq, head, row0 + 128 * w, rows, wq, lane, smem + w * L::q_tile, facs + 128 * w, unit);
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(&bar.q[w]);
            const int r = row0 + 128 * w + 32 * wq + lane;
            const bool on = r < rows;
            const int tok = on ? r / a.group : 0, h = head * a.group + (on ? r - tok * a.group : 0);
            const int pos = on ? sq.first + tok : -1;
            const float fac = facs[128 * w + 32 * wq + lane];
            const uint32_t sm = tmem + ((uint32_t)(32 * wq) << 16) + 128 * w, om = tmem + ((uint32_t)(32 * wq) << 16) + L::tm_r + HD * w;
            const uint32_t am = om - L::tm_r + L::tm_o;  // the accumulator
            float m = -FLT_MAX, l = 0.f;
            for (int j = 0; j < steps; ++j) {
                const int p0 = lo + j * kKeys;
                // the row sees positions p0 + [b0, b1)
                const int b1 = min(min(pos + 1, hi) - p0, kKeys), b0 = max(kv8_first_seen(pos, a.window) - p0, 0);
                const bool whole = __all_sync(kFull, b0 == 0 && b1 == kKeys);
                ok = bar_wait(&bar.group[j & 7], (j >> 3) & 1, fail) && bar_wait(&bar.s[w], j & 1, fail);
                if (!(ok = __all_sync(kFull, ok))) break;
                fence_after();
                const Group *gp = groups + (j & 7) * 8;
                uint32_t x[4][32];
#pragma unroll
                for (int k = 0; k < 4; ++k) tm_ld32(sm + 32 * k, x[k]);
#pragma unroll
                for (int k = 0; k < 4; ++k) tm_wait(x[k]);
                auto weigh = [&](float &big) {
                    return whole ? row_weights<PP, true>(x, sm, gp, fac, 6.f - m, b0, b1, big)
                                 : row_weights<PP, false>(x, sm, gp, fac, 6.f - m, b0, b1, big);
                };
                auto find = [&]() { return whole ? row_top<true>(x, gp, fac, b0, b1) : row_top<false>(x, gp, fac, b0, b1); };
                float f = 1.f, big, sum = 0.f;
                bool fresh;
                auto raise = [&](float top) {
                    const float n = fmaxf(top, m);
                    f = kv8_exp2(m - n);
                    m = n;
                    l *= f;
                };
                if constexpr (PP == 1) {
                    // The maximum of the steps before serves as long as no weight is above 2^14 (float16 ends at 2^16); with
                    // this step's looked for first the three prompts took 334 us in place of 298.
                    fresh = j == 0;
                    if (!fresh) {
                        sum = weigh(big);
                        fresh = __any_sync(kFull, !(big <= 16384.f));
                    }
                    if (fresh) {
                        raise(find());
                        tm_st_wait();  // (stores of one thread have no order of their own)
                        sum = weigh(big);
                    }
                } else {  // (two pieces leave no registers for weighing twice: it spilled and was slower)
                    const float top = find();
                    fresh = __any_sync(kFull, top - m > 8.f);
                    if (fresh) raise(top);
                    sum = weigh(big);
                }
                l += sum;
                // (every product issued before this step's S is done)
                const bool add = SUM > 0 && j > 0 && j % SUM1 == 0;
                if (j > 0 && (fresh || add)) {
#pragma unroll 1
                    for (int k = 0; k < HD; k += 16) {
                        uint32_t r[16], v[16];
                        const bool both = SUM > 0 && j > SUM;  // there is a result already
                        tm_ld16(am + k, v);
                        if (both) tm_ld16(om + k, r);
                        tm_wait(v);
                        if (both) tm_wait(r);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float y = both ? __uint_as_float(r[e]) : 0.f, z = __uint_as_float(v[e]);
                            r[e] = __float_as_uint((add ? y + z : y) * f);
                            v[e] = __float_as_uint(z * f);
                        }
                        if (SUM > 0 && (both || add)) tm_st16(om + k, r);
                        if (!add) tm_st16(am + k, v);
                    }
                }
                tm_st_wait();
                fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&bar.p[w]);
            }
            // (without a step, until the other warps' queries are where results go by)
            if (ok) ok = bar_wait(steps > 0 ? &bar.o[w] : &bar.q[w], 0, fail);
            fence_after();
            ok = __all_sync(kFull, ok);
            // The rows' results, CW columns at a time by way of the tile's queries' place (their products are done), so that
            // lanes store neighbouring elements: a lane for each row would touch 32 lines an instruction (3.5 K cycles).
            constexpr int CW = L::q_tile >= 4 * 32 * (32 + 4) * 4 ? 32 : 16, PITCH = CW + 4, LR = CW / 4;  // lanes of a row
            static_assert(L::q_tile >= 4 * 32 * PITCH * 4, "the results' place");
            float *stage = reinterpret_cast<float *>(smem + w * L::q_tile) + wq * 32 * PITCH;
            const int64_t part = ((int64_t)(sq.start + tok) * a.heads + h) * a.splits + blockIdx.x;
            const bool split = a.splits > 1;
            // where the lane's row goes (-1: nowhere), and the rows that it stores pieces of
            const int64_t own = !on ? -1 : split ? part * HD : (int64_t)(sq.start + tok) * a.out_stride + h * HD;
            const float inv = split ? unit * SU : l == 0.f ? 0.f : unit * SU / l;
            if (on && split) a.part_ml[part] = make_float2(m, ok ? l : NAN);
#pragma unroll 1
            for (int k = 0; k < HD / CW; ++k) {
#pragma unroll
                for (int k2 = 0; k2 < CW; k2 += 16) {
                    uint32_t x[16];
                    if (steps > 0 && ok) {
                        tm_ld16(am + CW * k + k2, x);
                        tm_wait(x);
                        if (SUM > 0 && steps > SUM) {
                            uint32_t r2[16];
                            tm_ld16(om + CW * k + k2, r2);
                            tm_wait(r2);
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(r2[e]));
                        }
                    }
                    float y[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[e] = !ok ? NAN : steps == 0 || (!split && l == 0.f) ? 0.f : __uint_as_float(x[e]) * inv;
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4 *>(stage + lane * PITCH + k2 + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < LR; ++i) {
                    const int row = i * (32 / LR) + lane / LR, c4 = lane % LR * 4;
                    const int64_t to = __shfl_sync(kFull, own, row);
                    const float4 v = *reinterpret_cast<const float4 *>(stage + row * PITCH + c4);
                    if (to < 0) continue;
                    if (split) {
                        *reinterpret_cast<float4 *>(a.part_o + to + CW * k + c4) = v;
                    } else {
                        T *dst = static_cast<T *>(a.out) + to + CW * k + c4;
                        if constexpr (sizeof(T) == 4) {
                            *reinterpret_cast<float4 *>(dst) = v;
                        } else {
                            const T o[4] = {kv8_from<T>(v.x), kv8_from<T>(v.y), kv8_from<T>(v.z), kv8_from<T>(v.w)};
                            *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(o);
                        }
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegCopy));
        // K and V of one step after the other, 16 bytes a thread and piece
        constexpr int PC = HD / 16, NP = PC, D = L::copies;  // pieces of a row, of a thread
        const int t = threadIdx.x - 256, key0 = t / PC, seg = t % PC;
        const uint8_t *raw = smem + L::raw + 16 * t;
        for (int i = 0; i < 2 * steps; ++i) {
            const int slot = i % NS;
            ok = bar_wait(&bar.raw[i % D], (i / D) & 1, fail) && (i < NS || bar_wait(&bar.empty[slot], (i / NS - 1) & 1, fail));
            if (!(ok = __all_sync(kFull, ok))) break;
            // The row's chunks 2 seg and 2 seg + 1 (its key is key0 modulo 8 in every piece).  Both panels' chunks lie in
            // the same banks, so the second panel's odd chunks are stored with the first one's even ones.
            const bool odd = HD == 128 && seg >= 4;
            uint8_t *dst = smem + L::ring + slot * L::slot + seg / 4 * L::panel + key0 * 128;
            const int c0 = ((2 * (seg & 3) + odd) ^ (key0 & 7)) << 4, c1 = c0 ^ 16;
            const uint8_t *src = raw + (i % D) * 128 * HD;
            uint4 x[NP];
#pragma unroll
            for (int n = 0; n < NP; ++n) x[n] = *reinterpret_cast<const uint4 *>(src + n * 2048);
            __syncwarp();
            if (lane == 0) bar_arrive(&bar.free[i % D]);
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const uint32_t a0 = odd ? x[n].z : x[n].x, a1 = odd ? x[n].w : x[n].y;
                const uint32_t b0 = odd ? x[n].x : x[n].z, b1 = odd ? x[n].y : x[n].w;
                *reinterpret_cast<uint4 *>(dst + n * (128 / PC) * 128 + c0) =
                    make_uint4(kv8_half2<E4M3>(__byte_perm(a0, 0, 0x4140)), kv8_half2<E4M3>(__byte_perm(a0, 0, 0x4342)),
                               kv8_half2<E4M3>(__byte_perm(a1, 0, 0x4140)), kv8_half2<E4M3>(__byte_perm(a1, 0, 0x4342)));
                *reinterpret_cast<uint4 *>(dst + n * (128 / PC) * 128 + c1) =
                    make_uint4(kv8_half2<E4M3>(__byte_perm(b0, 0, 0x4140)), kv8_half2<E4M3>(__byte_perm(b0, 0, 0x4342)),
                               kv8_half2<E4M3>(__byte_perm(b1, 0, 0x4140)), kv8_half2<E4M3>(__byte_perm(b1, 0, 0x4342)));
            }
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(&bar.full[slot]);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegIssue));
        if (warp == 12) {
            // the whole warp goes along, so that descriptors stay uniform; one lane issues
            const bool one = elect();
            const uint32_t ring = su32(smem + L::ring);
            const uint64_t d0 = sdesc(0, L::panel), q_base = d0 + (su32(smem) >> 4), r_base = d0 + (ring >> 4);
            auto qk = [&](int w, int i) {  // S of tile w from the K in item i's slot
                const uint64_t q0 = q_base + ((w * L::q_tile) >> 4), k0 = r_base + (((i % NS) * L::slot) >> 4);
#pragma unroll
                for (int p = QP - 1; p >= 0; --p)  // the small products first: sums are cut to 24 bits
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k) {
                        const uint64_t off = (uint64_t)((k / 4) * L::panel + (k % 4) * 32) >> 4;
                        mma_ss(one, tmem + 128 * w, q0 + off + (uint64_t)((p * PN * L::panel) >> 4), k0 + off, idesc(kKeys, 0),
                               p < QP - 1 || k > 0);
                    }
                commit(one, &bar.s[w]);
            };
            auto pv = [&](int w, int j) {  // O of tile w from its weights and the V of step j
                const uint64_t v0 = r_base + ((((2 * j + 1) % NS) * L::slot) >> 4);
#pragma unroll
                for (int p = PP - 1; p >= 0; --p)
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        mma_ts(one, tmem + L::tm_o + HD * w, tmem + 128 * w + 32 * (k / 2) + 8 * (k % 2) + 16 * p,
                               v0 + (uint64_t)((k * 2048) >> 4), idesc(HD, 1),
                               (SUM > 0 ? j % SUM1 > 0 : j > 0) || k > 0 || p < PP - 1);
            };
            auto wait = [&](uint64_t *b, uint32_t parity) { return __all_sync(kFull, bar_wait(b, parity, fail)) != 0; };
            auto full = [&](int i) { return wait(&bar.full[i % NS], (i / NS) & 1); };
            if (steps > 0) {
                ok = full(0);
                for (int w = 0; ok && w < tiles; ++w) {
                    if (!(ok = wait(&bar.q[w], 0))) break;
                    fence_after();
                    qk(w, 0);
                }
                if (ok) commit(one, &bar.empty[0]);
            }
            for (int j = 0; ok && j < steps; ++j) {
                if (!(ok = full(2 * j + 1))) break;
                for (int w = 0; ok && w < tiles; ++w) {
                    if (!(ok = wait(&bar.p[w], j & 1))) break;
                    fence_after();
                    pv(w, j);
                    if (w == tiles - 1) commit(one, &bar.empty[(2 * j + 1) % NS]);
                    if (j + 1 < steps) {
                        if (w == 0 && !(ok = full(2 * j + 2))) break;
                        fence_after();
                        qk(w, 2 * j + 2);
                        if (w == tiles - 1) commit(one, &bar.empty[(2 * j + 2) % NS]);
                    } else {
                        commit(one, &bar.o[w]);
                    }
                }
            }
            if (steps > 0) {  // nothing is in flight when tensor memory is given back, after a failure either
                uint32_t never = 0;
                commit(one, &bar.done);
                bar_wait(&bar.done, 0, &never);
            }
        } else if (warp == 13) {
            // Lane g has group g of 16 positions; a group without a block keeps what lies there, which is finite and gets no
            // weight.
            constexpr int D = L::copies;
            auto block_of = [&](int j) {
                const int p = lo + j * kKeys + 16 * lane;
                return lane < 8 && p < hi ? kv8_block(c, s, p >> c.bshift) : -1;
            };
            int b = steps > 0 ? block_of(0) : -1, sent = 0, low = kKv8NoExp;
            for (int j = 0; ok && j < steps; ++j) {
                const int ahead = j + 1 < steps ? block_of(j + 1) : -1;
                const int64_t off = b < 0 ? 0 : b * c.bstride + ((int64_t)head * c.block + ((lo + j * kKeys + 16 * lane) & (c.block - 1))) * HD;
                float ks = 0.f, vs = 0.f;
                if (b >= 0) ks = __ldg(c.ks + (int64_t)b * c.kvh + head), vs = __ldg(c.vs + (int64_t)b * c.kvh + head);
                // the groups of a block lie one after the other: the lane of its first one copies them all
                const int per = c.block >> 4, in_block = ((lo + j * kKeys) >> 4) + lane & (per - 1);
                const bool first = b >= 0 && (lane == 0 || in_block == 0);
                const int n = min(min(per - in_block, 8 - lane), ((hi - lo - j * kKeys + 15) >> 4) - lane);
                const bool scaled = vs >= kv8_pow2(kKv8LeastScale) && vs <= FLT_MAX;
                const uint32_t bytes = 16 * HD * __popc(__ballot_sync(kFull, b >= 0));
                for (int i = 2 * j; i < 2 * j + 2; ++i) {
                    ok = i < D || bar_wait(&bar.free[i % D], (i / D - 1) & 1, fail);
                    if (!(ok = __all_sync(kFull, ok))) break;
                    // blocks whose values are 0, whatever their bytes
                    const uint32_t none = PP == 1 && (i & 1) ? __ballot_sync(kFull, b >= 0 && !scaled) : 0;
                    for (uint32_t left = none; left; left &= left - 1)
                        for (int k = lane; k < HD; k += 32)
                            *reinterpret_cast<uint4 *>(smem + L::raw + (i % D) * 128 * HD + (__ffs(left) - 1) * 16 * HD + 16 * k) =
                                make_uint4(0, 0, 0, 0);
                    if (none) fence_async();  // later copies come after these stores
                    __syncwarp();
                    if (lane == 0) bar_expect(&bar.raw[i % D], bytes - 16 * HD * __popc(none));
                    __syncwarp();
                    if (first && !(none >> lane & 1))
                        bulk(smem + L::raw + (i % D) * 128 * HD + lane * 16 * HD, (i & 1 ? c.v : c.k) + off, n * 16 * HD, &bar.raw[i % D]);
                    sent = i + 1;
                }
                if (!ok) break;
                // The groups' scales.  Their place was last read in step j - 8, which was over: this step's V is copied to
                // where V of step j - copies / 2 was, after that was stored to a slot, after the products that used the
                // slot before, of a step j - 6 at the earliest, and so the weights of the step before that, were done.
                Group g = {0.f, -INFINITY, 0.f, 0.f};  // no block: -inf as a score
                const int ex = kv8_v_scale(vs, g.mv, low);
                if (b >= 0) {
                    g.ks = ks, g.lv = (float)ex, g.unlv = kv8_pow2(-ex) * SU;
                    if (PP == 1 && scaled) g.lv = log2f(vs), g.unlv = SU / vs;
                }
                if (lane < 8) groups[(j & 7) * 8 + lane] = g;
                __syncwarp();
                if (lane == 0) bar_arrive(&bar.group[j & 7]);
                b = ahead;
            }
            if (!ok)  // copies that were sent arrive before the block ends
                for (int i = max(sent - D, 0); i < sent; ++i) {
                    uint32_t never = 0;
                    bar_wait(&bar.raw[i % D], (i / D) & 1, &never);
                }
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

template <class T, bool E4M3, int HD>
cudaError_t launch(const Kv8 &c, const Kv8Att &a, dim3 grid, int device, cudaStream_t st) noexcept {
    constexpr int bytes = Layout<T, HD>::total;
    const cudaError_t e = op_shared<k_kv8_chunk<T, E4M3, HD>>(device, bytes);
    if (e == cudaSuccess) k_kv8_chunk<T, E4M3, HD><<<grid, kThreads, bytes, st>>>(c, a);
    return e;
}

template <class T>
cudaError_t launch(bool e4m3, int hd, const Kv8 &c, const Kv8Att &a, dim3 grid, int device, cudaStream_t st) noexcept {
    if (e4m3) return hd == 64 ? launch<T, true, 64>(c, a, grid, device, st) : launch<T, true, 128>(c, a, grid, device, st);
    return hd == 64 ? launch<T, false, 64>(c, a, grid, device, st) : launch<T, false, 128>(c, a, grid, device, st);
}

}  // namespace

cudaError_t kv8_chunk_launch(int type, bool e4m3, int hd, const Kv8 &c, const Kv8Att &a, dim3 grid, int device,
                             cudaStream_t st) noexcept {
    if (type == LLMB_F32) return launch<float>(e4m3, hd, c, a, grid, device, st);
    if (type == LLMB_F16) return launch<__half>(e4m3, hd, c, a, grid, device, st);
    return launch<__nv_bfloat16>(e4m3, hd, c, a, grid, device, st);
}

}  // namespace llmb
