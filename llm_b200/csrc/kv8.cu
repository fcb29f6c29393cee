// The 8-bit key/value cache: append, read, and attention for few rows
// (llmb_kv8_append, llmb_kv8_read, llmb_kv8_attention).
#include <cuda_fp8.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "kv8.hpp"
#include "kv8_chunk.hpp"
#include "ops.hpp"
#include "ptx.hpp"

namespace llmb {
namespace {

// ------------------------------------------------------------- append --

template <bool E4M3>
__host__ __device__ constexpr float kv8_top() { return E4M3 ? 448.f : 127.f; }

constexpr float kFit = 1.f / 4096.f;        // a scale still fits top + kFit steps: the scale a (1 / top) made for a fits a, whatever its roundings
constexpr float kTiny = 7.888609052e-31f;   // 2^-100
constexpr float kRestart = 1048576.f;       // 2^20

// Four values to 8 bits: to the nearest, ties to even, saturated; NaN becomes 0.  FINITE: none of the products is infinite or
// NaN and none above the top by more than a quarter, so that rounding alone ends at the top.
template <bool E4M3, bool FINITE>
__device__ __forceinline__ uint32_t kv8_pack(const float (&x)[4], float inv) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = __fmul_rn(x[i], inv);
        if (!FINITE) y[i] = y[i] == y[i] ? fminf(fmaxf(y[i], -kv8_top<E4M3>()), kv8_top<E4M3>()) : 0.f;
    }
    if constexpr (E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        return lo | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3) << 16;
    } else {
        // 1.5 2^23 + y: the rounded y is in the low bits (a conversion to int runs at a quarter of an addition's rate)
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = __float_as_uint(__fadd_rn(y[i], 12582912.f));
        return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
}

// The largest magnitude's bits of the 16 bytes, in the upper half for 16-bit types: they order like the values, with
// infinity and NaN above the finite ones (from kv8_inf on).
template <class T>
__device__ __forceinline__ uint32_t kv8_top_bits(const uint4 &r, uint32_t m) {
    if (sizeof(T) == 4)
        return max(max(max(m, r.x & 0x7fffffffu), r.y & 0x7fffffffu), max(r.z & 0x7fffffffu, r.w & 0x7fffffffu));
    return __vmaxu2(__vmaxu2(__vmaxu2(m, r.x & 0x7fff7fffu), __vmaxu2(r.y & 0x7fff7fffu, r.z & 0x7fff7fffu)), r.w & 0x7fff7fffu);
}
template <class T>
constexpr uint32_t kv8_inf = 0x7f800000u;
template <>
constexpr uint32_t kv8_inf<__half> = 0x7c00u;
template <>
constexpr uint32_t kv8_inf<__nv_bfloat16> = 0x7f80u;
template <class T>
__device__ __forceinline__ float kv8_of_bits(uint32_t m) {
    if (sizeof(T) == 4) return __uint_as_float(m);
    const unsigned short h = (unsigned short)m;
    return kv8_float<T>(*reinterpret_cast<const T *>(&h));
}

// A block's new scale from the largest magnitude a of the rows it receives
// and the scale s0 of the rows it holds (0: none); old_factor is what the
// values it holds are multiplied by.
template <bool E4M3>
__device__ __forceinline__ float kv8_grow(float a, float s0, float &old_factor) {
    old_factor = 1.f;
    if (a < kTiny) return s0;
    const float fresh = __fmul_rn(a, 1.f / kv8_top<E4M3>());
    if (s0 == 0.f) return fresh;
    const float r = __fdiv_rn(a, __fmul_rn(kv8_top<E4M3>() + kFit, s0));
    if (r <= 1.f) return s0;
    if (!(r <= kRestart)) {
        old_factor = 0.f;
        return fresh;
    }
    // the least k with r <= 2^k: r = m 2^e, m in [1, 2), gives e, or e + 1 where m > 1
    const uint32_t u = __float_as_uint(r);
    const int k = (int)(u >> 23) - 127 + ((u & 0x7fffffu) != 0);
    old_factor = __uint_as_float((uint32_t)(127 - k) << 23);
    return __fmul_rn(s0, __uint_as_float((uint32_t)(127 + k) << 23));
}

template <class T>
__device__ __forceinline__ void kv8_unpack(const uint4 &r, float (&x)[16 / sizeof(T)]) {
    const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
    for (int i = 0; i < (int)(16 / sizeof(T)); ++i) x[i] = kv8_float<T>(e[i]);
}

// One block of a sequence, and `tiles` of its 2 kv_heads tiles (K and V of one
// head after the other): a tile's new rows are held in registers (U pieces of
// 16 bytes a thread) between the maximum and the rounding, so they are read
// once, and the next tile's are on their way meanwhile.  Bound by the memory's
// rate (64 bfloat16 prompts of up to 1000 positions, 16 tiles of 64 x 128: 202
// MB in 44 us, 70 % of the measured copy rate; with one tile a block of
// threads, whose three look-ups, lengths, table and scale, come before its
// first load, and a conversion a value 65 us).  A decoding step is 2 us, a
// launch's latency.
template <class T, bool E4M3, int HD, int U>
__global__ void __launch_bounds__(256) k_kv8_append(const Kv8 c, const T *__restrict__ k, const T *__restrict__ v,
                                                    int64_t row_stride, int tiles) {
    constexpr int E = 16 / (int)sizeof(T), PR = HD / E;  // elements of a piece, pieces of a row
    const int s = blockIdx.z;
    const Kv8Seq q = kv8_seq(c, s);
    if (q.n <= 0) return;
    const int first = max(q.first, 0);
    const int j = (first >> c.bshift) + blockIdx.x;
    const int b = kv8_block(c, s, j);
    if (b < 0) return;
    const int p0 = j << c.bshift, end = q.first + q.n;
    if (p0 >= end) return;
    const int lo = max(first - p0, 0), hi = min(end - p0, c.block), total = (hi - lo) * PR;
    const int64_t row = (int64_t)(q.start + p0 + lo - q.first) * row_stride;
    const int t1 = min((int)(blockIdx.y + 1) * tiles, 2 * c.kvh);
    __shared__ uint32_t red[2][8];
    uint4 x[U], y[U];
    float s0 = 0.f, s1 = 0.f;
    auto load = [&](int t, uint4 (&r)[U], float &held) {  // tile t: head t / 2, V where t is odd
        const T *src = (t & 1 ? v : k) + row + (t >> 1) * HD;
        held = lo > 0 ? (t & 1 ? c.vs : c.ks)[(int64_t)b * c.kvh + (t >> 1)] : 0.f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            if (u < total) r[i] = __ldg(reinterpret_cast<const uint4 *>(src + (int64_t)(u / PR) * row_stride + u % PR * E));
        }
    };
    auto store = [&](int t, const uint4 (&r)[U], float s0) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if ((int)(threadIdx.x + i * blockDim.x) < total) m = kv8_top_bits<T>(r[i], m);
        if (sizeof(T) == 2) m = max(m & 0xffffu, m >> 16);
        if (!(s0 > 0.f && s0 <= FLT_MAX)) s0 = 0.f;
        m = __reduce_max_sync(kFull, m);
        if ((threadIdx.x & 31) == 0) red[t & 1][threadIdx.x >> 5] = m;
        __syncthreads();  // and every thread has read this tile's scale
        for (int w = 0; w < (int)blockDim.x / 32; ++w) m = max(m, red[t & 1][w]);
        const bool finite = m < kv8_inf<T>;
        float a = kv8_of_bits<T>(m);
        if (!finite) {  // the largest of the finite ones
            a = 0.f;
#pragma unroll
            for (int i = 0; i < U; ++i)
                if ((int)(threadIdx.x + i * blockDim.x) < total) {
                    float f[E];
                    kv8_unpack<T>(r[i], f);
#pragma unroll
                    for (int e = 0; e < E; ++e) a = fabsf(f[e]) <= FLT_MAX ? fmaxf(a, fabsf(f[e])) : a;
                }
            m = __reduce_max_sync(kFull, __float_as_uint(a));
            __syncthreads();
            if ((threadIdx.x & 31) == 0) red[t & 1][threadIdx.x >> 5] = m;
            __syncthreads();
            for (int w = 0; w < (int)blockDim.x / 32; ++w) m = max(m, red[t & 1][w]);
            a = __uint_as_float(m);
        }
        float old;
        const float sc = kv8_grow<E4M3>(a, s0, old);
        if (s0 == 0.f) old = 0.f;  // rows without a scale are 0
        uint8_t *tile = (t & 1 ? c.v : c.k) + b * c.bstride + (int64_t)(t >> 1) * c.block * HD;
        if (threadIdx.x == 0) (t & 1 ? c.vs : c.ks)[(int64_t)b * c.kvh + (t >> 1)] = sc;
        const float inv = sc > 0.f ? __fdiv_rn(1.f, sc) : 0.f;
        auto write = [&](auto all_finite) {
            constexpr bool F = decltype(all_finite)::value;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const int u = threadIdx.x + i * blockDim.x;
                if (u < total) {
                    float f[E];
                    kv8_unpack<T>(r[i], f);
                    uint32_t *dst = reinterpret_cast<uint32_t *>(tile + lo * HD + u * E);
                    if constexpr (E == 4) {
                        *dst = kv8_pack<E4M3, F>(f, inv);
                    } else {
                        const float f0[4] = {f[0], f[1], f[2], f[3]}, f1[4] = {f[4], f[5], f[6], f[7]};
                        *reinterpret_cast<uint2 *>(dst) = make_uint2(kv8_pack<E4M3, F>(f0, inv), kv8_pack<E4M3, F>(f1, inv));
                    }
                }
            }
        };
        // (rows below kTiny take a scale as it is, and one of the caller's may be too small for them, its inverse infinite)
        finite && __fmul_rn(a, inv) <= kv8_top<E4M3>() + 0.25f ? write(std::true_type{}) : write(std::false_type{});
        if (old != 1.f)
            for (int u = threadIdx.x; u < lo * HD / 4; u += blockDim.x) {
                uint32_t *w = reinterpret_cast<uint32_t *>(tile) + u;
                float f[4];
                kv8_floats<E4M3>(*w, f);
                *w = kv8_pack<E4M3, false>(f, old);  // (a byte may be anything)
            }
    };
    int t = blockIdx.y * tiles;
    if (t >= t1) return;
    load(t, x, s0);
    for (; t < t1; t += 2) {
        if (t + 1 < t1) load(t + 1, y, s1);
        store(t, x, s0);
        if (t + 1 >= t1) break;
        if (t + 2 < t1) load(t + 2, x, s0);
        store(t + 1, y, s1);
    }
}

// Tiles of a block that one block of threads takes: as many as spread its look-ups without leaving SMs idle.
int tiles_each(const Kv8 &c, int64_t touched, int tile_bytes) {
    const int64_t all = touched * c.nseq * 2 * c.kvh;
    return (int)std::max<int64_t>(1, std::min<int64_t>({all / (148 * 8), 2 * c.kvh, 65536 / tile_bytes}));
}

template <class T, bool E4M3, int HD>
void append_launch(const Kv8 &c, const void *k, const void *v, int64_t row_stride, int touched, cudaStream_t st) {
    const int tiles = tiles_each(c, touched, c.block * HD * (int)sizeof(T));
    const dim3 grid(touched, (2 * c.kvh + tiles - 1) / tiles, c.nseq);
    const int pieces = min(c.max_new, c.block) * HD * (int)sizeof(T) / 16;
    const T *kp = static_cast<const T *>(k), *vp = static_cast<const T *>(v);
    // the fewest threads that hold the rows with few pieces each: a decoding step's single row needs one warp
    // (a block has at most 128 rows: HD sizeof(T) / 32 pieces for each of 256 threads)
    if (pieces <= 64) k_kv8_append<T, E4M3, HD, 2><<<grid, 32, 0, st>>>(c, kp, vp, row_stride, tiles);
    else if (HD * (int)sizeof(T) <= 128 || pieces <= 1024) k_kv8_append<T, E4M3, HD, 4><<<grid, 256, 0, st>>>(c, kp, vp, row_stride, tiles);
    else k_kv8_append<T, E4M3, HD, HD * (int)sizeof(T) / 32><<<grid, 256, 0, st>>>(c, kp, vp, row_stride, tiles);
}

// The four 8-bit values of w as two pairs of float16, exactly (bytes 0 and 1, bytes 2 and 3).
template <bool E4M3>
__device__ __forceinline__ void halves(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (E4M3) {
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {  // u = q + 128 under 1024's exponent is 1024 + u
        const uint32_t u = w ^ 0x80808080u, a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 k = __half2half2(__float2half_rn(1152.f));
        const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), k), y = __hsub2(*reinterpret_cast<const __half2 *>(&b), k);
        lo = *reinterpret_cast<const uint32_t *>(&x), hi = *reinterpret_cast<const uint32_t *>(&y);
    }
}

// --------------------------------------------------------------- read --

// One block of a sequence and `tiles` of its 2 kv_heads tiles, 16 bytes of
// result a thread and step, two steps' loads in flight.  A thread keeps its
// place in a row: its steps are whole rows and whole tiles apart, so that
// addresses cost additions only.  Bound by the memory's rate: 352 MB of 32 x
// 128 tiles of e4m3, two thirds of them written, in 66 us, 82 % of the measured
// copy rate, and 202 MB of 64 x 128 tiles of int8 in 46 us (with a division a
// step and 48 registers 76 and 49 us; four steps in flight: 70 and 46).  The
// conversions are the ones that measured best here: of e4m3 the machine's own
// (by shifts and a factor 72 us), of int8 by kv8_half2 (by `halves` 54 us).
template <class T, bool E4M3, int HD>
__global__ void __launch_bounds__(256) k_kv8_read(const Kv8 c, T *__restrict__ k, T *__restrict__ v,
                                                  int64_t row_stride, int tiles) {
    constexpr int E = 16 / (int)sizeof(T), PR = HD / E, N = 2;  // values of a step, steps of a row, steps in flight
    const int s = blockIdx.z;
    const Kv8Seq q = kv8_seq(c, s);
    if (q.n <= 0) return;
    // blocks counted from the one that holds the first row's position, which may be below 0
    const int j = (q.first >> c.bshift) + (int)blockIdx.x, end = q.first + q.n;
    if ((int64_t)j * c.block >= end) return;  // (a longer sequence's blocks, counted from the largest length, pass 2^31)
    const int p0 = j * c.block;
    const int b = kv8_block(c, s, j);
    const int lo = max(q.first - p0, 0), hi = min(end - p0, c.block);
    // the threads take 256 / per tiles at once, or a tile in per / 256 steps (both powers of two)
    const int shift = c.bshift + (PR == 32 ? 5 : PR == 16 ? 4 : 3), per = 1 << shift;
    const int steps = shift > 8 ? shift - 8 : 0, at_once = shift < 8 ? 8 - shift : 0;  // (their logarithms)
    const int in_tile = threadIdx.x & (per - 1), row0 = in_tile / PR, rows = min(per, 256) / PR;
    const int t0 = blockIdx.y * tiles + ((int)threadIdx.x >> min(shift, 8)), t1 = min((int)(blockIdx.y + 1) * tiles, 2 * c.kvh);
    const int64_t to = (int64_t)(q.start + p0 - q.first + row0) * row_stride + in_tile % PR * E;
    const int64_t from = (b < 0 ? 0 : b * c.bstride) + in_tile * E, apart = (int64_t)rows * row_stride;
    const float *ks = c.ks + (b < 0 ? 0 : (int64_t)b * c.kvh), *vs = c.vs + (b < 0 ? 0 : (int64_t)b * c.kvh);
    const int n = t1 > t0 ? (((t1 - t0 - 1) >> at_once) + 1) << steps : 0;
    for (int i0 = 0; i0 < n; i0 += N) {
        uint2 w[N];
        float sc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int t = t0 + ((i0 + i) >> steps << at_once), y = (i0 + i) & ((1 << steps) - 1);
            w[i] = make_uint2(0, 0), sc[i] = 0.f;
            if (i0 + i < n && b >= 0) {
                const uint8_t *src = (t & 1 ? c.v : c.k) + from + ((t >> 1) * c.block + y * rows) * HD;
                if constexpr (E == 8) w[i] = __ldg(reinterpret_cast<const uint2 *>(src));
                else w[i].x = __ldg(reinterpret_cast<const uint32_t *>(src));
                sc[i] = __ldg((t & 1 ? vs : ks) + (t >> 1));
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int t = t0 + ((i0 + i) >> steps << at_once), y = (i0 + i) & ((1 << steps) - 1), r = row0 + y * rows;
            T *dst = t & 1 ? v : k;
            if (i0 + i >= n || r < lo || r >= hi || !dst) continue;
            const uint32_t words[2] = {w[i].x, w[i].y};
            T o[E];
#pragma unroll
            for (int z = 0; z < E; z += 4) {
                float f[4];
                if constexpr (E4M3) {
                    uint32_t h[2];
                    halves<true>(words[z / 4], h[0], h[1]);
                    const float2 x0 = __half22float2(*reinterpret_cast<const __half2 *>(&h[0]));
                    const float2 x1 = __half22float2(*reinterpret_cast<const __half2 *>(&h[1]));
                    f[0] = x0.x, f[1] = x0.y, f[2] = x1.x, f[3] = x1.y;
                } else {
                    kv8_floats<false>(words[z / 4], f);
                }
                // (no block: a byte 0 is the value 0, and the scale is 0)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[z + x] = kv8_from<T>(__fmul_rn(f[x], sc[i]));
            }
            *reinterpret_cast<uint4 *>(dst + to + y * apart + (t >> 1) * HD) = *reinterpret_cast<const uint4 *>(o);
        }
    }
}

// ---------------------------------------------------------- attention --

constexpr int kAttWarps = 4;

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b)[2]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}

// The 8 x 8 matrix of 16-bit values whose row `lane / 4`, columns 2 (lane % 4) .. + 1 this lane holds, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// What 16 positions share: where they lie in the pools (below 0: nowhere), K's scale, V's scale = mv 2^lv with 2^-lv.
struct Place {
    int64_t at;
    float ks, lv, mv, unlv;
};

// Attention of 8 NB rows of one (sequence, kv head) over one part of the
// positions: softmax with a running maximum, both products as m16n8k16 with
// the 8-bit values exact in float16.  The cache is the left operand of both
// (S^T = K Q^T, O^T = V^T P^T), so the few rows fill the 8 columns and each
// value of the cache is converted once.
//
// A warp takes every 4th group of 16 positions, the next ones on their way
// (asynchronous copies) while one is worked on.  The contraction's index may
// be permuted as long as both operands agree, so lane (g, t) = (lane / 4,
// lane % 4) copies 16 contiguous bytes of the K rows g and g + 8 and uses them
// as its A fragments, and HD / 8 contiguous bytes of the V rows 2t, 2t + 1,
// 2t + 8, 2t + 9, whose bytes j, paired by two rows, are A fragments of
// elements g HD / 8 + j: each lane reads back only what it copied itself.  P
// comes out as accumulators of S^T and is transposed 8 x 8 into B fragments.
// A lane looks up the place of one group in 32 ahead of time.
//
// Bound, B200: one sequence of 131071 positions (32 heads on 8, size 128,
// e4m3, bfloat16 rows) 66 us with its join, 4.1 TB/s, 63 % of the measured copy
// rate: copies in flight and the ends of the one wave.  64 sequences of up to
// 2048 (9 heads on 3, size 64, int8, float32) 17.7 us, 1.9 TB/s: 324
// instructions a group and the sequences' different lengths.  300 positions of
// one sequence 6 us: latency.
//
// float32 rows (PIECES = 2) are the sum of two float16 pieces, which hold 22
// bits of the row's largest element after a power of two has brought it to
// [2^14, 2^15); the weights go into the second product the same way.
// float16 rows fit one piece, but a weight rounded to float16 is off as much
// as the result's own rounding (2^-12 and 2^-11 relative), so they take the
// two-piece form as well.  bfloat16 rows and their weights are one piece: a
// weight is off by 2^-12 at most, a sixteenth of the result's own rounding
// (2^-8), and the weights' errors are independent, so that a mean over many
// positions is off by less.  exp2 is the machine's approximation (2^-22
// relative).
//
// The scale of V's block enters the weights' exponent (its power of two, so
// that the largest weight of all stays near 2^6 and float16 holds the small
// ones) and mantissa (kv8_v_scale).
template <class T>
constexpr int kPieces = 2;
template <>
constexpr int kPieces<__nv_bfloat16> = 1;

// Groups of a warp in flight, as many as four CTAs an SM have room for (a group is 32 HD bytes), and their bytes.
__host__ __device__ constexpr int att_depth(int hd) { return hd == 64 ? 6 : 3; }
// Groups worked on at once: two where the registers of four CTAs an SM hold them (us with one / with two, the cache in L2: 64
// sequences 16.6 / 16.4, 33 with a window of 4000 in bfloat16 15.4 / 14.8, a chunk of 64 behind 1920 17.0 / 16.4).
__host__ __device__ constexpr int att_groups(int hd, int nb) { return hd == 64 && nb == 1 ? 2 : 1; }
__host__ __device__ constexpr int att_smem(int hd) { return kAttWarps * att_depth(hd) * 32 * hd; }

__device__ __forceinline__ void cp16(void *dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(su32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp8(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(su32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, bool E4M3, int HD, int NB>
__global__ void __launch_bounds__(kAttWarps * 32, NB == 1 ? 4 : 2) k_kv8_attend(const Kv8 c, const Kv8Att a) {
    constexpr int PIECES = kPieces<T>, ROWS = 8 * NB, KS = HD / 16, NT = HD / 16;  // k steps; tiles of 16 elements of V
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int s = blockIdx.z, head = blockIdx.y % c.kvh, row0 = blockIdx.y / c.kvh * ROWS;
    cudaTriggerProgrammaticLaunchCompletion();  // the join waits for this kernel's end itself
    const Kv8Seq sq = kv8_seq(c, s);
    const int rows = sq.n * a.group;
    if (row0 >= rows) return;
    const int last = min(row0 + ROWS, rows) - 1;
    const int tok0 = row0 / a.group, tok1 = last / a.group;
    int lo, hi;
    kv8_span(sq, a.window, tok0, tok1, lo, hi);
    if (blockIdx.x > 0 && lo + (int64_t)blockIdx.x * a.part >= hi) return;
    lo += blockIdx.x * a.part;
    hi = min(hi, lo + a.part);
    // every row sees all of [all0, all1)
    const int all0 = max(kv8_first_seen(sq.first + tok1, a.window), lo), all1 = min(sq.first + tok0 + 1, hi);

    constexpr int step = 16 * kAttWarps;
    int low = kKv8NoExp;
    auto look_up = [&](int p) {  // by the whole warp
        Place x = {-1, 0.f, 0.f, 0.f, 0.f};
        const int b = p < hi ? kv8_block(c, s, p >> c.bshift) : -1;
        float vs = 0.f;
        if (b >= 0) {
            x.at = b * c.bstride + ((int64_t)head * c.block + (p & (c.block - 1))) * HD;
            x.ks = __ldg(c.ks + (int64_t)b * c.kvh + head);
            vs = __ldg(c.vs + (int64_t)b * c.kvh + head);
        }
        const int ex = kv8_v_scale(vs, x.mv, low);
        x.lv = (float)ex, x.unlv = kv8_pow2(-ex);
        return x;
    };
    auto of_lane = [&](const Place &x, int i) {
        Place y;
        y.at = __shfl_sync(kFull, x.at, i);
        y.ks = __shfl_sync(kFull, x.ks, i), y.lv = __shfl_sync(kFull, x.lv, i);
        y.mv = __shfl_sync(kFull, x.mv, i), y.unlv = __shfl_sync(kFull, x.unlv, i);
        return y;
    };
    // a group of 16 positions as a lane holds it
    struct Group {
        uint4 k[2][HD / 64];
        uint32_t v[4][HD / 32];
        Place at;
    };
    const int k_lane = g * HD + 16 * t, v_lane = 2 * t * HD + g * (HD / 8);
    extern __shared__ __align__(16) uint8_t ring[];  // [warp][depth]: K's pieces [2][HD / 64][lane] of 16 bytes, V's [4][lane] of HD / 8
    constexpr int D = att_depth(HD), VB = HD / 8;
    uint8_t *mine = ring + warp * D * 32 * HD;
    int p = lo + 16 * warp, copied = 0;  // groups of the warp whose copies were started
    Place ahead = {-1, 0.f, 0.f, 0.f, 0.f};
    // starts the copies of the warp's next group, if there is one, and closes their set
    auto copy = [&]() {
        const int p1 = p + copied * step;
        if (p1 < hi) {
            if (copied % 32 == 0) ahead = look_up(p1 + lane * step);
            const int64_t at = __shfl_sync(kFull, ahead.at, copied % 32);
            if (at >= 0) {
                const uint8_t *kp = c.k + at + k_lane, *vp = c.v + at + v_lane;
                uint8_t *dst = mine + copied % D * 32 * HD;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int i = 0; i < HD / 64; ++i) cp16(dst + ((n * (HD / 64) + i) * 32 + lane) * 16, kp + 8 * n * HD + 64 * i);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    uint8_t *to = dst + 16 * HD + (n * 32 + lane) * VB;
                    const uint8_t *from = vp + ((n & 1) + 8 * (n >> 1)) * HD;
                    if constexpr (HD == 64) cp8(to, from);
                    else cp16(to, from);
                }
            }
            ++copied;
        }
        cp_commit();
    };
    // the first groups are on their way before the queries are read
#pragma unroll
    for (int i = 0; i < D - att_groups(HD, NB); ++i) copy();

    // the rows' queries as B fragments: row g of each 8
    uint32_t qf[NB][PIECES][KS][2];
    float fac[NB][2];   // rows 2t and 2t + 1, as the accumulators have them
    int pos[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int r = min(row0 + 8 * i + g, last), tok = r / a.group, h = head * a.group + r - tok * a.group;
        const T *qp = static_cast<const T *>(a.q) + (int64_t)(sq.start + tok) * a.q_stride + h * HD;
        float x[KS][4];
        uint32_t m = 0;  // the largest magnitude's bits; infinity and NaN are above the finite ones
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            // 16 bytes of K hold the 4 values of 4 steps: value e of step ks is element 64 (ks / 4) + 16 t + 4 (ks % 4) + e
            const T *e = qp + 64 * (ks / 4) + 16 * t + 4 * (ks % 4);
            T v[4];
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(e);
            else *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(e);
#pragma unroll
            for (int e2 = 0; e2 < 4; ++e2) x[ks][e2] = kv8_float<T>(v[e2]), m = max(m, __float_as_uint(x[ks][e2]) & 0x7fffffffu);
        }
        m = max(m, __shfl_xor_sync(kFull, m, 1));
        m = max(m, __shfl_xor_sync(kFull, m, 2));
        float up, down;
        const bool fine = kv8_query_scale(m, up, down);
        const float f = fine ? a.scale * down : NAN;  // a row that is not finite has NaN as its factor
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fine ? x[ks][e] * up : 0.f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t w = pack_half2(y[2 * j], y[2 * j + 1]);
                qf[i][0][ks][j] = w;
                if constexpr (PIECES == 2) {
                    const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&w));
                    qf[i][1][ks][j] = pack_half2(y[2 * j] - b.x, y[2 * j + 1] - b.y);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            fac[i][e] = __shfl_sync(kFull, f, 4 * (2 * t + e));
            const int r2 = row0 + 8 * i + 2 * t + e;
            pos[i][e] = r2 <= last ? max(sq.first + r2 / a.group, -1) : -1;  // (less any window it is an int)
        }
    }

    float o[NB][NT][4], m[NB][2], l[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
        m[i][0] = m[i][1] = -FLT_MAX, l[i][0] = l[i][1] = 0.f;
    }

    // G groups at once: their chains of products and exponentials do not wait for one another.
    auto use = [&](auto groups, Group *x, int p0) {
        constexpr int G = decltype(groups)::value;
        bool whole = true;
#pragma unroll
        for (int y = 0; y < G; ++y) whole = whole && p0 + y * step >= all0 && p0 + y * step + 16 <= all1;
        float sc[G][NB][4];
#pragma unroll
        for (int y = 0; y < G; ++y)
#pragma unroll
            for (int i = 0; i < NB; ++i) sc[y][i][0] = sc[y][i][1] = sc[y][i][2] = sc[y][i][3] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int y = 0; y < G; ++y) {
                uint32_t k0[2], k1[2];
                auto word = [&](const uint4 &w) { return ks % 4 == 0 ? w.x : ks % 4 == 1 ? w.y : ks % 4 == 2 ? w.z : w.w; };
                halves<E4M3>(word(x[y].k[0][ks / 4]), k0[0], k1[0]);
                halves<E4M3>(word(x[y].k[1][ks / 4]), k0[1], k1[1]);
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int q = PIECES - 1; q >= 0; --q) mma16816(sc[y][i], k0[0], k0[1], k1[0], k1[1], qf[i][q][ks]);
            }
        // sc[.][.][e]: position p0 + g + 8 (e / 2), row 2t + e % 2
        if (!whole) {
#pragma unroll
            for (int y = 0; y < G; ++y) {
                const int p1 = p0 + y * step;
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int q = p1 + g + 8 * (e >> 1);
                        const bool seen = q <= pos[i][e & 1] && q < hi && (a.window == 0 || q > pos[i][e & 1] - a.window);
                        if (!seen) sc[y][i][e] = -INFINITY;
                    }
                // a byte behind the sequence's end may be a NaN of e4m3, which a weight of 0 would not stop
#pragma unroll
                for (int n = 0; n < 4; ++n)
                    if (p1 + 2 * t + (n & 1) + 8 * (n >> 1) >= hi)
#pragma unroll
                        for (int j = 0; j < HD / 32; ++j) x[y].v[n][j] = 0;
            }
        }
        float f[G][NB][2], top[NB][2];
        bool up = false;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[i][e] = -FLT_MAX;
#pragma unroll
                for (int y = 0; y < G; ++y) {
                    f[y][i][e] = fac[i][e] * x[y].at.ks;
                    // scores in log2, V's exponent added (a position not seen and a factor 0: -inf * 0 is NaN, passed over)
                    top[i][e] = fmaxf(top[i][e], fmaf(fmaxf(sc[y][i][e], sc[y][i][2 + e]), f[y][i][e], x[y].at.lv));
                }
                up |= top[i][e] - m[i][e] > 8.f;
            }
        if (__any_sync(kFull, up)) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                float r[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float n = top[i][e];
                    n = fmaxf(n, __shfl_xor_sync(kFull, n, 4));
                    n = fmaxf(n, __shfl_xor_sync(kFull, n, 8));
                    n = fmaxf(n, __shfl_xor_sync(kFull, n, 16));
                    n = fmaxf(n, m[i][e]);
                    r[e] = kv8_exp2(m[i][e] - n);
                    m[i][e] = n;
                    l[i][e] *= r[e];
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) o[i][j][0] *= r[0], o[i][j][1] *= r[1], o[i][j][2] *= r[0], o[i][j][3] *= r[1];
            }
        }
        uint32_t pf[G][NB][PIECES][2];
#pragma unroll
        for (int y = 0; y < G; ++y)
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = kv8_exp2(fmaf(sc[y][i][e], f[y][i][e & 1], x[y].at.lv + 6.f - m[i][e & 1]));
                    if (!whole && sc[y][i][e] == -INFINITY) w[e] = 0.f;
                }
                l[i][0] = fmaf(w[0] + w[2], x[y].at.unlv, l[i][0]), l[i][1] = fmaf(w[1] + w[3], x[y].at.unlv, l[i][1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float w0 = w[2 * h] * x[y].at.mv, w1 = w[2 * h + 1] * x[y].at.mv;
                    const uint32_t z = pack_half2(w0, w1);
                    pf[y][i][0][h] = transpose8(z);
                    if constexpr (PIECES == 2) {
                        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&z));
                        pf[y][i][1][h] = transpose8(pack_half2(w0 - b.x, w1 - b.y));
                    }
                }
            }
#pragma unroll
        for (int j = 0; j < NT; j += 2)
#pragma unroll
            for (int y = 0; y < G; ++y) {
                // tiles j and j + 1 are the bytes 0, 1 and 2, 3 of word j / 2 of each V row
                const uint32_t v0 = x[y].v[0][j / 2], v1 = x[y].v[1][j / 2], v2 = x[y].v[2][j / 2], v3 = x[y].v[3][j / 2];
                uint32_t a0[2], a1[2], b0[2], b1[2];
                halves<E4M3>(__byte_perm(v0, v1, 0x5140), a0[0], a0[1]);  // byte 0 and byte 1 of rows 2t, 2t + 1
                halves<E4M3>(__byte_perm(v0, v1, 0x7362), a1[0], a1[1]);
                halves<E4M3>(__byte_perm(v2, v3, 0x5140), b0[0], b0[1]);
                halves<E4M3>(__byte_perm(v2, v3, 0x7362), b1[0], b1[1]);
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int q = PIECES - 1; q >= 0; --q) {
                        mma16816(o[i][j], a0[0], a0[1], b0[0], b0[1], pf[y][i][q]);
                        mma16816(o[i][j + 1], a1[0], a1[1], b1[0], b1[1], pf[y][i][q]);
                    }
            }
    };

    auto fetch = [&](Group &x, const Place &place, int i) {  // the warp's group i from its place in the ring
        x.at = place;
        const uint8_t *src = mine + i % D * 32 * HD;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int j = 0; j < HD / 64; ++j) x.k[n][j] = *reinterpret_cast<const uint4 *>(src + ((n * (HD / 64) + j) * 32 + lane) * 16);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const uint8_t *from = src + 16 * HD + (n * 32 + lane) * VB;
            if constexpr (HD == 64) {
                const uint2 w = *reinterpret_cast<const uint2 *>(from);
                x.v[n][0] = w.x, x.v[n][1] = w.y;
            } else {
                const uint4 w = *reinterpret_cast<const uint4 *>(from);
                x.v[n][0] = w.x, x.v[n][1] = w.y, x.v[n][2] = w.z, x.v[n][3] = w.w;
            }
        }
    };
    // The places of the groups at hand, looked up in sets of 32, of which a turn's groups are of one; the copies, fewer
    // than 32 groups ahead, may already be in the next set.
    constexpr int GR = att_groups(HD, NB);
    Place now = ahead;
    for (int used = 0; p + used * step < hi; used += GR) {
        if (used % 32 == 0) now = ahead;
        // (into the places of the groups of the last turn)
#pragma unroll
        for (int y = 0; y < GR; ++y) copy();
        cp_wait<D - GR>();
        Group x[GR];
        Place at[GR];
        bool all = true;
#pragma unroll
        for (int y = 0; y < GR; ++y) {
            at[y] = of_lane(now, used % 32 + y);
            all = all && at[y].at >= 0 && p + (used + y) * step < hi;
        }
        const int q = p + used * step;
        if (all) {
#pragma unroll
            for (int y = 0; y < GR; ++y) fetch(x[y], at[y], used + y);
            use(std::integral_constant<int, GR>{}, x, q);
        } else {
#pragma unroll 1
            for (int y = 0; y < GR; ++y) {
                const Place one = of_lane(now, used % 32 + y);
                if (one.at < 0 || q + y * step >= hi) continue;
                fetch(x[0], one, used + y);
                use(std::integral_constant<int, 1>{}, x, q + y * step);
            }
        }
    }

    // the warps' results, joined 64 elements at a time
    static_assert(att_smem(HD) >= kAttWarps * ROWS * 68 * 4, "the results lie where the ring was");
    float (*so)[ROWS][64 + 4] = reinterpret_cast<float (*)[ROWS][64 + 4]>(ring);
    __shared__ float2 sml[kAttWarps][ROWS];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l[i][e] += __shfl_xor_sync(kFull, l[i][e], 4);
            l[i][e] += __shfl_xor_sync(kFull, l[i][e], 8);
            l[i][e] += __shfl_xor_sync(kFull, l[i][e], 16);
            if (g == 0) sml[warp][8 * i + 2 * t + e] = make_float2(m[i][e], l[i][e]);
        }
    const int nrow = last - row0 + 1;
    cp_wait<0>();
    for (int d0 = 0; d0 < HD; d0 += 64) {
        __syncthreads();
        // o[j][e] is element g HD / 8 + 2 j + e / 2 of row 2t + e % 2
        const int c0 = g * (HD / 8) - d0;
        if (c0 >= 0 && c0 < 64) {
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        *reinterpret_cast<float2 *>(&so[warp][8 * i + 2 * t + e][c0 + 2 * j]) = make_float2(o[i][j][e], o[i][j][2 + e]);
        }
        __syncthreads();
        for (int u = threadIdx.x; u < nrow * 64; u += kAttWarps * 32) {
            const int r = u / 64, d = u % 64;
            float M = -FLT_MAX, L = 0.f, O = 0.f;
#pragma unroll
            for (int w = 0; w < kAttWarps; ++w) M = fmaxf(M, sml[w][r].x);
#pragma unroll
            for (int w = 0; w < kAttWarps; ++w) {
                const float f = kv8_exp2(sml[w][r].x - M);
                L = fmaf(f, sml[w][r].y, L);
                O = fmaf(f, so[w][r][d], O);
            }
            const int rr = row0 + r, tok = rr / a.group, h = head * a.group + rr - tok * a.group;
            if (a.splits == 1) {
                // no position seen: every warp's sum is 0
                static_cast<T *>(a.out)[(int64_t)(sq.start + tok) * a.out_stride + h * HD + d0 + d] =
                    kv8_from<T>(L == 0.f ? 0.f : O / L);
            } else {
                const int64_t at = ((int64_t)(sq.start + tok) * a.heads + h) * a.splits + blockIdx.x;
                a.part_o[at * HD + d0 + d] = O;
                if (d0 + d == 0) a.part_ml[at] = make_float2(M, L);
            }
        }
    }
}

// Joins the parts of one (row, query head): W warps of a block each.  Few rows have many parts (a single long sequence),
// whose loads one warp would make one after the other: 37 parts 20 us with one warp, 3 us with eight.
template <class T, int HD, int W>
__global__ void __launch_bounds__(256) k_kv8_join(const Kv8 c, const Kv8Att a) {
    constexpr int E = HD / 32;  // elements of a lane
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, s = blockIdx.z;
    const Kv8Seq sq = kv8_seq(c, s);
    const int64_t r = (int64_t)blockIdx.x * (8 / W) + warp / W;
    const bool on = r < (int64_t)sq.n * a.heads;
    const int tok = on ? (int)(r / a.heads) : 0, h = on ? (int)(r % a.heads) : 0, kvr = tok * a.group + h % a.group;
    // the span of the row's tile, as its parts were cut
    const int row0 = kvr / a.tile * a.tile, last = min(row0 + a.tile, sq.n * a.group) - 1;
    int lo, hi;
    kv8_span(sq, a.window, row0 / a.group, last / a.group, lo, hi);
    const int parts = on ? max((hi - lo + a.part - 1) / a.part, 1) : 0;
    const int64_t at = ((int64_t)(sq.start + tok) * a.heads + h) * a.splits;
    float M = -FLT_MAX, L = 0.f, O[E];
#pragma unroll
    for (int k = 0; k < E; ++k) O[k] = 0.f;
    // (what is read above was written before the attention began)
    cudaGridDependencySynchronize();
    // the warp's parts are warp % W, + W, ...; a lane weighs one in 32
    for (int i0 = warp % W; i0 < parts; i0 += 32 * W) {
        const int mine = i0 + lane * W, n = min((parts - i0 + W - 1) / W, 32);
        const float2 ml = mine < parts ? a.part_ml[at + mine] : make_float2(-FLT_MAX, 0.f);
        float top = ml.x;
        for (int k = 16; k; k >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, k));
        top = fmaxf(top, M);
        const float old = kv8_exp2(M - top), f = kv8_exp2(ml.x - top);
        M = top;
        L = fmaf(L, old, f * ml.y);
#pragma unroll
        for (int k = 0; k < E; ++k) O[k] *= old;
        const float *src = a.part_o + (at + i0) * HD + lane * E;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float w = __shfl_sync(kFull, f, i);
            float v[E];
            if constexpr (E == 4) *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(src + (int64_t)i * W * HD);
            else *reinterpret_cast<float2 *>(v) = *reinterpret_cast<const float2 *>(src + (int64_t)i * W * HD);
#pragma unroll
            for (int k = 0; k < E; ++k) O[k] = fmaf(w, v[k], O[k]);
        }
    }
    for (int k = 16; k; k >>= 1) L += __shfl_xor_sync(kFull, L, k);
    if constexpr (W > 1) {
        __shared__ float so[W][HD], sl[W], sm[W];
#pragma unroll
        for (int k = 0; k < E; ++k) so[warp][lane * E + k] = O[k];
        if (lane == 0) sl[warp] = L, sm[warp] = M;
        __syncthreads();
        if (warp > 0 || !on) return;
        for (int w = 0; w < W; ++w) M = fmaxf(M, sm[w]);
        L = 0.f;
#pragma unroll
        for (int k = 0; k < E; ++k) O[k] = 0.f;
        for (int w = 0; w < W; ++w) {
            const float f = kv8_exp2(sm[w] - M);
            L = fmaf(f, sl[w], L);
#pragma unroll
            for (int k = 0; k < E; ++k) O[k] = fmaf(f, so[w][lane * E + k], O[k]);
        }
    }
    if (!on) return;
    T v[E];
#pragma unroll
    for (int k = 0; k < E; ++k) v[k] = kv8_from<T>(L == 0.f ? 0.f : O[k] / L);
    T *out = static_cast<T *>(a.out) + (int64_t)(sq.start + tok) * a.out_stride + h * HD + lane * E;
#pragma unroll
    for (int k = 0; k < E; ++k) out[k] = v[k];
}

// --------------------------------------------------------------- host --

int esize(int type) { return type == LLMB_F32 ? 4 : 2; }

// The sizes of a cache and a batch (no pointer): LLMB_OK, and what the kernels take.
int kv8_sizes(const char *what, const llmb_kv8_cache *c, const llmb_kv8_batch *b, Kv8 &k) noexcept {
    if (!c || !b) return op_error(LLMB_ERR_ARG, "llm: %s: no cache or no batch", what);
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return op_error(LLMB_ERR_ARG, "llm: %s: blocks of %d positions (16, 32, 64 or 128)", what, c->block);
    if (c->head_dim != 64 && c->head_dim != 128)
        return op_error(LLMB_ERR_ARG, "llm: %s: head_dim %d (64 or 128)", what, c->head_dim);
    if (c->type != LLMB_KV8_INT8 && c->type != LLMB_KV8_E4M3)
        return op_error(LLMB_ERR_ARG, "llm: %s: no cache type %d", what, c->type);
    if (c->kv_heads < 1 || c->kv_heads > 4096 || c->n_blocks < 1)
        return op_error(LLMB_ERR_ARG, "llm: %s: %d blocks of %d kv heads", what, c->n_blocks, c->kv_heads);
    if (c->block_stride % 16 != 0 || c->block_stride < (int64_t)c->kv_heads * c->block * c->head_dim)
        return op_error(LLMB_ERR_ARG, "llm: %s: block_stride %lld", what, (long long)c->block_stride);
    if (b->n_seq < 1 || b->n_seq > 65535 || b->table_stride < 1 || b->n_rows < 0 || b->max_new < 0 || b->max_len < 0)
        return op_error(LLMB_ERR_ARG, "llm: %s: %d sequences, %d table entries, %d rows, max_new %d, max_len %d", what,
                        b->n_seq, b->table_stride, b->n_rows, b->max_new, b->max_len);
    const int64_t held = (int64_t)b->table_stride * c->block;
    if (held > kKv8MaxLen)
        return op_error(LLMB_ERR_ARG, "llm: %s: tables of more than 2^31 positions", what);
    k = Kv8{};
    k.bstride = c->block_stride, k.nblocks = c->n_blocks, k.block = c->block, k.kvh = c->kv_heads;
    k.bshift = c->block == 16 ? 4 : c->block == 32 ? 5 : c->block == 64 ? 6 : 7;
    k.nseq = b->n_seq, k.tstride = b->table_stride, k.nrows = b->n_rows;
    k.max_new = b->max_new > 0 && b->max_new < b->n_rows ? b->max_new : b->n_rows;
    k.cap = b->max_len > 0 && b->max_len < held ? b->max_len : (int)held;
    k.k = static_cast<uint8_t *>(c->k), k.v = static_cast<uint8_t *>(c->v);
    k.ks = c->k_scale, k.vs = c->v_scale;
    k.lens = b->lens, k.tables = b->tables, k.starts = b->starts;
    if (!b->starts) {
        if (b->n_rows % b->n_seq != 0)
            return op_error(LLMB_ERR_ARG, "llm: %s: %d rows do not divide among %d sequences", what, b->n_rows, b->n_seq);
        k.max_new = b->n_rows / b->n_seq < k.max_new ? b->n_rows / b->n_seq : k.max_new;
    }
    return LLMB_OK;
}

int kv8_rows(const char *what, int type, int64_t stride, int64_t width) noexcept {
    if (type != LLMB_F32 && type != LLMB_F16 && type != LLMB_BF16)
        return op_error(LLMB_ERR_ARG, "llm: %s: no type %d", what, type);
    if (stride < width || stride * esize(type) % 16 != 0)
        return op_error(LLMB_ERR_ARG, "llm: %s: rows %lld elements apart (at least %lld, a multiple of 16 bytes)", what,
                        (long long)stride, (long long)width);
    return LLMB_OK;
}

int kv8_pointers(const char *what, int *device, const Kv8 &c, const void *x, const char *nx, const void *y,
                 const char *ny, bool optional) noexcept {
    const std::initializer_list<OpPointer> ps = {
        {c.k, "cache k", 16, false},     {c.v, "cache v", 16, false},   {c.ks, "k_scale", 4, false},
        {c.vs, "v_scale", 4, false},     {c.lens, "lens", 4, false},    {c.tables, "tables", 4, false},
        {c.starts, "starts", 4, true},   {x, nx, 16, optional},         {y, ny, 16, optional}};
    int rc = op_alignment(what, ps);
    if (rc == LLMB_OK) rc = op_device(what, device);
    if (rc == LLMB_OK) rc = op_pointers(what, *device, ps);
    return rc;
}

// Blocks that n consecutive positions can touch.
int64_t touched(const Kv8 &c) { return ((int64_t)c.max_new + c.block - 2) / c.block + 1; }

template <class F>
void by_type(int type, F &&f) {
    if (type == LLMB_F32) f(float{});
    else if (type == LLMB_F16) f(__half{});
    else f(__nv_bfloat16{});
}

struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };

template <class F>
void by_cache(int type, int hd, F &&f) {
    if (type == LLMB_KV8_E4M3) hd == 64 ? f(Yes{}, std::integral_constant<int, 64>{}) : f(Yes{}, std::integral_constant<int, 128>{});
    else hd == 64 ? f(No{}, std::integral_constant<int, 64>{}) : f(No{}, std::integral_constant<int, 128>{});
}

template <class T, bool E4M3, int HD, int NB>
cudaError_t attend_launch(const Kv8 &c, const Kv8Att &a, dim3 grid, int device, cudaStream_t st) noexcept {
    const cudaError_t e = op_shared<k_kv8_attend<T, E4M3, HD, NB>>(device, att_smem(HD));
    if (e == cudaSuccess) k_kv8_attend<T, E4M3, HD, NB><<<grid, kAttWarps * 32, att_smem(HD), st>>>(c, a);
    return e;
}

// How the attention cuts its work: rows into tiles, a tile's positions into parts.
struct Cut {
    bool chunk;  // by the kernel for many rows
    int tile, tiles, splits, part;
};

// Parts of the kernel for many rows: one CTA takes an SM, so with `units` CTAs of one part each the last wave may be
// nearly empty; parts fill it, at the price of the join.  Measured on a B200: a step of 128 positions 3 us, a CTA's start
// 4 us, the join 3 us and its traffic at 4 TB/s.
double join_us(int64_t slots, int hd) { return (double)slots * hd * 8 / 4e6; }  // for each part

// No more parts than these can be the least time.  s parts take units s / 148 waves or more, of steps / s steps or more, one
// takes less than units / 148 + 1: s parts gain less than 3 steps + 4 - 4 (s - 1) units / 148, and their join costs 3 + s join_us.
int chunk_most_parts(int64_t units, int64_t span, int64_t slots, int hd) {
    const double steps = (double)((span + 127) / 128), wave = 4.0 * (double)units / 148;
    return (int)std::max(std::min({(3 * steps + 1 + wave) / (wave + join_us(slots, hd)), steps, 64.0}), 1.0);
}

int chunk_parts(int64_t units, int64_t span, int64_t slots, int hd) {
    const int64_t steps = (span + 127) / 128;
    const int most = chunk_most_parts(units, span, slots, hd);
    int best = 1;
    double least = 0;
    for (int s = 1; s <= most; ++s) {
        const double waves = (double)((units * s + 147) / 148);
        const double us = waves * (3.0 * (double)((steps + s - 1) / s) + 4.0) + (s > 1 ? 3.0 + s * join_us(slots, hd) : 0.0);
        if (s == 1 || us < least) least = us, best = s;
    }
    return best;
}

// Parts of the kernel for few rows: enough for four CTAs an SM, of 128 positions or more.  Measured on a B200 (us): 64
// sequences of up to 2048 with 148, 296, 444, 592, 1184 CTAs in all 21.8, 19.3, 19.0, 16.8, 21.2; one of 2048 with parts of
// 128, 256, 512: 6.6, 7.7, 9.1.
int64_t attend_parts(const Kv8 &c, int64_t units, int64_t span) {
    if (span < 512) return 1;  // (300 positions: 5.3 us, in two parts 7.1)
    // (one token of sequences of any lengths: rather more than a wave; a chunk's tiles are alike: rather less)
    const int64_t fill = c.max_new > 1 ? std::max<int64_t>(4 * 148 / units, 1) : (4 * 148 + units - 1) / units;
    return std::min<int64_t>({fill, span / 128, 128});
}

// The same for float32 rows too: a warp sums every 4th group of 16 positions, and the tensor cores cut sums off towards 0
// (about 1e-8 a step), so their results are joined from parts of at most 1024 positions.
int64_t few_parts(const Kv8 &c, int64_t units, int64_t span, int type) {
    const int64_t want = attend_parts(c, units, span);
    return type == LLMB_F32 ? std::max<int64_t>(want, (span + 1023) / 1024) : want;
}

// Whether the kernel for many rows takes the call.  It starts slower and does more for each byte of the cache: below about
// 2 million (row, query head, position) of 64 elements the kernel for few rows is faster, 2.5 million where rows are two
// pieces and its tiles 8 rows (B200, us, few / many rows; bfloat16: 1.3 M 14.5 / 16.5, 1.8 M 15.9 / 15.6, 2.2 M 19.0 / 15.3;
// float32: 1.8 M 16.2 / 17.0, 2.2 M 16.5 / 17.7 and 17.0 / 21.3, 2.6 M 24.1 / 19.6).  A tile of 128 rows with few of them
// is no gain: a decoding step stays with the other.
constexpr double few_work(int type) { return type == LLMB_BF16 ? 2e6 : 2.5e6; }

bool many_rows(const Kv8 &c, int heads, int hd, int type, int window) {
    const int64_t seen = window > 0 ? std::min<int64_t>(c.cap, (int64_t)window + c.max_new) : c.cap;
    return (int64_t)c.max_new * (heads / c.kvh) > 32 && (double)c.nrows * heads * (double)seen * (hd / 64) > few_work(type);
}

int few_tile(int64_t rows, int type) { return type == LLMB_BF16 && rows > 8 ? 16 : 8; }

Cut attention_cut(const Kv8 &c, int heads, int hd, int type, int window) {
    Cut k{};
    const int group = heads / c.kvh;
    const int64_t rows = (int64_t)c.max_new * group;
    k.chunk = many_rows(c, heads, hd, type, window);
    const int tile = k.chunk ? kv8_chunk_rows(type == LLMB_F32, hd) : few_tile(rows, type);
    k.tile = tile;
    k.tiles = (int)((rows + tile - 1) / tile);
    // the most positions that a tile's rows see between them
    auto span_of = [&](int w) -> int64_t {
        if (w <= 0 || w >= c.cap) return c.cap;
        const int64_t tokens = std::min<int64_t>(c.max_new, (tile + group - 2) / group + 1);
        return std::min<int64_t>(c.cap, (int64_t)w + tokens + 15);
    };
    const int64_t units = (int64_t)c.nseq * c.kvh * std::max(k.tiles, 1);
    const int64_t span = span_of(window);
    const int64_t want = k.chunk ? chunk_parts(units, span, (int64_t)c.nrows * heads, hd) : few_parts(c, units, span, type);
    k.part = (int)((span + want - 1) / want + 127) / 128 * 128;
    k.splits = std::max((int)((span + k.part - 1) / k.part), 1);
    return k;
}

// The most parts that any type and window give, by either kernel: what the workspace has room for.  Fewer positions are never
// cut into more parts, and more work never leaves the kernel for many rows.
int64_t most_parts(const Kv8 &c, int heads, int hd) {
    const int64_t rows = (int64_t)c.max_new * (heads / c.kvh);
    auto units = [&](int tile) { return (int64_t)c.nseq * c.kvh * std::max<int64_t>((rows + tile - 1) / tile, 1); };
    int64_t most = 1;
    for (int type : {LLMB_F32, LLMB_BF16}) {  // (float16 has the tiles and rules of one or the other)
        int64_t span = c.cap;
        if (many_rows(c, heads, hd, type, 0)) {
            for (bool f32 : {false, true})
                most = std::max<int64_t>(most, chunk_most_parts(units(kv8_chunk_rows(f32, hd)), c.cap, (int64_t)c.nrows * heads, hd));
            // the kernel for few rows is left windows with so little work: positions a tile sees, 15 more for a start within 16
            span = std::min<int64_t>(span, (int64_t)(few_work(type) / ((double)c.nrows * heads * (hd / 64))) + 15);
        }
        most = std::max(most, few_parts(c, units(few_tile(rows, type)), span, type));
    }
    return most;
}

}  // namespace
}  // namespace llmb

using namespace llmb;

extern "C" {

int llmb_kv8_append(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, const void *k, const void *v, int type,
                    int64_t row_stride, void *stream) {
    const char *what = "kv8_append";
    Kv8 c;
    int rc = kv8_sizes(what, cache, batch, c);
    if (rc == LLMB_OK) rc = kv8_rows(what, type, row_stride, (int64_t)c.kvh * cache->head_dim);
    int dev = 0;
    if (rc == LLMB_OK) rc = kv8_pointers(what, &dev, c, k, "k", v, "v", c.nrows == 0);
    if (rc != LLMB_OK) return rc;
    if (c.max_new == 0) return LLMB_OK;
    by_type(type, [&](auto t) {
        by_cache(cache->type, cache->head_dim, [&](auto e4m3, auto hd) {
            append_launch<decltype(t), decltype(e4m3)::value, decltype(hd)::value>(
                c, k, v, row_stride, (int)touched(c), static_cast<cudaStream_t>(stream));
        });
    });
    return op_launched(what);
}

int llmb_kv8_read(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, void *k, void *v, int type,
                  int64_t row_stride, void *stream) {
    const char *what = "kv8_read";
    Kv8 c;
    int rc = kv8_sizes(what, cache, batch, c);
    if (rc == LLMB_OK) rc = kv8_rows(what, type, row_stride, (int64_t)c.kvh * cache->head_dim);
    int dev = 0;
    if (rc == LLMB_OK) rc = kv8_pointers(what, &dev, c, k, "k", v, "v", true);
    if (rc != LLMB_OK) return rc;
    if (c.max_new == 0 || (!k && !v)) return LLMB_OK;
    by_type(type, [&](auto t) {
        by_cache(cache->type, cache->head_dim, [&](auto e4m3, auto hd) {
            using T = decltype(t);
            const int tiles = tiles_each(c, touched(c), c.block * decltype(hd)::value * (int)sizeof(T));
            k_kv8_read<T, decltype(e4m3)::value, decltype(hd)::value>
                <<<dim3((unsigned)touched(c), (2 * c.kvh + tiles - 1) / tiles, c.nseq), 256, 0, static_cast<cudaStream_t>(stream)>>>(
                    c, static_cast<T *>(k), static_cast<T *>(v), row_stride, tiles);
        });
    });
    return op_launched(what);
}

int64_t llmb_kv8_attention_workspace(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, int heads) {
    Kv8 c;
    if (kv8_sizes("kv8_attention_workspace", cache, batch, c) != LLMB_OK) return -1;
    if (heads < 1 || heads % c.kvh != 0 || heads / c.kvh > kKv8MaxGroup) {
        op_error(LLMB_ERR_ARG, "llm: kv8_attention_workspace: %d heads on %d kv heads", heads, c.kvh);
        return -1;
    }
    const int64_t splits = most_parts(c, heads, cache->head_dim);
    return splits == 1 ? 0 : (int64_t)c.nrows * heads * splits * (8 + 4 * (int64_t)cache->head_dim);
}

int llmb_kv8_attention(const llmb_kv8_cache *cache, const llmb_kv8_batch *batch, const void *q, int64_t q_stride,
                       void *out, int64_t out_stride, int type, int heads, float scale, int window, void *workspace,
                       int64_t workspace_bytes, void *stream) {
    const char *what = "kv8_attention";
    Kv8 c;
    int rc = kv8_sizes(what, cache, batch, c);
    if (rc != LLMB_OK) return rc;
    const int hd = cache->head_dim;
    if (heads < 1 || heads % c.kvh != 0 || heads / c.kvh > kKv8MaxGroup)
        return op_error(LLMB_ERR_ARG, "llm: %s: %d heads on %d kv heads", what, heads, c.kvh);
    if (window < 0 || !(scale >= 0.f && scale <= FLT_MAX))
        return op_error(LLMB_ERR_ARG, "llm: %s: window %d, scale %g", what, window, (double)scale);
    if ((rc = kv8_rows(what, type, q_stride, (int64_t)heads * hd)) != LLMB_OK) return rc;
    if ((rc = kv8_rows(what, type, out_stride, (int64_t)heads * hd)) != LLMB_OK) return rc;
    if (out == q && c.nrows > 1 && out_stride != q_stride)
        return op_error(LLMB_ERR_ARG, "llm: %s: out is q with another stride", what);
    Kv8Att a{};
    const Cut cut = attention_cut(c, heads, hd, type, window);
    if ((int64_t)c.kvh * cut.tiles > 65535 || (int64_t)c.max_new * heads > INT32_MAX)
        return op_error(LLMB_ERR_ARG, "llm: %s: %d rows of a sequence are too many", what, c.max_new);
    const int64_t slots = c.max_new > 0 && cut.splits > 1 ? (int64_t)c.nrows * heads * cut.splits : 0;
    const std::initializer_list<OpPointer> ws = {{workspace, "workspace", 16, slots == 0}};
    if (slots > 0) {
        if ((rc = op_alignment(what, ws)) != LLMB_OK) return rc;
        if (workspace_bytes < slots * (8 + 4 * (int64_t)hd))
            return op_error(LLMB_ERR_ARG, "llm: %s: a workspace of %lld bytes, not %lld", what, (long long)workspace_bytes,
                            (long long)(slots * (8 + 4 * (int64_t)hd)));
        a.part_o = static_cast<float *>(workspace);
        a.part_ml = reinterpret_cast<float2 *>(a.part_o + slots * hd);
    }
    int dev = 0;
    if ((rc = kv8_pointers(what, &dev, c, q, "q", out, "out", c.nrows == 0)) != LLMB_OK) return rc;
    if (slots > 0 && (rc = op_pointers(what, dev, ws)) != LLMB_OK) return rc;
    if (c.max_new == 0) return LLMB_OK;
    a.q = q, a.out = out, a.q_stride = q_stride, a.out_stride = out_stride;
    a.heads = heads, a.group = heads / c.kvh, a.window = window;
    a.scale = (float)((scale != 0.f ? (double)scale : 1.0 / std::sqrt((double)hd)) * 1.4426950408889634);
    a.tile = cut.tile, a.splits = cut.splits, a.part = cut.part;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(cut.splits, c.kvh * cut.tiles, c.nseq);
    cudaError_t e = cudaSuccess;
    if (cut.chunk) e = kv8_chunk_launch(type, cache->type == LLMB_KV8_E4M3, hd, c, a, grid, dev, st);
    else by_type(type, [&](auto t) {
        by_cache(cache->type, hd, [&](auto e4m3, auto d) {
            using T = decltype(t);
            constexpr int HD = decltype(d)::value;
            constexpr bool E4 = decltype(e4m3)::value;
            if constexpr (kPieces<T> == 1) {
                if (cut.tile == 16) {
                    e = attend_launch<T, E4, HD, 2>(c, a, grid, dev, st);
                    return;
                }
            }
            e = attend_launch<T, E4, HD, 1>(c, a, grid, dev, st);
        });
    });
    if (e != cudaSuccess) {
        cudaGetLastError();
        return op_error(LLMB_ERR_CUDA, "llm: %s: %s", what, cudaGetErrorString(e));
    }
    if ((rc = op_launched(what)) != LLMB_OK || cut.splits == 1) return rc;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    const bool many = cut.splits > 8;
    cfg.gridDim = dim3((unsigned)(many ? (int64_t)c.max_new * heads : ((int64_t)c.max_new * heads + 7) / 8), 1, c.nseq);
    cfg.blockDim = dim3(256);
    cfg.stream = st, cfg.attrs = &attr, cfg.numAttrs = 1;
    by_type(type, [&](auto t) {
        using T = decltype(t);
        if (hd == 64) many ? cudaLaunchKernelEx(&cfg, k_kv8_join<T, 64, 8>, c, a) : cudaLaunchKernelEx(&cfg, k_kv8_join<T, 64, 1>, c, a);
        else many ? cudaLaunchKernelEx(&cfg, k_kv8_join<T, 128, 8>, c, a) : cudaLaunchKernelEx(&cfg, k_kv8_join<T, 128, 1>, c, a);
    });
    return op_launched(what);
}

}  // extern "C"
