// The 8-bit key/value cache on the device: what its kernels (kv8.cu,
// kv8_chunk.cu) share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace llmb {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kKv8MaxLen = 0x7fffffff - 16384;  // sums of positions and a block, a step or a set of them stay below 2^31

// The cache and the batch of a call as the kernels take them (include/llm_b200.h describes the fields).
struct Kv8 {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t bstride;
    const int *lens, *tables, *starts;
    int nblocks, block, bshift, kvh;  // block = 1 << bshift
    int nseq, tstride, nrows, max_new, cap;  // cap: the most positions a sequence can have here
};

// A sequence's share of the call: rows start .. start + n - 1 are its positions first .. first + n - 1 (below 0 for the
// first rows of one that has more rows than positions: they have none); it sees positions below len.
struct Kv8Seq {
    int start, n, len, first;
};

// Read from device memory and clamped, so that no value there leads outside the buffers.
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8 &c, int s) {
    Kv8Seq q;
    int a, b;
    if (c.starts) {
        a = min(max(__ldg(c.starts + s), 0), c.nrows);
        b = min(max(__ldg(c.starts + s + 1), a), c.nrows);
    } else {
        const int per = c.nrows / c.nseq;
        a = s * per, b = a + per;
    }
    const int len = min(max(__ldg(c.lens + s), 0), kKv8MaxLen);
    q.start = a;
    q.n = min(b - a, c.max_new);
    q.len = min(len, c.cap);
    q.first = len - (b - a);
    return q;
}

// The block of a sequence's j-th table entry, or -1 where the pool has no such block.
__device__ __forceinline__ int kv8_block(const Kv8 &c, int s, int j) {
    if (j < 0 || j >= c.tstride) return -1;
    const int b = __ldg(c.tables + (int64_t)s * c.tstride + j);
    return b >= 0 && b < c.nblocks ? b : -1;
}

template <class T>
__device__ __forceinline__ float kv8_float(T x);
template <>
__device__ __forceinline__ float kv8_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float kv8_float<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float kv8_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T>
__device__ __forceinline__ T kv8_from(float x);
template <>
__device__ __forceinline__ float kv8_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half kv8_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 kv8_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Two 8-bit values as float16, exactly.  w holds them in its bytes 0 and 2
// (E4M3: times 2^-8, and bytes that are NaN come out finite, so that no byte
// of a masked position can make a product NaN).
//   int8: the byte with its sign bit flipped, u = q + 128, in the low bits of
//   1024.0 reads 1024 + u; minus 1152 is q.
//   e4m3: its 4 exponent and 3 mantissa bits one bit below float16's
//   exponent top read the value times 2^(7 - 15), subnormals included.
template <bool E4M3>
__device__ __forceinline__ uint32_t kv8_half2(uint32_t w) {
    if (E4M3) return ((w & 0x00800080u) << 8) | ((w & 0x007f007fu) << 7);
    const uint32_t h = (w ^ 0x00800080u) | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&h), __half2half2(__float2half_rn(1152.f)));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <bool E4M3>
__host__ __device__ constexpr float kv8_unit() { return E4M3 ? 256.f : 1.f; }  // what kv8_half2's values are to be multiplied by

// Four 8-bit values (the bytes of w) as float, exactly.
template <bool E4M3>
__device__ __forceinline__ void kv8_floats(uint32_t w, float (&f)[4]) {
    const uint32_t a = kv8_half2<E4M3>(__byte_perm(w, 0, 0x4140)), b = kv8_half2<E4M3>(__byte_perm(w, 0, 0x4342));
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&a));
    const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&b));
    constexpr float u = kv8_unit<E4M3>();
    f[0] = x.x * u, f[1] = x.y * u, f[2] = y.x * u, f[3] = y.y * u;
}

__device__ __forceinline__ float kv8_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The power of two that brings a query row whose largest magnitude has the bits m to [2^14, 2^15) (rows below 2^-100 by
// the factor of 2^-100), and its inverse; false where the row is not finite (up is 0 then).
__device__ __forceinline__ bool kv8_query_scale(uint32_t m, float &up, float &down) {
    const bool fine = m < 0x7f800000u;
    const int ex = m == 0 ? 0 : max((int)(m >> 23) - 127, -100);
    up = fine ? __uint_as_float((uint32_t)(127 + 14 - ex) << 23) : 0.f;
    down = __uint_as_float((uint32_t)(127 - 14 + (fine ? ex : 0)) << 23);
    return fine;
}

// V's scale as mv 2^ex, for the whole warp, a group of positions a lane.  For every scale that append makes but 0 (2^-109 to
// 2^121) mv is in [1, 2), or down to 2^-8 at the least ones: 2^-ex times the largest weight (2^6) must leave the sum of 2^21
// positions finite, and weights times 2^-8 still have their 22 bits.  A group whose scale is 0 or smaller than those counts
// in the softmax's sum, and its weights' size must not hide those of values that are not 0 (float16 ends 2^31 below the
// largest): it takes the least exponent of the walk so far (low), or before the walk has one kKv8ZeroExp, from which any up
// to 2^60 that is met later is in reach.
constexpr int kKv8LeastScale = -109, kKv8LeastExp = -101, kKv8ZeroExp = -64, kKv8NoExp = 0x7fffffff;
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int kv8_v_scale(float vs, float &mv, int &low) {
    const uint32_t u = __float_as_uint(vs) & 0x7fffffffu;
    const bool has = u >= (uint32_t)(127 + kKv8LeastScale) << 23 && u < 0x7f800000u;
    int ex = has ? min(max((int)(u >> 23) - 127, kKv8LeastExp), 126) : kKv8NoExp;
    low = min(low, __reduce_min_sync(kFull, ex));
    if (!has) ex = low == kKv8NoExp ? kKv8ZeroExp : low;
    mv = vs * kv8_pow2(-ex);
    return ex;
}

constexpr int kKv8MaxGroup = 64;  // query heads of one kv head

// ---- the attention's split of positions, as both its kernels see it

// One call's sizes.  Rows of one kv head are its tokens' query heads: row r
// of a sequence is query head r % group of token r / group.
struct Kv8Att {
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    int heads, group;
    float scale;  // times log2(e)
    int window;   // 0: none
    int tile;     // rows of a tile
    int splits;   // parts that a tile's positions are cut into at most
    int part;     // positions of one part
    float2 *part_ml;  // [rows][heads][splits]: maximum (log2) and sum
    float *part_o;    // [rows][heads][splits][head_dim]
};

// The first position that a row at position pos sees (pos may be below 0, and the window the largest integer).
__device__ __forceinline__ int kv8_first_seen(int pos, int window) { return window > 0 && pos >= window ? pos - window + 1 : 0; }

// Positions [lo, hi) that the tokens t0 .. t1 (inclusive) of a sequence see between them; lo a multiple of 16.
__device__ __forceinline__ void kv8_span(const Kv8Seq &q, int window, int t0, int t1, int &lo, int &hi) {
    hi = max(min(q.first + t1 + 1, q.len), 0);
    lo = kv8_first_seen(q.first + t0, window) & ~15;
    if (lo > hi) lo = hi;
}

}  // namespace llmb
