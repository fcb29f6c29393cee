// The attention for many rows (kv8_chunk.cu).
#pragma once

#include "../../include/llm_b200.h"
#include "kv8.hpp"

namespace llmb {

// Rows of a CTA: two tiles of 128, or one where float32 results take their space in tensor memory.
__host__ __device__ constexpr int kv8_chunk_rows(bool f32, int hd) { return f32 && hd == 128 ? 128 : 256; }

// grid: (parts, kv heads * tiles, sequences), as for the kernel for few rows.
cudaError_t kv8_chunk_launch(int type, bool e4m3, int hd, const Kv8 &c, const Kv8Att &a, dim3 grid, int device,
                             cudaStream_t st) noexcept;

}  // namespace llmb
