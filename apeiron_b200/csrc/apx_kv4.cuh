// apx_kv4.cuh — the 4-bit KV cache's tile and the batch's positions, shared by the kernels that
// write it (apx_rope.cu) and read it (apx_attn.cu).
//
// A tile is 16 tokens of one KV head (layout in include/apeiron_cuda.h): K codes, V codes, K
// scales, V scales; page_tokens / 16 tiles follow each other in a page.
#pragma once

#include <cuda_fp16.h>

#include <cstddef>
#include <cstdint>

#include "../../include/apeiron_cuda.h"

namespace apx {

constexpr int kKvTile = 16;   // tokens of a tile
constexpr int kKvGroup = 32;  // dims that share a scale

__host__ __device__ constexpr int kv4_tile_bytes(int dim) {
  return kKvTile * dim + 2 * kKvTile * (dim / kKvGroup) * 2;
}
// Offsets inside a tile of head dim `dim`.
__host__ __device__ constexpr int kv4_v_off(int dim) { return kKvTile * dim / 2; }
__host__ __device__ constexpr int kv4_ks_off(int dim) { return kKvTile * dim; }
__host__ __device__ constexpr int kv4_vs_off(int dim) {
  return kKvTile * dim + kKvTile * (dim / kKvGroup) * 2;
}
// The byte of V's codes that holds token r's dim i (low nibble when i % 16 < 8).
__host__ __device__ constexpr int kv4_v_byte(int i, int r) {
  const int m = i / 16, g = i % 8, t = (r % 8) / 2;
  return 4 * (((m / 4) * 32 + g * 4 + t) * 4 + m % 4) + (r % 2) * 2 + r / 8;
}

}  // namespace apx
