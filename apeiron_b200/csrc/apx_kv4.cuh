// apx_kv4.cuh — the 4-bit KV cache's tile, shared by the kernels that write it (apx_rope.cu) and
// read it (apx_attn.cu, apx_attn_tc.cu), and what the two attention kernels share.
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
// Cached tokens of a sequence at most: a step of keys past them still has its number in an int.
constexpr int kMaxKvLen = INT32_MAX - 511;

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

#ifdef __CUDACC__

// One attention call, as both kernels take it.
struct AttnArgs {
  const void *q;
  void *out;
  const uint8_t *pages;
  const int *cu, *kv_len, *table;
  unsigned long long *status;
  unsigned long long ldq, ldo;
  unsigned long long page_bytes;
  float *part;      // apx_attn.cu: two partial items per CTA
  unsigned *count;  // apx_attn.cu: CTAs that have arrived at an item (zero between calls)
  int n_pages, n_seqs, max_pages, kv_heads, group, page_shift;
  int window, sinks, type, n_tokens, max_q;
  unsigned group_mul;  // 2^32 / group + 1, for by_group
  float scale;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// The constants of the unpacking, held in registers: what the compiler does not see through it
// does not build again at every use.
struct Unpack {
  uint32_t magic, sixteenth, minus72;
  __device__ __forceinline__ Unpack() {
    asm volatile("mov.u32 %0, 0x64006400;" : "=r"(magic));
    asm volatile("mov.u32 %0, 0x2C002C00;" : "=r"(sixteenth));
    asm volatile("mov.u32 %0, 0xD480D480;" : "=r"(minus72));
  }
  // Two codes of x (bits 0-3 and 16-19, or 4-7 and 20-23) as (c - 8) * s: the bits behind 0x6400
  // read 1024 + c, or 1024 + 16 c.
  __device__ __forceinline__ uint32_t low2(uint32_t x, __half2 s) const {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(v) : "r"(x), "r"(magic));
    return h2u(__hmul2(__hsub2(u2h(v), u2h(0x64086408u)), s));
  }
  __device__ __forceinline__ uint32_t high2(uint32_t x, __half2 s) const {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(v) : "r"(x), "r"(magic));
    return h2u(__hmul2(__hfma2(u2h(v), u2h(sixteenth), u2h(minus72)), s));
  }
};

__device__ __forceinline__ void attn_refuse(const AttnArgs &p, int seq, int code) {
  if (p.status)
    atomicMin(p.status, (unsigned long long)seq << 24 | (unsigned long long)code << 16);
}

// r / group for 0 <= r < 2^31: the product's high word is the quotient or one more.
__host__ __device__ __forceinline__ int by_group(const AttnArgs &p, int r) {
  if (p.group == 1) return r;
  const unsigned q = (unsigned)((unsigned long long)(unsigned)r * p.group_mul >> 32);
  return (int)(q - (q * (unsigned)p.group > (unsigned)r ? 1u : 0u));
}

// The first key of the window of the query at `pos`, which may stand before token 0.
__host__ __device__ __forceinline__ int window_start(const AttnArgs &p, int pos) {
  return p.window == 0 || pos < p.window ? 0 : pos - p.window + 1;
}

// Whether the n keys from `key` on are all behind every window that starts at `low` or later.
__host__ __device__ __forceinline__ bool unseen(const AttnArgs &p, int key, int n, int low) {
  return key + n <= low && key >= p.sinks;
}

// A power of two that brings a row's largest |q| to [2^9, 2^10) (exponents outside the f32
// normals are clamped), as its exponent's distance: q 2^(9 - e).
__device__ __forceinline__ int row_exponent(float top) {
  return min(max((int)(__float_as_uint(top) >> 23 & 255), 32), 254) - 127;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// A sequence's query rows (token, head of the group) in blocks of R, and the keys each sees, in
// steps of KEYS.
template <int R, int KEYS>
struct SeqRows {
  int first, rows, kv, p0, nblk;  // first query token, rows, usable keys, position of row 0
  bool bad;  // lengths outside the batch or the cache, or more query tokens than the launch is for

  __host__ __device__ void load(const AttnArgs &p, int s) {
    const int a = p.cu[s], b = p.cu[s + 1], n = p.kv_len[s];
    const long long room = (long long)p.max_pages << p.page_shift;
    bad = a < 0 || b < a || b > p.n_tokens || b - a > p.max_q || n < 0 || n > room ||
          n > kMaxKvLen;
    first = a;
    rows = bad ? 0 : (b - a) * p.group;
    kv = bad ? 0 : n;
    p0 = n - (b - a);
    nblk = (rows + R - 1) / R;
  }
  __host__ __device__ static int steps_to(int n) { return (max(n, 0) + KEYS - 1) / KEYS; }
  // Block b sees keys below `end`: those of the sinks' steps [0, sink) and of steps low / KEYS on;
  // of these none from the sinks' end up to `low`, whose pages may be gone (unseen).
  __host__ __device__ void range(const AttnArgs &p, int b, int &end, int &sink, int &low) const {
    const int lo = p0 + by_group(p, b * R), hi = p0 + by_group(p, min((b + 1) * R - 1, rows - 1));
    end = max(min(kv, hi + 1), 0);
    low = window_start(p, lo);
    sink = p.window ? min(steps_to(min(p.sinks, end)), low / KEYS) : 0;
  }
};

#endif  // __CUDACC__

}  // namespace apx
