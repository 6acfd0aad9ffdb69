// apx_attn.cu — attention over the paged 4-bit cache (layout: apx_kv4.cuh).
//
// out_i = sum_j p_ij v_j, p = softmax over the visible keys of scale q_i.k_j, in one pass over
// the keys with a running maximum m and sum l: a chunk of keys with scores s_j turns (m, l, o)
// into m' = max(m, max s_j), l' = l e^(m-m') + sum e^(s_j-m'), o' = o e^(m-m') + sum e^(s_j-m') v_j.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "apx_common.cuh"
#include "apx_kv4.cuh"
#include "apx_step.h"

namespace apx {

struct AttnArgs {
  apx_attn_args a;
  const int *cu, *kv_len, *table;
  const uint8_t *pages;
  size_t n_pages, page_bytes;
  int n_seqs, max_pages, kv_heads, group, dim, page_tokens;
};

__device__ __forceinline__ float load_q(const void *q, size_t i, int type) {
  if (type == APX_DTYPE_F32) return static_cast<const float *>(q)[i];
  if (type == APX_DTYPE_F16) return __half2float(static_cast<const __half *>(q)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(q)[i]);
}

// One query row (token, head) per CTA of 128 threads, 128 keys at a time: thread j scores key
// j, then thread i gathers output dim i.
__global__ void __launch_bounds__(128) attn_row_kernel(AttnArgs p) {
  __shared__ float s_q[128], s_p[128], s_red[4];
  const int t = blockIdx.x, head = blockIdx.y, h = head / p.group, tid = threadIdx.x;
  int lo = 0, hi = p.n_seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (p.cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  const long long room = (long long)p.max_pages * p.page_tokens;
  const int kv = (int)min((long long)p.kv_len[lo], room);
  if (p.kv_len[lo] > room && tid == 0 && p.a.d_status)
    atomicMin(&p.a.d_status->first,
              (unsigned long long)lo << 24 | (unsigned long long)APX_ERR_INVALID_ARGUMENT << 16);
  const int pos = p.kv_len[lo] - p.cu[lo + 1] + t;
  const int end = min(pos + 1, kv);
  if (tid < p.dim) s_q[tid] = load_q(p.a.d_q, (size_t)t * p.a.ldq + (size_t)head * p.dim + tid, p.a.type);
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  const int tb = kv4_tile_bytes(p.dim);
  auto tile_of = [&](int j) -> const uint8_t * {
    const int page = p.table[(size_t)lo * p.max_pages + j / p.page_tokens];
    if (page < 0 || (size_t)page >= p.n_pages) return nullptr;
    return p.pages + ((size_t)page * p.kv_heads + h) * p.page_bytes +
           (size_t)(j % p.page_tokens / kKvTile) * tb;
  };
  for (int j0 = 0; j0 < end; j0 += 128) {
    if (p.a.window && j0 >= p.a.sinks && j0 + 127 <= pos - p.a.window) continue;
    const int j = j0 + tid;
    const bool seen = j < end && (!p.a.window || j < p.a.sinks || j > pos - p.a.window);
    float s = -INFINITY;
    if (seen) {
      const uint8_t *tile = tile_of(j);
      if (!tile) {
        if (p.a.d_status)
          atomicMin(&p.a.d_status->first, (unsigned long long)lo << 24 |
                                              (unsigned long long)APX_ERR_INVALID_ARGUMENT << 16);
      } else {
        const int r = j % kKvTile;
        const __half *ks = reinterpret_cast<const __half *>(tile + kv4_ks_off(p.dim));
        s = 0.0f;
        for (int g = 0; g < p.dim / kKvGroup; g++) {
          float dot = 0.0f;
          for (int i = 0; i < kKvGroup / 2; i++) {
            const unsigned b = tile[r * (p.dim / 2) + g * (kKvGroup / 2) + i];
            dot = fmaf((float)((int)(b & 15) - 8), s_q[g * kKvGroup + 2 * i], dot);
            dot = fmaf((float)((int)(b >> 4) - 8), s_q[g * kKvGroup + 2 * i + 1], dot);
          }
          s = fmaf(dot, __half2float(ks[g * kKvTile + r]), s);
        }
        s *= p.a.scale;
      }
    }
    float top = s;
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
    if (tid % 32 == 0) s_red[tid / 32] = top;
    __syncthreads();
    top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    __syncthreads();
    if (top == -INFINITY) continue;
    const float mn = fmaxf(m, top), keep = m == -INFINITY ? 0.0f : expf(m - mn);
    const float e = s == -INFINITY ? 0.0f : expf(s - mn);
    s_p[tid] = e;
    float sum = e;
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
    if (tid % 32 == 0) s_red[tid / 32] = sum;
    __syncthreads();
    l = l * keep + (s_red[0] + s_red[1] + s_red[2] + s_red[3]);
    m = mn;
    if (tid < p.dim) {
      float acc = 0.0f;
      for (int k = 0; k < 128 && j0 + k < end; k++) {
        if (s_p[k] == 0.0f) continue;  // masked keys may hold anything
        const uint8_t *tile = tile_of(j0 + k);
        if (!tile) continue;
        const int r = (j0 + k) % kKvTile;
        const unsigned b = tile[kv4_v_off(p.dim) + kv4_v_byte(tid, r)];
        const int c = (int)(tid % 16 < 8 ? b & 15 : b >> 4) - 8;
        const __half *vs = reinterpret_cast<const __half *>(tile + kv4_vs_off(p.dim));
        acc = fmaf(s_p[k], (float)c * __half2float(vs[tid / kKvGroup * kKvTile + r]), acc);
      }
      o = o * keep + acc;
    }
    __syncthreads();
  }
  if (tid < p.dim) {
    const float y = l > 0.0f ? o / l : 0.0f;
    const size_t at = (size_t)t * p.a.ldo + (size_t)head * p.dim + tid;
    if (p.a.type == APX_DTYPE_F32) static_cast<float *>(p.a.d_out)[at] = y;
    else if (p.a.type == APX_DTYPE_F16) static_cast<__half *>(p.a.d_out)[at] = __float2half_rn(y);
    else static_cast<__nv_bfloat16 *>(p.a.d_out)[at] = __float2bfloat16_rn(y);
  }
}

cudaError_t launch_attn_kv4(const apx_attn_args &a, const apx_kv4_cache &c,
                            const apx_seq_batch &b, cudaStream_t stream) {
  AttnArgs p;
  p.a = a;
  p.cu = b.d_cu;
  p.kv_len = b.d_kv_len;
  p.table = b.d_table;
  p.pages = static_cast<const uint8_t *>(c.d_pages);
  p.n_pages = c.n_pages;
  p.page_bytes = apx_kv4_page_bytes(c.head_dim, c.page_tokens);
  p.n_seqs = b.n_seqs;
  p.max_pages = b.max_pages;
  p.kv_heads = c.n_kv_heads;
  p.group = a.n_heads / c.n_kv_heads;
  p.dim = c.head_dim;
  p.page_tokens = c.page_tokens;
  attn_row_kernel<<<dim3((unsigned)b.n_tokens, (unsigned)a.n_heads), 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace apx
