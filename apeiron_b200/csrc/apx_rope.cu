// apx_rope.cu — rotary positions and the append of K and V to the paged 4-bit cache.
//
// A pair (a, b) at position p turns by the table's angle: (a c - b s, b c + a s), each operation
// one f32 rounding.  K (turned) and V then go to 4 bits per 32 dims: m the group's value of
// largest magnitude, d = f16(bf16(-m / 8)) (8 significant bits: d (c - 8) is exact in f16, so the
// attention's operand conversion loses nothing), c = clamp(rint(x (1 / d)) + 8, 0, 15).
//
// What bounds it: 4 bytes read a value and 2 or 4 (q) or 9/16 (K, V) written; 512 tokens of 64 + 2 x
// 8 heads of 128 move 41 MB in 12.8 us, 3.2 TB/s, with three quarters of the issue slots used.  A
// thread takes four dims, the eight lanes of a scale's group reduce by shuffles; it has two heads
// at most to go round, so that eight CTAs an SM (32 registers) hide the chain position, page,
// values (the coefficients kept over more heads, the next head's values loaded ahead: 48 to 62
// registers, 12.6 to 14 us).  32 decoded tokens: 3.7 us, all of it that chain.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_kv4.cuh"
#include "apx_pack.cuh"
#include "apx_step.h"

namespace apx {

constexpr float kKvMax = 65280.0f;  // 8 * 8160: past it d (c - 8) could leave f16

// ---- the table -------------------------------------------------------------------------------

__global__ void rope_table_kernel(apx_rope_freqs f, size_t n_pos, float2 *table) {
  const int half = f.rot_dim / 2;
  const size_t at = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (at >= n_pos * half) return;
  const int i = (int)(at % half);
  const double pos = (double)(at / half), tau = 6.283185307179586476925;
  double w = pow(f.base, -2.0 * i / f.rot_dim);
  if (f.scaling == APX_ROPE_LINEAR) {
    w /= f.factor;
  } else if (f.scaling == APX_ROPE_BANDS) {
    const double turns = f.original * w / tau;  // over the original length
    if (turns < f.low) {
      w /= f.factor;
    } else if (turns <= f.high) {
      const double s = (turns - f.low) / (f.high - f.low);
      w = w * (s + (1.0 - s) / f.factor);
    }
  } else if (f.scaling == APX_ROPE_RAMP) {
    const double per = f.rot_dim / (2.0 * log(f.base));
    const double first = fmax(floor(per * log(f.original / (tau * f.high))), 0.0);
    const double last = fmin(ceil(per * log(f.original / (tau * f.low))), f.rot_dim - 1.0);
    const double s = fmin(fmax((i - first) / fmax(last - first, 1e-3), 0.0), 1.0);
    w = w * (1.0 - s) + w / f.factor * s;
  }
  double sn, cs;
  sincos(pos * w, &sn, &cs);
  table[at] = make_float2((float)(cs * f.mscale), (float)(sn * f.mscale));
}

cudaError_t launch_rope_table(const apx_rope_freqs &f, size_t n_pos, float *table,
                              cudaStream_t stream) {
  const size_t n = n_pos * (f.rot_dim / 2), grid = (n + 255) / 256;
  if (grid > 0x7FFFFFFFull) return cudaErrorInvalidValue;
  rope_table_kernel<<<(unsigned)grid, 256, 0, stream>>>(f, n_pos,
                                                        reinterpret_cast<float2 *>(table));
  return cudaGetLastError();
}

// ---- rotation and append ---------------------------------------------------------------------

struct RopeArgs {
  apx_rope_args a;
  const int *cu, *kv_len, *table;
  uint8_t *pages;
  size_t n_pages, page_bytes;
  int n_seqs, max_pages, kv_heads, dim, page_shift;
};

// Four dims of a head at x, turned.  i: the first dim, a multiple of 4 (rot is a multiple of 8).
__device__ __forceinline__ float4 turn4(const float *x, int i, int rot, int layout,
                                        const float2 *cs) {
  const float4 v = *reinterpret_cast<const float4 *>(x + i);
  if (i >= rot) return v;
  if (layout == APX_ROPE_INTERLEAVED) {
    const float4 t = *reinterpret_cast<const float4 *>(cs + i / 2);
    return make_float4(__fsub_rn(__fmul_rn(v.x, t.x), __fmul_rn(v.y, t.y)),
                       __fadd_rn(__fmul_rn(v.y, t.x), __fmul_rn(v.x, t.y)),
                       __fsub_rn(__fmul_rn(v.z, t.z), __fmul_rn(v.w, t.w)),
                       __fadd_rn(__fmul_rn(v.w, t.z), __fmul_rn(v.z, t.w)));
  }
  const int half = rot / 2;
  const bool hi = i >= half;
  const int j = hi ? i - half : i;
  const float4 o = *reinterpret_cast<const float4 *>(x + (hi ? j : i + half));
  const float4 t0 = *reinterpret_cast<const float4 *>(cs + j);
  const float4 t1 = *reinterpret_cast<const float4 *>(cs + j + 2);
  auto one = [hi](float p, float q, float c, float s) {
    return hi ? __fadd_rn(__fmul_rn(p, c), __fmul_rn(q, s))
              : __fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s));
  };
  return make_float4(one(v.x, o.x, t0.x, t0.y), one(v.y, o.y, t0.z, t0.w),
                     one(v.z, o.z, t1.x, t1.y), one(v.w, o.w, t1.z, t1.w));
}

// The largest index s with cu[s] <= t (cu ascending, cu[0] = 0).
__device__ __forceinline__ int find_seq(const int *cu, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint2 pack4(const float4 v, bool bf16) {
  if (bf16) {
    __nv_bfloat162 p = __floats2bfloat162_rn(v.x, v.y), q = __floats2bfloat162_rn(v.z, v.w);
    return make_uint2(*reinterpret_cast<uint32_t *>(&p), *reinterpret_cast<uint32_t *>(&q));
  }
  __half2 p = __floats2half2_rn(v.x, v.y), q = __floats2half2_rn(v.z, v.w);
  return make_uint2(*reinterpret_cast<uint32_t *>(&p), *reinterpret_cast<uint32_t *>(&q));
}

// A token per blockIdx.x; dim / 4 threads take a head (query heads, then K heads, then V heads),
// the heads shared by the CTAs of blockIdx.y.
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ RopeArgs r) {
  const apx_rope_args &a = r.a;
  const int t = blockIdx.x, per = r.dim / 4;
  pdl_launch_dependents();
  pdl_wait();
  const int seq = find_seq(r.cu, r.n_seqs, t);
  const int begin = r.cu[seq], end = r.cu[seq + 1], kv = r.kv_len[seq];
  const int pos = kv - (end - t);
  const int slot = pos >> r.page_shift;
  // a token that the lengths leave to no request has no position
  bool ok = begin <= t && t < end && kv >= end - t && slot < r.max_pages &&
            (a.rot_dim == 0 || (size_t)pos < a.n_pos);
  int page = -1;
  if (ok) {
    page = r.table[(size_t)seq * r.max_pages + slot];
    ok = page >= 0 && (size_t)page < r.n_pages;
  }
  if (!ok) {
    if (threadIdx.x == 0 && blockIdx.y == 0 && a.d_status)
      atomicMin(&a.d_status->first,
                (unsigned long long)t << 24 | (unsigned long long)APX_ERR_INVALID_ARGUMENT << 16);
    return;
  }
  const float2 *cs = reinterpret_cast<const float2 *>(a.d_table) + (size_t)pos * (a.rot_dim / 2);
  const int row = pos % kKvTile, tile = (pos & ((1 << r.page_shift) - 1)) / kKvTile;
  const int nq = a.d_q ? a.n_heads : 0, heads = nq + 2 * r.kv_heads;
  for (int w = blockIdx.y * blockDim.x + threadIdx.x; w < heads * per;
       w += gridDim.y * blockDim.x) {  // whole groups of 8 lanes
    const int head = w / per, i = w % per * 4;
    if (head < nq) {
      const float4 v = turn4(a.d_q + (size_t)t * a.ldq + (size_t)head * r.dim, i, a.rot_dim,
                             a.layout, cs);
      const size_t at = (size_t)t * a.ldq_out + (size_t)head * r.dim + i;
      // the head's lanes, all of one warp, have read it before one writes where it stands
      if (a.d_q_out == a.d_q) __syncwarp(per == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16));
      if (a.q_type == APX_DTYPE_F32)
        *reinterpret_cast<float4 *>(static_cast<float *>(a.d_q_out) + at) = v;
      else
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.d_q_out) + at) =
            pack4(v, a.q_type == APX_DTYPE_BF16);
      continue;
    }
    const bool is_k = head < nq + r.kv_heads;
    const int h = is_k ? head - nq : head - nq - r.kv_heads;
    const float4 v =
        is_k ? turn4(a.d_k + (size_t)t * a.ldk + (size_t)h * r.dim, i, a.rot_dim, a.layout, cs)
             : *reinterpret_cast<const float4 *>(a.d_v + (size_t)t * a.ldv + (size_t)h * r.dim + i);
    const unsigned mask = 0xFFu << (threadIdx.x & 24);  // the group's 8 lanes
    float hi = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
    float lo = fminf(fminf(v.x, v.y), fminf(v.z, v.w));
    bool bad = !(fabsf(v.x) <= kKvMax && fabsf(v.y) <= kKvMax && fabsf(v.z) <= kKvMax &&
                 fabsf(v.w) <= kKvMax);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
      lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
      bad |= __shfl_xor_sync(mask, (int)bad, o) != 0;
    }
    __half d = __float2half_rn(
        __bfloat162float(__float2bfloat16_rn(__fmul_rn(hi >= -lo ? hi : lo, -0.125f))));
    if (bad) {
      d = __ushort_as_half(0);
      if (a.d_status)
        atomicMin(&a.d_status->first,
                  (unsigned long long)t << 24 | (unsigned long long)APX_ERR_QUANT_REFUSED << 16);
    }
    const float f = __half2float(d), inv = f == 0.0f ? 0.0f : __frcp_rn(f);
    auto code = [&](float x) {
      const float c = rintf(__fmul_rn(x, inv)) + 8.0f;
      return bad || f == 0.0f ? 8u : (unsigned)fminf(fmaxf(c, 0.0f), 15.0f);
    };
    const unsigned c0 = code(v.x), c1 = code(v.y), c2 = code(v.z), c3 = code(v.w);
    uint8_t *tp = r.pages + ((size_t)page * r.kv_heads + h) * r.page_bytes +
                  (size_t)tile * kv4_tile_bytes(r.dim);
    if (is_k) {
      *reinterpret_cast<uint16_t *>(tp + row * (r.dim / 2) + i / 2) =
          (uint16_t)(c0 | c1 << 4 | c2 << 8 | c3 << 12);
    } else {
      // dims 16 m + g and 16 m + g + 8 share a byte: the partner is two quads on
      const unsigned mine = c0 | c1 << 8 | c2 << 16 | c3 << 24;
      const unsigned other = __shfl_xor_sync(mask, mine, 2);
      if ((i & 8) == 0) {
        const unsigned both = mine | other << 4;
#pragma unroll
        for (int k = 0; k < 4; k++)
          tp[kv4_v_off(r.dim) + kv4_v_byte(i + k, row)] = (uint8_t)(both >> (8 * k));
      }
    }
    if ((i & 31) == 0)
      *reinterpret_cast<__half *>(tp + (is_k ? kv4_ks_off(r.dim) : kv4_vs_off(r.dim)) +
                                  (i / kKvGroup * kKvTile + row) * 2) = d;
    uint16_t *deq = is_k ? a.d_k_deq : a.d_v_deq;
    if (deq) {
      const float4 q = make_float4(f * (float)((int)c0 - 8), f * (float)((int)c1 - 8),
                                   f * (float)((int)c2 - 8), f * (float)((int)c3 - 8));
      *reinterpret_cast<uint2 *>(deq + ((size_t)t * r.kv_heads + h) * r.dim + i) =
          pack4(q, false);
    }
  }
}

cudaError_t launch_rope_kv4_append(const apx_rope_args &a, const apx_kv4_cache &c,
                                   const apx_seq_batch &b, cudaStream_t stream) {
  RopeArgs r;
  r.a = a;
  r.cu = b.d_cu;
  r.kv_len = b.d_kv_len;
  r.table = b.d_table;
  r.pages = static_cast<uint8_t *>(c.d_pages);
  r.n_pages = c.n_pages;
  r.page_bytes = apx_kv4_page_bytes(c.head_dim, c.page_tokens);
  r.n_seqs = b.n_seqs;
  r.max_pages = b.max_pages;
  r.kv_heads = c.n_kv_heads;
  r.dim = c.head_dim;
  r.page_shift = 0;
  while (1 << r.page_shift < c.page_tokens) r.page_shift++;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // two heads' worth a thread: more CTAs hide the chain position, page, values of each
  const unsigned work = (unsigned)((a.d_q ? a.n_heads : 0) + 2 * c.n_kv_heads) * (c.head_dim / 4);
  cfg.gridDim = dim3((unsigned)b.n_tokens, (work + 511) / 512);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_allowed() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, rope_append_kernel, r);
}

}  // namespace apx
