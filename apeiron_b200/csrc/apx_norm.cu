// apx_norm.cu — residual add + RMS norm + quant_act: what stands between a projection's f32
// output and the next projection's 8-bit activation, in one pass over the row.
//
// h = x + add; r = 1 / sqrt(sum h^2 / n + eps); y = h r w; then quant_act of y per 32 lanes
// (apx_quant.cuh: the same codes as apx_quant_f32_cols_async of y).  A code is one step off where y
// is off by less than its last bit, so y is formed from more bits than it has: the squares' sum and
// the products carry a second f32 with the roundings' rest, r is f64, and y is rounded once.
//
// A CTA has a row, each thread four lanes (a quad) of every turn of the CTA over it; the row stays
// in registers between its sum and its quantization; rows past 16384 are read again.
//
// What bounds it: for many rows the bytes, 4 n read (8 n and 4 n written with a residual) and
// 1 + 1/32 n written, and some 65 instructions an element beside them: 512 rows of 8192 with
// residual and 16-bit values move 63 MB in 19.7 us, 3.2 TB/s, half of what a large copy reaches,
// with half of the issue slots used.  One row: the chain load, sum over the CTA, root, quantize,
// store (896 wide: 2.4 us).
#include <cuda_bf16.h>

#include <algorithm>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_pack.cuh"
#include "apx_quant.cuh"
#include "apx_step.h"

namespace apx {

namespace {

struct Stat {
  double sum;
  int emin, emax, status;
  unsigned nz;
};

template <bool FULL>
__device__ __forceinline__ float4 load4(const float *p, size_t j, size_t n, bool quads) {
  if (FULL)
    return j < n ? *reinterpret_cast<const float4 *>(p + j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (quads && j + 4 <= n) return *reinterpret_cast<const float4 *>(p + j);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (j < n) v.x = p[j];
  if (j + 1 < n) v.y = p[j + 1];
  if (j + 2 < n) v.z = p[j + 2];
  if (j + 3 < n) v.w = p[j + 3];
  return v;
}

template <bool FULL>
__device__ __forceinline__ void store4f(float *p, size_t j, size_t n, bool quads, const float4 v) {
  if (FULL) {
    if (j < n) *reinterpret_cast<float4 *>(p + j) = v;
    return;
  }
  if (quads && j + 4 <= n) {
    *reinterpret_cast<float4 *>(p + j) = v;
    return;
  }
  if (j < n) p[j] = v.x;
  if (j + 1 < n) p[j + 1] = v.y;
  if (j + 2 < n) p[j + 2] = v.z;
  if (j + 3 < n) p[j + 3] = v.w;
}

// (s, c) += h^2, c the rest of the roundings, for s >= h^2: then t <= 2 s and s - t is exact.
__device__ __forceinline__ void add_square(float &s, float &c, float h) {
  const float t = __fmaf_rn(h, h, s);
  c += __fmaf_rn(h, h, __fsub_rn(s, t));
  s = t;
}
// The same for any s: the sum's rest by Knuth's two-sum, the square's by the fused product.
__device__ __forceinline__ void add_any_square(float &s, float &c, float h) {
  const float p = __fmul_rn(h, h), t = __fadd_rn(s, p), b = __fsub_rn(t, s);
  c += __fadd_rn(__fadd_rn(__fsub_rn(s, __fsub_rn(t, b)), __fsub_rn(p, b)), __fmaf_rn(h, h, -p));
  s = t;
}

// h w r rounded once, r = rh + rl, where the products stay within f32.
__device__ __forceinline__ float scaled(float h, float w, float rh, float rl) {
  const float p = __fmul_rn(h, w), e = __fmaf_rn(h, w, -p);
  const float t = __fmul_rn(p, rh), f = __fmaf_rn(p, rh, -t);
  return __fadd_rn(t, __fmaf_rn(e, rh, __fmaf_rn(p, rl, f)));
}

// The largest magnitude, NaN if any is one.
__device__ __forceinline__ float max_abs(const float4 v) {
  float m;
  asm("{ .reg .f32 a; max.NaN.f32 a, %1, %2; max.NaN.f32 %0, %3, %4; max.NaN.f32 %0, %0, a; }"
      : "=&f"(m)
      : "f"(fabsf(v.x)), "f"(fabsf(v.y)), "f"(fabsf(v.z)), "f"(fabsf(v.w)));
  return m;
}

// quant_quad (apx_quant.cuh) in f32 arithmetic, for blocks whose S is 2^-7 or more (e >= 25: their
// largest value above 0.49, and below kFastAbsMax).  There a value that round(|y| 2^32) changes at
// all lies below every code's boundary, so one rounding is left: |y| / S is exact, and additions
// that round toward zero add the half and cut at the unit.  False, for the whole warp, where some
// block is another or holds a NaN; `m` is the quad's max_abs, `code` are the codes as f32.
__device__ __forceinline__ bool quant_quad_f32(const float4 y, float m, uint32_t &packed, int &e,
                                               float4 &code) {
  unsigned top = __float_as_uint(m);  // a NaN's is above kFastAbsMax
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  const int exp = (int)(top >> 23) - 101;
  e = exp + ((top & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);  // fast_scale_exp for E >= 118
  if (!__all_sync(0xFFFFFFFFu, exp >= 25 && top <= kFastAbsMax)) return false;
  const float inv = __int_as_float((127 + 32 - e) << 23);  // 1 / S
  auto one = [inv](float v, float &c) {
    const float cut = __fadd_rz(__fmaf_rz(fabsf(v), inv, 0.5f), 8388608.0f);
    c = copysignf(cut - 8388608.0f, v);
    return __float_as_uint(c + 12582912.0f);  // its low byte: c in two's complement
  };
  const unsigned a = one(y.x, code.x), b = one(y.y, code.y), c = one(y.z, code.z),
                 d = one(y.w, code.w);
  packed = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
  return true;
}

// QUADS: quads of the row in registers; 0 reads it twice.  FULL: quads are whole (n a multiple of
// 4) and every array's rows aligned.
template <int QUADS, int THREADS, bool FULL>
__global__ void __launch_bounds__(THREADS) norm_quant_kernel(const __grid_constant__ apx_norm_args a,
                                                             size_t padded, int vec) {
  constexpr int W = THREADS / 32;
  __shared__ double s_sum[W], s_r;
  __shared__ Stat s_stat[W];
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const float *x = a.d_x + row * a.ldx;
  const float *add = a.d_add ? a.d_add + row * a.ld_add : nullptr;
  const bool vx = vec & 1, va = vec & 2, vr = vec & 4, vy = vec & 8, vw = vec & 16, vd = vec & 32;
  constexpr int N = QUADS ? QUADS : 1;
  constexpr bool kFewRows = QUADS > 0 && QUADS <= 2;  // the weights in the values' round trip
  float4 h[N], w[kFewRows ? N : 1];
  const float4 one = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
  pdl_launch_dependents();
  pdl_wait();  // every input may be the output of the kernel before, the weights too
  auto value = [&](size_t j) {
    float4 v = load4<FULL>(x, j, a.n, vx);
    if (add) {
      const float4 b = load4<FULL>(add, j, a.n, va);
      v = make_float4(__fadd_rn(v.x, b.x), __fadd_rn(v.y, b.y), __fadd_rn(v.z, b.z),
                      __fadd_rn(v.w, b.w));
    }
    return v;
  };
  float s = 0.0f, c = 0.0f, s0 = 0.0f;
  if (QUADS) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const size_t j = 4 * (size_t)(i * THREADS + tid);
      h[i] = value(j);
      if (kFewRows) w[kFewRows ? i : 0] = a.d_weight ? load4<FULL>(a.d_weight, j, a.n, vw) : one;
    }
    // the sum starts at (no less than) its largest square, and gives it back
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++)
      top = fmaxf(top, fmaxf(fmaxf(fabsf(h[i].x), fabsf(h[i].y)),
                             fmaxf(fabsf(h[i].z), fabsf(h[i].w))));
    s = s0 = __fmul_ru(top, top);
#pragma unroll
    for (int i = 0; i < N; i++) {
      add_square(s, c, h[i].x);
      add_square(s, c, h[i].y);
      add_square(s, c, h[i].z);
      add_square(s, c, h[i].w);
    }
  } else {
    for (size_t j = 4 * (size_t)tid; j < a.n; j += 4 * THREADS) {
      const float4 v = value(j);
      add_any_square(s, c, v.x);
      add_any_square(s, c, v.y);
      add_any_square(s, c, v.z);
      add_any_square(s, c, v.w);
    }
  }
  // squares near f32's ends (or a value that is not finite) leave no rest: the sum in f64
  double sum = ((double)s - (double)s0) + (double)c;
  if (!(s > 1e-25f && s < 3e38f)) {
    sum = 0.0;
    for (size_t j = 4 * (size_t)tid; j < a.n; j += 4 * THREADS) {
      const float4 v = value(j);
      sum += (double)v.x * v.x + (double)v.y * v.y + (double)v.z * v.z + (double)v.w * v.w;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (W > 1) {
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    if (kFewRows || warp == 0) {
      sum = lane < W ? s_sum[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
  }
  double r = 0.0;
  if (kFewRows || warp == 0) r = 1.0 / sqrt(sum / (double)a.n + (double)a.eps);
  if (!kFewRows) {  // many rows: its instructions once a row
    if (tid == 0) s_r = r;
    __syncthreads();
    r = s_r;
  }
  const float rh = (float)r, rl = fabsf(rh) < 3e38f ? (float)(r - (double)rh) : 0.0f;
  // f64 from here up, where h w may pass f32's end; everywhere where r lifts an h w below the normal
  // numbers by more than 2^20 (less: an error below 2^-129)
  const float most = rh < 1048576.0f ? 1e37f : -1.0f;

  int emin = 1 << 30, emax = -1, status = APX_OK;
  unsigned nz = 0;
  auto quad = [&](size_t j, const float4 v, const float4 g) {
    float4 y = make_float4(scaled(v.x, g.x, rh, rl), scaled(v.y, g.y, rh, rl),
                           scaled(v.z, g.z, rh, rl), scaled(v.w, g.w, rh, rl));
    float m = max_abs(y);
    if (!(m < most)) {
      auto wide = [r](float h, float w) { return (float)((double)h * (double)w * r); };
      y = make_float4(wide(v.x, g.x), wide(v.y, g.y), wide(v.z, g.z), wide(v.w, g.w));
      m = max_abs(y);
    }
    if (a.d_resid) store4f<FULL>(a.d_resid + row * a.ld_resid, j, a.n, vr, v);
    if (a.d_y) store4f<FULL>(a.d_y + row * a.ldy, j, a.n, vy, y);
    if (!a.d_codes && !a.d_deq) return;
    uint32_t packed;
    int e;
    bool ok = true;
    float4 code;
    if (!quant_quad_f32(y, m, packed, e, code)) {
      quant_quad(y, packed, e, ok);
      if (!ok || e < 0) packed = 0;
      code = make_float4((float)(int8_t)packed, (float)(int8_t)(packed >> 8),
                         (float)(int8_t)(packed >> 16), (float)(int8_t)(packed >> 24));
    }
    if (a.d_codes && j < padded)
      *reinterpret_cast<uint32_t *>(a.d_codes + row * padded + j) = packed;
    if (a.d_deq) {
      const float q = ok && e >= 0 ? __int_as_float((127 + e - 32) << 23) : 0.0f;
      const float4 d = make_float4(q * code.x, q * code.y, q * code.z, q * code.w);
      if (a.deq_type == APX_DTYPE_F32) {
        store4f<FULL>(static_cast<float *>(a.d_deq) + row * a.ld_deq, j, a.n, vd, d);
      } else {
        __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(a.d_deq) + row * a.ld_deq + j;
        const __nv_bfloat162 lo = __floats2bfloat162_rn(d.x, d.y), hi = __floats2bfloat162_rn(d.z, d.w);
        if (FULL ? j < a.n : vd && j + 4 <= a.n) {
          *reinterpret_cast<uint2 *>(dst) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo),
                                                       *reinterpret_cast<const uint32_t *>(&hi));
        } else if (!FULL) {
          if (j < a.n) dst[0] = lo.x;
          if (j + 1 < a.n) dst[1] = lo.y;
          if (j + 2 < a.n) dst[2] = hi.x;
          if (j + 3 < a.n) dst[3] = hi.y;
        }
      }
    }
    if ((lane & 7) == 0 && j < padded) {
      if (a.d_exps)
        a.d_exps[(row * padded + j) / 32] = e < 0 || !ok ? (uint8_t)APX_EXP_ZERO : (uint8_t)e;
      if (j < a.n) {
        if (!ok) {
          status = APX_ERR_QUANT_REFUSED;
        } else if (e >= 0) {
          emin = min(emin, e);
          emax = max(emax, e);
          nz++;
        }
      }
    }
  };
  if (QUADS) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const size_t j = 4 * (size_t)(i * THREADS + tid);
      quad(j, h[i], kFewRows ? w[kFewRows ? i : 0]
                    : a.d_weight  ? load4<FULL>(a.d_weight, j, a.n, vw)
                                  : one);
    }
  } else {
    // whole warps: quant_quad's shuffles take every lane
    const size_t end = (padded + 4 * THREADS - 1) / (4 * THREADS) * (4 * THREADS);
    for (size_t j = 4 * (size_t)tid; j < end; j += 4 * THREADS)
      quad(j, value(j), a.d_weight ? load4<FULL>(a.d_weight, j, a.n, vw) : one);
  }
  if (!a.d_descs) return;
  emin = __reduce_min_sync(0xFFFFFFFFu, emin);
  emax = __reduce_max_sync(0xFFFFFFFFu, emax);
  status = __reduce_max_sync(0xFFFFFFFFu, status);
  nz = __reduce_add_sync(0xFFFFFFFFu, nz);
  if (W > 1) {
    if (lane == 0) s_stat[warp] = Stat{0.0, emin, emax, status, nz};
    __syncthreads();
    if (warp == 0) {
      const Stat t = s_stat[lane % W];
      emin = __reduce_min_sync(0xFFFFFFFFu, t.emin);
      emax = __reduce_max_sync(0xFFFFFFFFu, t.emax);
      status = __reduce_max_sync(0xFFFFFFFFu, t.status);
      nz = __reduce_add_sync(0xFFFFFFFFu, lane < W ? t.nz : 0u);
    }
  }
  if (tid == 0) {
    ActDesc d = {};
    d.status = status;
    d.emin = emax >= 0 ? emin : 0;
    d.emax = emax;
    d.n_in = (int32_t)a.n;
    d.nz = nz;
    reinterpret_cast<ActDesc *>(a.d_descs)[row] = d;
  }
}

template <int QUADS, int THREADS, bool FULL>
cudaError_t launch_full(const apx_norm_args &a, size_t padded, int vec, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.k);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_allowed() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, norm_quant_kernel<QUADS, THREADS, FULL>, a, padded, vec);
}

template <int QUADS, int THREADS>
cudaError_t launch(const apx_norm_args &a, size_t padded, int vec, cudaStream_t stream) {
  return a.n % 4 == 0 && vec == 63 ? launch_full<QUADS, THREADS, true>(a, padded, vec, stream)
                                   : launch_full<QUADS, THREADS, false>(a, padded, vec, stream);
}

}  // namespace

cudaError_t launch_add_rms_norm_quant(const apx_norm_args &a, int sms, cudaStream_t stream) {
  const size_t padded = apx_act_padded_len(a.n);
  // which arrays have 16-byte (the 16-bit values: 8-byte) aligned rows
  auto whole = [](const void *p, size_t ld, size_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && ld % 4 == 0;
  };
  int vec = 0;
  if (whole(a.d_x, a.ldx, 16)) vec |= 1;
  if (whole(a.d_add, a.ld_add, 16)) vec |= 2;
  if (whole(a.d_resid, a.ld_resid, 16)) vec |= 4;
  if (whole(a.d_y, a.ldy, 16)) vec |= 8;
  if (whole(a.d_weight, 0, 16)) vec |= 16;
  if (whole(a.d_deq, a.ld_deq, a.deq_type == APX_DTYPE_F32 ? 16 : 8)) vec |= 32;
  const size_t quads = padded / 4;  // padded is what has to be written
  // Few rows: as many threads as the row has quads, the loads of a row one round trip.  Many rows
  // fill the GPU with smaller CTAs of more quads a thread (512 rows of 8192: 4 quads of 512 threads
  // 20.0 us, 8 of 256 19.7).
  if (quads <= 256) return launch<1, 256>(a, padded, vec, stream);
  const bool few = a.k <= (size_t)sms;
  if (few && quads <= 1024) return launch<1, 1024>(a, padded, vec, stream);
  if (few && quads <= 2048) return launch<2, 1024>(a, padded, vec, stream);
  if (quads <= 512) return launch<2, 256>(a, padded, vec, stream);
  if (quads <= 1024) return launch<4, 256>(a, padded, vec, stream);
  if (quads <= 2048) return launch<8, 256>(a, padded, vec, stream);
  if (quads <= 4096) return launch<4, 1024>(a, padded, vec, stream);
  return launch<0, 1024>(a, padded, vec, stream);
}

}  // namespace apx
