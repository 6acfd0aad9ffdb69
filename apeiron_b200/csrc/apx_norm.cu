// apx_norm.cu — residual add + RMS norm + quant_act: what stands between a projection's f32
// output and the next projection's 8-bit activation, in one pass over the row.
//
// h = x + add; r = 1 / sqrt(sum h^2 / n + eps); y = h r w; then quant_act of y per 32 lanes
// (apx_quant.cuh: the same codes as apx_quant_f32_cols_async of y).  The square sum and the
// product h r w are carried in f64 and rounded once: a code changes only where y itself lies
// within half an f32 rounding of a code's boundary.
#include <cuda_bf16.h>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_quant.cuh"
#include "apx_step.h"

namespace apx {

struct NormDesc {
  int emin, emax, status;
  unsigned nz;
};

// One CTA per row, a quad of lanes per thread and turn.
__global__ void __launch_bounds__(256) norm_quant_kernel(apx_norm_args a, size_t padded) {
  __shared__ double s_sum[8];
  __shared__ NormDesc s_d;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const float *x = a.d_x + row * a.ldx;
  const float *add = a.d_add ? a.d_add + row * a.ld_add : nullptr;
  if (tid == 0) s_d = NormDesc{1 << 30, -1, APX_OK, 0u};
  auto value = [&](size_t j) {
    return j < a.n ? (add ? __fadd_rn(x[j], add[j]) : x[j]) : 0.0f;
  };
  double sum = 0.0;
  for (size_t j = tid; j < a.n; j += blockDim.x) {
    const double h = value(j);
    sum += h * h;
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < 8; i++) sum += s_sum[i];
  const double r = 1.0 / sqrt(sum / (double)a.n + (double)a.eps);
  int emin = 1 << 30, emax = -1, status = APX_OK;
  unsigned nz = 0;
  const size_t end = (padded + 1023) / 1024 * 1024;
  for (size_t j = 4 * (size_t)tid; j < end; j += 4 * blockDim.x) {
    float h[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      h[i] = value(j + i);
      const double w = a.d_weight && j + i < a.n ? (double)a.d_weight[j + i] : 1.0;
      y[i] = (float)((double)h[i] * w * r);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (j + i < a.n) {
        if (a.d_resid) a.d_resid[row * a.ld_resid + j + i] = h[i];
        if (a.d_y) a.d_y[row * a.ldy + j + i] = y[i];
      }
    uint32_t packed;
    int e;
    bool ok;
    quant_quad(make_float4(y[0], y[1], y[2], y[3]), packed, e, ok);
    if (!ok || e < 0) packed = 0;
    if (a.d_codes) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (j + i < padded) a.d_codes[row * padded + j + i] = (int8_t)(packed >> (8 * i));
    }
    if (a.d_deq) {
      const float s = ok && e >= 0 ? __int_as_float((127 + e - 32) << 23) : 0.0f;
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (j + i < a.n) {
          const float v = s * (float)(int8_t)(packed >> (8 * i));
          if (a.deq_type == APX_DTYPE_F32)
            static_cast<float *>(a.d_deq)[row * a.ld_deq + j + i] = v;
          else
            static_cast<__nv_bfloat16 *>(a.d_deq)[row * a.ld_deq + j + i] = __float2bfloat16(v);
        }
    }
    if ((lane & 7) == 0 && j < padded) {
      if (a.d_exps) a.d_exps[(row * padded + j) / 32] = e < 0 || !ok ? APX_EXP_ZERO : (uint8_t)e;
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
  }
  if (!a.d_descs) return;
  if (status != APX_OK) atomicMax(&s_d.status, status);
  if (nz) {
    atomicMin(&s_d.emin, emin);
    atomicMax(&s_d.emax, emax);
    atomicAdd(&s_d.nz, nz);
  }
  __syncthreads();
  if (tid == 0) {
    ActDesc d = {};
    d.status = s_d.status;
    d.emin = s_d.emax >= 0 ? s_d.emin : 0;
    d.emax = s_d.emax;
    d.n_in = (int32_t)a.n;
    d.nz = s_d.nz;
    reinterpret_cast<ActDesc *>(a.d_descs)[row] = d;
  }
}

cudaError_t launch_add_rms_norm_quant(const apx_norm_args &a, cudaStream_t stream) {
  norm_quant_kernel<<<(unsigned)a.k, 256, 0, stream>>>(a, apx_act_padded_len(a.n));
  return cudaGetLastError();
}

}  // namespace apx
