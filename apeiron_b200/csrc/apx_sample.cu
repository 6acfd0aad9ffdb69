// apx_sample.cu — one token per row of logits: temperature, top-k, top-p, min-p, from a given
// uniform number.
//
// The weights are integers, w = rint(e 2^31) with e = exp((l - max) / T) in the F32 carrier's
// binary32 arithmetic, so sums and comparisons are exact and no order of summation can change
// the token.  "Sorted by e, lower index first" needs no sort: the filters keep every token whose
// e exceeds some threshold and the first few, by index, of those equal to it.
#include <climits>

#include "apx_common.cuh"
#include "apx_step.h"
#include "apx_swiglu.cuh"

namespace apx {

constexpr int kSampleThreads = 1024;
constexpr float kWeightOne = 2147483648.0f;  // 2^31

struct SampleRow {
  const float *x;
  size_t vocab;
  float top, inv_t;
  // e as its bits: they order as e does (e >= 0)
  __device__ unsigned key(size_t i) const {
    const float l = x[i];
    if (!(l > -INFINITY)) return 0u;  // NaN and -inf
    if (l == top) return 0x3F800000u;
    return __float_as_uint(exp_ref(__fmul_rn(__fsub_rn(l, top), inv_t)));
  }
};

__device__ __forceinline__ unsigned weight_of(unsigned key) {
  return __float2uint_rn(__uint_as_float(key) * kWeightOne);
}

// Sum over the CTA, the same in every thread.
__device__ unsigned long long cta_sum(unsigned long long v, unsigned long long *s) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s[threadIdx.x / 32] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < (int)blockDim.x / 32; i++) v += s[i];
  return v;
}

__global__ void __launch_bounds__(kSampleThreads) sample_kernel(apx_sample_args a) {
  __shared__ unsigned long long s_sum[32], s_scan[kSampleThreads];
  __shared__ float s_top[32];
  __shared__ int s_at;
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x;
  SampleRow r;
  r.x = a.d_logits + row * a.ld;
  r.vocab = a.vocab;
  float top = -INFINITY;
  for (size_t i = tid; i < a.vocab; i += blockDim.x) top = fmaxf(top, r.x[i]);
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (tid % 32 == 0) s_top[tid / 32] = top;
  if (tid == 0) s_at = INT_MAX;
  __syncthreads();
  for (int i = 0; i < 32; i++) top = fmaxf(top, s_top[i]);
  r.top = top;
  const float temp = a.d_temperature ? a.d_temperature[row] : 1.0f;
  if (top == -INFINITY) {
    if (tid == 0) {
      a.d_token[row] = -1;
      if (a.d_prob) a.d_prob[row] = 0.0f;
      if (a.d_kept) a.d_kept[row] = 0;
    }
    return;
  }
  if (!(temp > 0.0f)) {
    for (size_t i = tid; i < a.vocab; i += blockDim.x)
      if (r.x[i] == top) {
        atomicMin(&s_at, (int)i);
        break;
      }
    __syncthreads();
    if (tid == 0) {
      a.d_token[row] = s_at;
      if (a.d_prob) a.d_prob[row] = 1.0f;
      if (a.d_kept) a.d_kept[row] = 1;
    }
    return;
  }
  r.inv_t = __frcp_rn(temp);
  // tokens with key > cut stay, and the first `ties` of those with key == cut
  unsigned cut = 0;
  unsigned long long ties = ULLONG_MAX;
  const long long k = a.d_top_k ? a.d_top_k[row] : 0;
  if (k > 0 && (size_t)k < a.vocab) {
    for (int bit = 29; bit >= 0; bit--) {  // the largest cut that k tokens reach
      const unsigned t = cut | 1u << bit;
      unsigned long long n = 0;
      for (size_t i = tid; i < a.vocab; i += blockDim.x) n += r.key(i) >= t;
      if (cta_sum(n, s_sum) >= (unsigned long long)k) cut = t;
    }
    unsigned long long n = 0;
    for (size_t i = tid; i < a.vocab; i += blockDim.x) n += r.key(i) > cut;
    ties = (unsigned long long)k - cta_sum(n, s_sum);
  }
  const float top_p = a.d_top_p ? a.d_top_p[row] : 1.0f;
  if (top_p < 1.0f) {
    unsigned long long above = 0, equal = 0;
    for (size_t i = tid; i < a.vocab; i += blockDim.x) {
      const unsigned key = r.key(i);
      if (key > cut) above += weight_of(key);
      equal += key == cut;
    }
    above = cta_sum(above, s_sum);
    equal = cta_sum(equal, s_sum);
    const unsigned long long first = ties < equal ? ties : equal;
    const double limit = (double)top_p * (double)(above + first * weight_of(cut));
    // the smallest t whose heavier tokens sum to less than limit
    unsigned t = 0x3F800000u;
    unsigned long long over = 0;  // the sum above t
    if (limit > 0.0) {
      unsigned lo = cut, hi = 0x3F800000u;
      while (lo < hi) {
        const unsigned mid = lo + (hi - lo) / 2;
        unsigned long long w = 0;
        for (size_t i = tid; i < a.vocab; i += blockDim.x) {
          const unsigned key = r.key(i);
          if (key > mid) w += weight_of(key);
        }
        w = cta_sum(w, s_sum);
        if ((double)w < limit) hi = mid;
        else lo = mid + 1;
      }
      t = lo;
      unsigned long long w = 0;
      for (size_t i = tid; i < a.vocab; i += blockDim.x) {
        const unsigned key = r.key(i);
        if (key > t) w += weight_of(key);
      }
      over = cta_sum(w, s_sum);
    }
    // of the tokens at t, those before which less than limit was summed; at least one at the top
    const unsigned long long each = weight_of(t);
    unsigned long long n = ULLONG_MAX;
    if (limit <= 0.0) {
      n = 1;
    } else if (each) {
      n = (unsigned long long)((limit - (double)over) / (double)each);
      n = n > 1 ? n - 1 : 0;
      while ((double)(over + n * each) < limit) n++;
    }
    if (t > cut) {
      cut = t;
      ties = n;
    } else {
      ties = n < ties ? n : ties;
    }
  }
  const double min_w = a.d_min_p ? (double)a.d_min_p[row] * (double)kWeightOne : 0.0;
  // two passes in vocabulary order: the kept weights' sum, then the token at which it passes
  // the aim; a CTA scan ranks the tokens that equal the cut
  unsigned long long total = 0, kept = 0, aim = 0;
  for (int pass = 0; pass < 2; pass++) {
    unsigned long long run = 0, seen = 0;
    for (size_t base = 0; base < a.vocab; base += blockDim.x) {
      const size_t i = base + tid;
      const unsigned key = i < a.vocab ? r.key(i) : 0u;
      const bool here = i < a.vocab;
      auto scan = [&](unsigned long long v, unsigned long long &sum) {  // exclusive
        __syncthreads();
        s_scan[tid] = v;
        __syncthreads();
        for (int o = 1; o < kSampleThreads; o <<= 1) {
          const unsigned long long u = tid >= o ? s_scan[tid - o] : 0;
          __syncthreads();
          s_scan[tid] += u;
          __syncthreads();
        }
        sum = s_scan[kSampleThreads - 1];
        return s_scan[tid] - v;
      };
      unsigned long long sum;
      const unsigned long long rank = seen + scan(here && key == cut, sum);
      seen += sum;
      unsigned w = here && (key > cut || (key == cut && rank < ties)) ? weight_of(key) : 0u;
      if ((double)w < min_w) w = 0;
      const unsigned long long before = run + scan(w, sum);
      if (pass == 1 && w && before <= aim && aim < before + w) {
        a.d_token[row] = (int)i;
        if (a.d_prob) a.d_prob[row] = (float)((double)w / (double)total);
      }
      run += sum;
      if (pass == 0) kept += w != 0;
    }
    if (pass == 0) {
      total = run;
      kept = cta_sum(kept, s_sum);
      if (tid == 0 && a.d_kept) a.d_kept[row] = (int)kept;
      if (total == 0) {
        if (tid == 0) {
          a.d_token[row] = -1;
          if (a.d_prob) a.d_prob[row] = 0.0f;
        }
        return;
      }
      aim = (unsigned long long)((double)a.d_u[row] * (double)total);
      if (aim >= total) aim = total - 1;
    }
  }
}

cudaError_t launch_sample(const apx_sample_args &a, cudaStream_t stream) {
  sample_kernel<<<(unsigned)a.rows, kSampleThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace apx
