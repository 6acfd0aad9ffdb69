// apx_sample.cu — one token per row of logits: temperature, top-k, top-p, min-p, from a given
// uniform number.
//
// The weights are integers, w = rint(e 2^31) with e = exp((l - max) / T) in the F32 carrier's
// binary32 arithmetic, so sums and comparisons are exact and no order of summation can change
// the token.  "Sorted by e, lower index first" needs no sort: the filters keep every token whose
// e exceeds some cut and the first few, by index, of those equal to it.
//
// A row's logits are read once, into the registers of a cluster of CTAs.  The bits of e order as
// e does, 30 of them: the cut is found ten bits at a time from a histogram of counts (top-k) or
// weight sums (top-p) over the tokens that share the bits found so far.  Each CTA counts in its
// own shared memory and adds its bins to the first CTA's, which scans them from the top and
// publishes the bin that crosses the target.  The first level's histogram serves both filters.
//
// Where that bin and those above it hold 1024 tokens at most (any top-k in the hundreds, most
// nuclei), they go to the first CTA, which sorts them, a token a thread: ranks and running sums
// decide every filter at once, and a second sort, by index, the token.  It takes two cluster
// barriers instead of two for each of up to five more levels.
//
// What bounds it: 4 bytes a logit is the floor (64 rows of 151936: 5.9 us); measured 54 us (top-k)
// to 71 us (a nucleus with min-p), with half of the issue slots of the SMs that hold a CTA in use
// (some 90 instructions a token: e in separately rounded steps, three shared-memory additions, the
// comparisons) and barriers the first reason to wait.  One row: the chain of barriers, scans and
// the list's sorts, 13.8 us.
#include <algorithm>
#include <climits>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_pack.cuh"
#include "apx_step.h"

namespace apx {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kBins = 1024;  // ten bits of the key a level
constexpr int kMaxCluster = 16;
constexpr unsigned kTopKey = 0x3F800000u;  // e = 1
constexpr float kWeightOne = 2147483648.0f;  // 2^31
typedef unsigned long long u64;

__device__ __forceinline__ unsigned weight_of(unsigned key) {
  return __float2uint_rn(__uint_as_float(key) * kWeightOne);
}

// exp_ref (apx_swiglu.cuh) bit for bit where e rounds to a weight above 0, -22.2 < x <= 0; there
// n = rint(x log2 e) comes from an addition that rounds at the unit, and the scaling by 2^n, n >=
// -33, is exact.  Below, 0: no weight, and no tie that could tell.
__device__ __forceinline__ unsigned exp_key(float x) {
  if (!(x > -22.2f)) return 0u;
  const float t = __fadd_rn(__fmul_rn(x, __int_as_float(0x3fb8aa3b)), 12582912.0f);
  const float n = __fsub_rn(t, 12582912.0f);
  const float r = __fsub_rn(__fsub_rn(x, __fmul_rn(n, __int_as_float(0x3f318000))),
                            __fmul_rn(n, __int_as_float((int)0xb95e8083u)));
  float p = __int_as_float(0x39506967);
  p = __fadd_rn(__fmul_rn(p, r), __int_as_float(0x3ab743ce));
  p = __fadd_rn(__fmul_rn(p, r), __int_as_float(0x3c088908));
  p = __fadd_rn(__fmul_rn(p, r), __int_as_float(0x3d2aa9c1));
  p = __fadd_rn(__fmul_rn(p, r), __int_as_float(0x3e2aaaaa));
  p = __fadd_rn(__fmul_rn(p, r), __int_as_float(0x3f000000));
  const float y = __fadd_rn(__fadd_rn(1.0f, r), __fmul_rn(__fmul_rn(r, r), p));
  return __float_as_uint(y) + (__float_as_uint(t) << 23);
}

__device__ __forceinline__ void cluster_sync() {
  cluster_arrive_release();
  cluster_wait_acquire();
}
__device__ __forceinline__ void red_cluster(uint32_t addr, unsigned v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v)
               : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ u64 ld_cluster(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}

// What the first CTA publishes of a level: the bin, and the counts and sums above it.
struct Found {
  u64 bin, count, sum;
};

struct Shared {
  unsigned cnt[kBins], lo[kBins], hi[kBins];     // this CTA's bins: sums in 16-bit halves
  unsigned mcnt[kBins], mlo[kBins], mhi[kBins];  // the cluster's (first CTA): 24-bit parts
  u64 warp_sum[kWarps];
  unsigned warp_cnt[kWarps];
  Found found[2];  // by turns: one is read while the next is written
  u64 total;       // the weights of the level scanned last
  unsigned floor_bin, floor_count, n_local, n_list;  // the candidates' lowest bin, their number
  u64 part[kMaxCluster][3];  // of each CTA: the weights above the cut, their number, the ties
  float top[kMaxCluster];
  int first[kMaxCluster];
  float wtop[kWarps];
  u64 chunk_w[8][kWarps];  // of 128 consecutive tokens
  unsigned chunk_e[8][kWarps];
  u64 pick[3];
};

// Sum over the CTA, in every thread.
__device__ u64 cta_sum(u64 v, Shared &s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.warp_sum[threadIdx.x / 32] = v;
  __syncthreads();
  v = s.warp_sum[threadIdx.x % 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Descending sort of v over the first n threads, which alone call it (a power of two from 32 to
// 1024).
__device__ u64 cta_sort(u64 v, int n, u64 *buf) {
  const int tid = threadIdx.x;
#pragma unroll 1
  for (int size = 2; size <= n; size <<= 1)
#pragma unroll 1
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      u64 other;
      if (stride >= 32) {
        asm volatile("bar.sync 1, %0;" ::"r"(n) : "memory");
        buf[tid] = v;
        asm volatile("bar.sync 1, %0;" ::"r"(n) : "memory");
        other = buf[tid ^ stride];
      } else {
        other = __shfl_xor_sync(0xFFFFFFFFu, v, stride);
      }
      const bool larger = ((tid & stride) == 0) == ((tid & size) == 0);
      v = larger == (v > other) ? v : other;
    }
  return v;
}

// Inclusive sum of v over the threads.
__device__ u64 cta_scan(u64 v, Shared &s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) s.warp_sum[warp] = v;
  __syncthreads();
  u64 b = lane < warp ? s.warp_sum[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) b += __shfl_xor_sync(0xFFFFFFFFu, b, o);
  return v + b;
}

// A thread's tokens: in its registers, or in shared memory, its own words.
template <int IPT, bool SHARED>
struct Keys {
  unsigned r[IPT];
  __device__ __forceinline__ unsigned &operator[](int i) { return r[i]; }
};
template <int IPT>
struct Keys<IPT, true> {
  __device__ __forceinline__ unsigned &operator[](int i) {
    extern __shared__ unsigned shared_keys[];
    return shared_keys[i * kThreads + threadIdx.x];
  }
};

// A cluster per row; IPT tokens per thread, in quads: quad j of thread t is 4 (j 1024 + t).
template <int IPT, bool SHARED, int PER_SM>
__global__ void __launch_bounds__(kThreads, PER_SM)
    sample_kernel(apx_sample_args a, int ctas) {
  __shared__ Shared s;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int rank = blockIdx.x % ctas;
  const size_t row = blockIdx.x / ctas;
  const unsigned vocab = (unsigned)a.vocab;
  const unsigned per = (vocab + 4 * ctas - 1) / (4 * ctas) * 4;  // tokens of a CTA
  const unsigned v0 = min(per * rank, vocab), v1 = min(v0 + per, vocab);
  pdl_launch_dependents();
  s.cnt[tid] = s.lo[tid] = s.hi[tid] = s.mcnt[tid] = s.mlo[tid] = s.mhi[tid] = 0;
  if (tid == 0) s.n_local = s.n_list = 0;
  cluster_arrive_release();  // this CTA runs, its bins are zero
  pdl_wait();
  const float *x = a.d_logits + row * a.ld;
  const float temp = a.d_temperature ? a.d_temperature[row] : 1.0f;
  const int k = a.d_top_k ? a.d_top_k[row] : 0;
  const float top_p = a.d_top_p ? a.d_top_p[row] : 1.0f;
  const float min_p = a.d_min_p ? a.d_min_p[row] : 0.0f;
  const float u = a.d_u[row];

  // ---- the logits, once; tokens past the end are excluded ones ----
  Keys<IPT, SHARED> key;  // the logit's bits, then e's
  const bool quads = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < IPT / 4; j++) {
    const unsigned i = v0 + 4 * (j * kThreads + tid);
    float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (quads && i + 4 <= v1) {
      f = *reinterpret_cast<const float4 *>(x + i);  // not the read-only path: pdl_wait's data
    } else {
      if (i < v1) f.x = x[i];
      if (i + 1 < v1) f.y = x[i + 1];
      if (i + 2 < v1) f.z = x[i + 2];
      if (i + 3 < v1) f.w = x[i + 3];
    }
    top = fmaxf(top, fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)));
    key[4 * j] = __float_as_uint(f.x), key[4 * j + 1] = __float_as_uint(f.y);
    key[4 * j + 2] = __float_as_uint(f.z), key[4 * j + 3] = __float_as_uint(f.w);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (lane == 0) s.wtop[warp] = top;
  __syncthreads();
  top = s.wtop[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  // every CTA's maximum to every CTA
  cluster_wait_acquire();
  if (tid < ctas)
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_map(&s.top[rank], tid)), "f"(top)
                 : "memory");
  cluster_sync();
  for (int i = 0; i < ctas; i++) top = fmaxf(top, s.top[i]);

  if (top == -INFINITY) {  // nothing left
    if (rank == 0 && tid == 0) {
      a.d_token[row] = -1;
      if (a.d_prob) a.d_prob[row] = 0.0f;
      if (a.d_kept) a.d_kept[row] = 0;
    }
    return;
  }
  if (!(temp > 0.0f)) {  // the largest logit, lowest index
    int at = INT_MAX;
#pragma unroll
    for (int i = IPT - 1; i >= 0; i--)
      if (__uint_as_float(key[i]) == top) at = (int)(v0 + 4 * (i / 4 * kThreads + tid) + i % 4);
    at = __reduce_min_sync(0xFFFFFFFFu, at);
    if (lane == 0) s.warp_cnt[warp] = (unsigned)at;
    __syncthreads();
    at = __reduce_min_sync(0xFFFFFFFFu, (int)s.warp_cnt[lane]);
    if (tid == 0)
      asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(cluster_map(&s.first[rank], 0)),
                   "r"(at)
                   : "memory");
    cluster_sync();
    if (rank == 0 && tid == 0) {
      for (int i = 0; i < ctas; i++) at = min(at, s.first[i]);
      a.d_token[row] = at;
      if (a.d_prob) a.d_prob[row] = 1.0f;
      if (a.d_kept) a.d_kept[row] = 1;
    }
    return;
  }

  // ---- e ----
  const float inv = __frcp_rn(temp);
#pragma unroll
  for (int i = 0; i < IPT; i++) {
    const float l = __uint_as_float(key[i]);
    key[i] = !(l > -INFINITY) ? 0u  // NaN and -inf
             : l == top       ? kTopKey
                              : exp_key(__fmul_rn(__fsub_rn(l, top), inv));
  }

  const bool by_k = k > 0 && (unsigned)k < vocab, by_p = top_p < 1.0f;
  const double min_w = (double)min_p * (double)kWeightOne;
  // (double)w < min_w for whole w: w below the next whole number
  const unsigned least = min_w > 0.0 ? (unsigned)fmin(ceil(min_w), 4294967295.0) : 0u;
  // tokens with key > cut stay, and the first `ties` of those with key == cut
  unsigned cut = 0;
  u64 ties = ULLONG_MAX;

  // One level's histogram over the keys in (floor, ..) whose bits above shift + 10 are `prefix`,
  // scanned by the first CTA from the top; thread t there holds bin 1023 - t: `count` and `sum`
  // of the bins above it, `own_count` and `own_sum` its own.
  u64 count = 0, sum = 0, own_count = 0, own_sum = 0, kept1 = 0, kept_own1 = 0;
  auto level = [&](int shift, unsigned prefix, unsigned floor, bool counts, bool sums, u64 lump,
                   unsigned lump_key) {
#pragma unroll
    for (int i = 0; i < IPT; i++) {
      const unsigned v = key[i];
      if (v > floor && (shift == 20 || v >> (shift + 10) == prefix)) {
        const unsigned b = v >> shift & (kBins - 1);
        if (counts) atomicAdd(&s.cnt[b], 1u);
        if (sums) {
          const unsigned w = weight_of(v);
          atomicAdd(&s.lo[b], w & 0xFFFFu);
          atomicAdd(&s.hi[b], w >> 16);
        }
      }
    }
    __syncthreads();
    // this CTA's bin to the first CTA's: a sum below 2^47 as two parts of 24 bits
    const unsigned c = s.cnt[tid];
    const u64 w = ((u64)s.hi[tid] << 16) + s.lo[tid];
    if (c) red_cluster(cluster_map(&s.mcnt[tid], 0), c);
    if (w) {
      red_cluster(cluster_map(&s.mlo[tid], 0), (unsigned)w & 0xFFFFFFu);
      red_cluster(cluster_map(&s.mhi[tid], 0), (unsigned)(w >> 24));
    }
    s.cnt[tid] = s.lo[tid] = s.hi[tid] = 0;
    cluster_sync();
    if (rank == 0) {
      const int b = kBins - 1 - tid;
      own_count = s.mcnt[b];
      own_sum = ((u64)s.mhi[b] << 24) + s.mlo[b];
      s.mcnt[b] = s.mlo[b] = s.mhi[b] = 0;
      if (lump && (shift == 20 || lump_key >> (shift + 10) == prefix) &&
          (lump_key >> shift & (kBins - 1)) == (unsigned)b)
        own_sum += lump;
      u64 rc = own_count, rs = own_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned tc = __shfl_up_sync(0xFFFFFFFFu, (unsigned)rc, o);
        const u64 ts = __shfl_up_sync(0xFFFFFFFFu, rs, o);
        if (lane >= o) rc += tc, rs += ts;
      }
      if (lane == 31) s.warp_cnt[warp] = (unsigned)rc, s.warp_sum[warp] = rs;
      __syncthreads();
      unsigned bc = lane < warp ? s.warp_cnt[lane] : 0;
      u64 bs = lane < warp ? s.warp_sum[lane] : 0;
      bc = __reduce_add_sync(0xFFFFFFFFu, bc);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) bs += __shfl_xor_sync(0xFFFFFFFFu, bs, o);
      count = rc + bc - own_count;
      sum = rs + bs - own_sum;
      if (tid == kThreads - 1) s.total = sum + own_sum;
    }
  };
  // The first CTA's word on the level just scanned, to every thread of the cluster.
  int turn = 0;
  auto publish = [&](bool crosses, u64 bin, u64 over_count, u64 over_sum) {
    turn ^= 1;
    if (rank == 0 && crosses) s.found[turn] = Found{bin, over_count, over_sum};
    cluster_sync();
    const uint32_t f = cluster_map(&s.found[turn], 0);
    Found r;
    r.bin = ld_cluster(f);
    r.count = ld_cluster(f + 8);
    r.sum = ld_cluster(f + 16);
    return r;
  };
  auto level_total = [&] { return ld_cluster(cluster_map(&s.total, 0)); };

  if (by_k || by_p) {
    level(20, 0, 0, true, !by_k, 0, 0);  // with top-k the sums can wait: a list has its own
    {
      // the lowest bin that can hold a token that stays, and the tokens from it up
      if (rank == 0) {
        if (tid == kThreads - 1) s.floor_bin = 0, s.pick[2] = 0;
        __syncthreads();
        const double limit = (double)top_p * (double)s.total;
        const bool crosses = by_k ? count < (u64)k && count + own_count >= (u64)k
                                  : (double)sum < limit && (double)(sum + own_sum) >= limit;
        if (crosses) s.floor_bin = kBins - 1 - tid, s.pick[2] = by_k;
        if (!by_k && limit <= 0.0 && tid == 0) s.floor_bin = kTopKey >> 20;
        __syncthreads();
        // tokens below min-p stay out, unless top-p's total needs those that top-k keeps
        unsigned f = s.floor_bin;
        if (!(by_k && by_p) && least > 1)
          f = max(f, __float_as_uint((float)(least - 1) / kWeightOne * 0.999999f) >> 20);
        f = min(f, kTopKey >> 20);
        __syncthreads();
        if (kBins - 1 - tid == (int)f) {
          if (s.floor_bin != f) s.pick[2] = 0;  // the bin is not where top-k cuts
          s.floor_bin = f;
          s.floor_count = (unsigned)(count + own_count);
          s.pick[0] = count;
        }
        __syncthreads();
      }
      Found c = publish(tid == 0, rank ? 0 : s.floor_bin, rank ? 0 : s.floor_count,
                        rank ? 0 : s.pick[2]);
      unsigned low = (unsigned)c.bin << 20;  // the lowest key of the candidates
      if (c.count > kThreads && c.sum) {
        // too many, most of them often in the bin where top-k cuts: ten bits more of those
        const u64 over = s.pick[0];
        kept1 = count, kept_own1 = own_count;
        level(10, (unsigned)c.bin, 0, true, false, 0, 0);
        const bool crosses = over + count < (u64)k && over + count + own_count >= (u64)k;
        c = publish(crosses, kBins - 1 - tid, over + count + own_count, 0);
        low |= (unsigned)c.bin << 10;
        count = kept1, own_count = kept_own1;
      }
      if (c.count <= kThreads) {
        // to a list here, then to the first CTA's
        u64 *local = reinterpret_cast<u64 *>(s.cnt), *list = reinterpret_cast<u64 *>(s.mcnt);
#pragma unroll
        for (int i = 0; i < IPT; i++)
          if (key[i] && key[i] >= low)
            local[atomicAdd(&s.n_local, 1u)] =
                (u64)key[i] << 32 | (0xFFFFFFFFu - (v0 + 4 * (i / 4 * kThreads + tid) + i % 4));
        __syncthreads();
        const unsigned mine = s.n_local;
        if (tid == 0 && mine) {
          unsigned at;
          asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;"
                       : "=r"(at)
                       : "r"(cluster_map(&s.n_list, 0)), "r"(mine)
                       : "memory");
          s.floor_count = at;
        }
        __syncthreads();
        if ((unsigned)tid < mine) st_cluster(cluster_map(list + s.floor_count + tid, 0), local[tid]);
        cluster_sync();
        if (rank) return;
        const int nc = (int)c.count;
        int n = 32;
        while (n < nc) n <<= 1;
        u64 v = tid < nc ? list[tid] : 0;
        if (tid < n) v = cta_sort(v, n, local);
        const unsigned w = tid < nc ? weight_of((unsigned)(v >> 32)) : 0u;
        u64 run = cta_scan(w, s);
        // the weights that top-p counts: of the first k, or of all
        u64 all = s.total;
        if (by_k && by_p) {  // fewer than k have weight: all of them are in the list
          if (tid == min(k, nc) - 1) s.pick[0] = run;
          __syncthreads();
          all = s.pick[0];
        }
        const bool stays = tid < nc && (!by_k || tid < k) && w >= least && w > 0 &&
                           (!by_p || tid == 0 ||
                            (double)(run - w) < (double)top_p * (double)all);
        const int kept = __syncthreads_count(stays);
        if (kept == 0) {
          if (tid == 0) {
            a.d_token[row] = -1;
            if (a.d_prob) a.d_prob[row] = 0.0f;
            if (a.d_kept) a.d_kept[row] = 0;
          }
          return;
        }
        // in the vocabulary's order: the lowest index is the largest of the complements
        v = stays ? (v & 0xFFFFFFFFull) << 32 | w : 0;
        if (tid < n) v = cta_sort(v, n, local);
        const u64 mine_w = v & 0xFFFFFFFFull;
        run = cta_scan(mine_w, s);
        if (tid == kThreads - 1) s.pick[1] = run;
        __syncthreads();
        const u64 total = s.pick[1];
        u64 aim = u > 0.0f ? (u64)((double)u * (double)total) : 0;
        if (aim >= total) aim = total - 1;
        if (mine_w && run - mine_w <= aim && aim < run) {
          a.d_token[row] = (int)(0xFFFFFFFFu - (unsigned)(v >> 32));
          if (a.d_prob) a.d_prob[row] = (float)((double)mine_w / (double)total);
          if (a.d_kept) a.d_kept[row] = kept;
        }
        return;
      }
    }
    if (by_k && by_p) level(20, 0, 0, true, true, 0, 0);
    const u64 sum1 = sum, own1 = own_sum;  // kept for top-p
    u64 all = 0;         // the weights of all tokens that stay
    unsigned bin_k = 0;  // the first ten bits of the cut
    Found f;
    if (by_k) {
      // key 0 is not counted: with fewer than k others the cut stays at 0
      u64 over = 0, over_sum = 0;
      unsigned prefix = 0;
      bool short_of_k = false;
      for (int shift = 20; shift >= 0; shift -= 10) {
        if (shift < 20) level(shift, prefix, 0, true, by_p, 0, 0);
        const bool few = shift == 20 && tid == kThreads - 1 && count + own_count < (u64)k;
        const bool crosses = over + count < (u64)k && over + count + own_count >= (u64)k;
        f = publish(crosses || few, few ? ULLONG_MAX : kBins - 1 - tid, over + count,
                    over_sum + sum);
        if (f.bin == ULLONG_MAX) {
          short_of_k = true;
          all = level_total();
          break;
        }
        if (shift == 20) bin_k = (unsigned)f.bin;
        over = f.count;
        over_sum = f.sum;
        prefix = prefix << 10 | (unsigned)f.bin;
      }
      if (!short_of_k) {
        cut = prefix;
        ties = (u64)k - over;
        all = over_sum + ties * weight_of(cut);
      }
    }
    if (by_p) {
      const bool cutting = cut != 0;
      if (!by_k) {  // the total is the first CTA's
        publish(false, 0, 0, 0);
        all = level_total();
      }
      const double limit = (double)top_p * (double)all;
      unsigned t = kTopKey;
      u64 over = 0, n = 1;
      if (limit > 0.0) {
        const u64 lump = cutting ? ties * weight_of(cut) : 0;
        unsigned prefix = 0;
        for (int shift = 20; shift >= 0; shift -= 10) {
          u64 own = own_sum;
          if (shift == 20) {
            const unsigned b = kBins - 1 - tid;
            sum = sum1;
            own = !cutting || b > bin_k ? own1 : b == bin_k ? all - sum1 : 0;
            if (cutting && b < bin_k) sum = all;
          } else {
            level(shift, prefix, cut, false, true, lump, cut);
            own = own_sum;
          }
          const bool crosses =
              (double)(over + sum) < limit && (double)(over + sum + own) >= limit;
          f = publish(crosses, kBins - 1 - tid, 0, over + sum);
          over = f.sum;
          prefix = prefix << 10 | (unsigned)f.bin;
        }
        t = prefix;
        // of the tokens at t, those before which less than limit was summed
        const u64 each = weight_of(t);
        n = (u64)((limit - (double)over) / (double)each);
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
  }

  // ---- the weights that stay, of each CTA to every CTA ----
  const unsigned cut_w = cut ? weight_of(cut) : 0u, tie_w = cut_w >= least ? cut_w : 0u;
  auto above = [&](unsigned v) {  // its weight if it stays for being above the cut
    const unsigned w = v > cut ? weight_of(v) : 0u;
    return w >= least ? w : 0u;
  };
  u64 w_above = 0, n_pair = 0;  // counts: above the cut in the low half, ties in the high
#pragma unroll
  for (int i = 0; i < IPT; i++) {
    const unsigned w = above(key[i]);
    w_above += w;
    n_pair += (u64)(w != 0) + ((u64)(cut != 0 && key[i] == cut) << 32);
  }
  w_above = cta_sum(w_above, s);
  n_pair = cta_sum(n_pair, s);
  if (tid < ctas) {
    const uint32_t at = cluster_map(&s.part[rank][0], tid);
    st_cluster(at, w_above);
    st_cluster(at + 8, n_pair & 0xFFFFFFFFull);
    st_cluster(at + 16, n_pair >> 32);
  }
  cluster_sync();
  u64 total = 0, kept = 0, before = 0, eq_before = 0, eq_seen = 0;
  for (int i = 0; i < ctas; i++) {
    const u64 eq = s.part[i][2];
    const u64 left = ties > eq_seen ? ties - eq_seen : 0;
    const u64 some = min(eq, left);  // of this CTA's ties, those that stay
    if (i == rank) {
      before = total;
      eq_before = eq_seen;
    }
    total += s.part[i][0] + some * tie_w;
    kept += s.part[i][1] + (tie_w ? some : 0);
    eq_seen += eq;
  }
  if (total == 0) {
    if (rank == 0 && tid == 0) {
      a.d_token[row] = -1;
      if (a.d_prob) a.d_prob[row] = 0.0f;
      if (a.d_kept) a.d_kept[row] = 0;
    }
    return;
  }
  u64 aim = u > 0.0f ? (u64)((double)u * (double)total) : 0;
  if (aim >= total) aim = total - 1;
  if (rank == 0 && tid == 0 && a.d_kept) a.d_kept[row] = (int)kept;
  const u64 eq_left = ties > eq_before ? ties - eq_before : 0;  // ties that stay from here on
  const u64 here = w_above + min(s.part[rank][2], eq_left) * tie_w;
  if (aim < before || aim >= before + here) return;

  // ---- the token: in this CTA, by runs of 128, then by lane ----
#pragma unroll
  for (int j = 0; j < IPT / 4; j++) {
    u64 w = 0;
    unsigned e = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w += above(key[4 * j + i]);
      e += cut != 0 && key[4 * j + i] == cut;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    e = __reduce_add_sync(0xFFFFFFFFu, e);
    if (lane == 0) s.chunk_w[j][warp] = w, s.chunk_e[j][warp] = e;
  }
  __syncthreads();
  if (warp == 0) {
    u64 run = before, eq = 0;
    for (int j = 0; j < IPT / 4; j++) {
      const u64 w = s.chunk_w[j][lane];
      const unsigned e = s.chunk_e[j][lane];
      unsigned ep = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xFFFFFFFFu, ep, o);
        if (lane >= o) ep += t;
      }
      const u64 e0 = eq + ep - e;  // ties of this CTA before the run
      const u64 some = min((u64)e, eq_left > e0 ? eq_left - e0 : 0);
      u64 mine = w + some * tie_w, wp = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xFFFFFFFFu, wp, o);
        if (lane >= o) wp += t;
      }
      const u64 w0 = run + wp - mine;
      if (w0 <= aim && aim < w0 + mine) {
        s.pick[0] = (u64)(j * 32 + lane);
        s.pick[1] = w0;
        s.pick[2] = e0;
      }
      run += __shfl_sync(0xFFFFFFFFu, wp, 31);
      eq += __shfl_sync(0xFFFFFFFFu, ep, 31);
    }
  }
  __syncthreads();
  if (warp != (int)(s.pick[0] % 32)) return;
  const int jj = (int)(s.pick[0] / 32);
#pragma unroll
  for (int j = 0; j < IPT / 4; j++) {
    if (j != jj) continue;
    unsigned e = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) e += cut != 0 && key[4 * j + i] == cut;
    unsigned ep = e;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned t = __shfl_up_sync(0xFFFFFFFFu, ep, o);
      if (lane >= o) ep += t;
    }
    u64 at = s.pick[2] + ep - e;
    unsigned w[4];
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      w[i] = above(key[4 * j + i]);
      if (cut != 0 && key[4 * j + i] == cut) {
        if (at < eq_left) w[i] = tie_w;
        at++;
      }
      mine += w[i];
    }
    u64 wp = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xFFFFFFFFu, wp, o);
      if (lane >= o) wp += t;
    }
    u64 w0 = s.pick[1] + wp - mine;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (w0 <= aim && aim < w0 + w[i]) {
        a.d_token[row] = (int)(v0 + 4 * (j * kThreads + tid) + i);
        if (a.d_prob) a.d_prob[row] = (float)((double)w[i] / (double)total);
      }
      w0 += w[i];
    }
  }
}

template <int IPT, bool SHARED, int PER_SM>
cudaError_t launch(const apx_sample_args &a, int ctas, cudaStream_t stream) {
  auto kern = sample_kernel<IPT, SHARED, PER_SM>;
  if (SHARED) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               IPT * kThreads * 4);
    if (e != cudaSuccess) return e;
  }
  if (ctas > 8) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.rows * ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = SHARED ? IPT * kThreads * 4 : 0;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_allowed() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a, ctas);
}

}  // namespace

cudaError_t launch_sample(const apx_sample_args &a, int sms, cudaStream_t stream) {
  // the fewest CTAs that hold the row in 20 tokens a thread, in 32 past 16 x 20; twice as many while
  // that makes 64 CTAs at most (four rows of 151936: 8 CTAs a row 16.2 us, 16 CTAs 13.9; eight rows,
  // whose clusters of 16 no longer all run at once: 16.3 and 23.2; five to seven would gain still)
  int ctas = 1;
  while (ctas < kMaxCluster && (size_t)ctas * kThreads * 20 < a.vocab) ctas *= 2;
  if (ctas < kMaxCluster && a.rows * ctas * 2 <= 64 && a.vocab > 8192 * (size_t)ctas) ctas *= 2;
  const size_t per = ((a.vocab + 4 * ctas - 1) / (4 * ctas) * 4 + kThreads - 1) / kThreads;
  if (per <= 4) return launch<4, false, 1>(a, ctas, stream);
  // more CTAs than SMs: two an SM, one's barriers behind the other's work (a nucleus with min-p: 64
  // rows of 151936 81.5 us with one an SM, 68.2 with two; 512 rows of 32003 135 and 102, with top-k
  // 119 and 88; 24 rows of 151936 43.7 and 42.4)
  if (a.rows * ctas > (size_t)sms && per <= 20)
    return per <= 12 ? launch<12, true, 2>(a, ctas, stream) : launch<20, true, 2>(a, ctas, stream);
  // more than 12 tokens a thread leave the levels too few registers (16 rows of 151936, a nucleus of
  // thousands: 60 us in registers, 54 in shared memory; one row of 524288, top-k 50: 20.0 and 21.0)
  if (per <= 12) return launch<12, false, 1>(a, ctas, stream);
  if (per <= 20) return launch<20, true, 1>(a, ctas, stream);
  return launch<32, true, 1>(a, ctas, stream);
}

}  // namespace apx
