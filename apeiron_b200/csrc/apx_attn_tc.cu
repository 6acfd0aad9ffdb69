// apx_attn_tc.cu — attention over the paged 4-bit cache for prompts: 128 query rows at a time on
// the tensor cores (apx_attn.cu serves few rows, and f32).
//
// A CTA holds 128 query rows of one KV head (a token's group of heads are neighbouring rows) and
// takes its keys 128 at a time: S = Q K^T into TMEM, the softmax warps turn S into probabilities
// in place (f16), O += P V with P read from TMEM.  Warps 4-7 unpack the next keys and values from
// the cache's pages to f16 operands in shared memory (exact: d (c - 8) fits f16), registers
// holding the bytes in flight.  Two CTAs share an SM, so that one's products run under the
// other's softmax.
//
// What bounds it, per 128 x 128 step at D = 128: the products 1024 cycles, the exponentials 1024
// (16 a cycle), shared memory 1280 (S reads both operands, P V one, the unpacked keys and values
// go in once).
//
// The running maximum is a stale one: O (in TMEM) and the row sum turn only when a row's maximum
// has grown by more than 2^8 since the last turn; probabilities are held at 2^6 e^(s - m), at most
// 2^14.  A row of q is scaled by a power of two to the top of f16's range: bf16 and f16 both fit.
//
// K's dims are stored in the order the unpacking yields them (0 4 1 5 2 6 3 7 of every eight), Q's
// the same.
#include <cuda_bf16.h>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_kv4.cuh"
#include "apx_pack.cuh"
#include "apx_tc.cuh"

namespace apx {

namespace {

constexpr int kRows = 128, kKeys = 128;
constexpr int kThreads = 288;       // 4 softmax warps, 4 unpacking warps, 1 that issues products
constexpr float kStale = 8.0f;      // log2 of how far a row's maximum may outgrow the stale one
constexpr float kOffset = 6.0f;     // probabilities are held at 2^6 e^(s - m)
constexpr int kTmemCols = 256;      // S (then P) in columns 0-127, O from 128 on
constexpr int kOCol = 128;

// K-major operands in the 128-byte swizzle: rows of 64 f16, 8-row groups 1024 bytes apart.
constexpr uint64_t kDesc = ((uint64_t)(16 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
                           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
// kind::f16: D f32 (1) at bits 4-5, A and B f16 (0), N >> 3 at bits 17-22, M >> 4 at bits 24-28.
__host__ __device__ constexpr uint32_t idesc_f16(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

template <int D>
struct Smem {
  // operands in panels of 64 columns: Q and K by dims, V^T by keys
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kRows * D * 2;
  static constexpr int kV = kK + kKeys * D * 2;
  static constexpr int kCq = kV + kKeys * D * 2;
  static constexpr int kBars = kCq + kRows * 4;
  static constexpr int kBytes = kBars + 64 + 1024;  // and the base's alignment
};

// 16-byte chunk c (of 8) of row r in a panel of 128-byte rows.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

template <int D>
__global__ void __launch_bounds__(kThreads, 2) attn_tc_kernel(AttnArgs p) {
  using L = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint64_t *k_full = bars, *v_full = bars + 1, *s_full = bars + 2, *p_full = bars + 3,
           *o_full = bars + 4;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 5);
  float *s_cq = reinterpret_cast<float *>(smem + L::kCq);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int seq = blockIdx.x / p.kv_heads, head = blockIdx.x % p.kv_heads;

  pdl_launch_dependents();
  pdl_wait();
  SeqRows<kRows, kKeys> q;
  q.load(p, seq);
  if (q.bad && blockIdx.y == 0 && head == 0 && tid == 0)
    attn_refuse(p, seq, APX_ERR_INVALID_ARGUMENT);
  const int blk = (int)(gridDim.y - 1 - blockIdx.y);  // the longest first
  if (blk >= q.nblk) return;
  int end, sink, from;
  q.range(p, blk, end, sink, from);
  const int n = sink + max(q.steps_to(end) - from, 0);
  auto key_of = [&](int j) { return (j < sink ? j : j - sink + from) * kKeys; };

  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    if (lane == 0) {
      mbar_init(k_full, 128);
      mbar_init(v_full, 128);
      mbar_init(s_full, 1);
      mbar_init(p_full, 128);
      mbar_init(o_full, 1);
    }
  } else {
    // ---- Q: two threads a row ----
    const int row = tid / 2, half = tid % 2;
    const int r = blk * kRows + row;
    uint4 x[D / 16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) x[i] = make_uint4(0, 0, 0, 0);
    if (r < q.rows) {
      const uint4 *src = reinterpret_cast<const uint4 *>(
          static_cast<const uint16_t *>(p.q) + (unsigned long long)(q.first + r / p.group) * p.ldq +
          (unsigned long long)(head * p.group + r % p.group) * D + half * (D / 2));
#pragma unroll
      for (int i = 0; i < D / 16; i++) x[i] = src[i];
    }
    const bool bf16 = p.type == APX_DTYPE_BF16;
    auto pair = [&](uint32_t w) {
      return bf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u))
                  : __half22float2(u2h(w));
    };
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 f = pair(w[j]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    const int e = row_exponent(top);
    const float up = p.scale < 0.0f ? -pow2(9 - e) : pow2(9 - e);  // so that scores grow with S
    if (half == 0) s_cq[row] = fabsf(p.scale) * 1.44269504088896341f * pow2(e - 9);
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
      const float2 a = pair(x[i].x), b = pair(x[i].y), c = pair(x[i].z), d = pair(x[i].w);
      auto two = [&](float u, float v) { return h2u(__floats2half2_rn(u * up, v * up)); };
      const int chunk = half * (D / 16) + i;
      *reinterpret_cast<uint4 *>(smem + L::kQ + chunk / 8 * (kRows * 128) +
                                 swizzled(row, chunk % 8)) =
          make_uint4(two(a.x, c.x), two(a.y, c.y), two(b.x, d.x), two(b.y, d.y));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp < 4) {
    // ---- softmax: one row a thread ----
    const int row = tid, r = blk * kRows + row;
    const bool live = r < q.rows;
    const int pos = q.p0 + r / p.group;
    const int hi = live ? min(pos, end - 1) : -1, lo = p.window ? pos - p.window + 1 : 0;
    // keys that every live row of the block sees
    const int all_hi = min(q.p0 + blk * kRows / p.group, end - 1);
    const int all_lo =
        p.window ? q.p0 + min((blk + 1) * kRows - 1, q.rows - 1) / p.group - p.window + 1 : 0;
    const float cq = s_cq[row];
    const uint32_t trow = tmem + ((uint32_t)(32 * warp) << 16);
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < n; j++) {
      const int key = key_of(j);
      ok = ok && mbar_wait(s_full, j & 1);
      // the product before it was complete by then: this keeps the parity of the last wait right
      if (j > 0) ok = ok && mbar_wait(o_full, (j - 1) & 1);
      __syncwarp();
      tc_fence_after();
      const bool masked = key + kKeys - 1 > all_hi || (key < all_lo && key + kKeys > p.sinks);
      auto seen = [&](int i) { return i <= hi && (i >= lo || i < p.sinks); };
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; c += 2) {
        uint32_t s0[32], s1[32];
        tmem_ld32_nowait(trow + 32 * c, s0);
        tmem_ld32_nowait(trow + 32 * c + 32, s1);
        tmem_wait_ld();
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; i++) {
            if (seen(key + 32 * c + i)) top = fmaxf(top, __uint_as_float(s0[i]));
            if (seen(key + 32 * c + 32 + i)) top = fmaxf(top, __uint_as_float(s1[i]));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i++)
            top = fmaxf(top, fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
        }
      }
      const float now = top == -INFINITY ? -INFINITY : top * cq;
      const bool grew = now > m + kStale || (m == -INFINITY && now > -INFINITY);
      if (__any_sync(0xFFFFFFFFu, grew)) {
        // every product so far is complete: O may be read and written
        float f = 1.0f;
        if (grew) {
          f = m == -INFINITY ? 0.0f : ex2(m - now);
          m = now;
          l *= f;
        }
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16_nowait(trow + kOCol + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(trow + kOCol + c, o);
          }
        }
      }
      const float base = kOffset - (m == -INFINITY ? 0.0f : m);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t s[32], h[16];
        tmem_ld32_nowait(trow + 32 * c, s);
        tmem_wait_ld();
        float e[32];
#pragma unroll
        for (int i = 0; i < 32; i++) e[i] = ex2(fmaf(__uint_as_float(s[i]), cq, base));
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (!seen(key + 32 * c + i)) e[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
          l += e[2 * i] + e[2 * i + 1];
          h[i] = h2u(__floats2half2_rn(e[2 * i], e[2 * i + 1]));
        }
        tmem_st16(trow + 16 * c, h);
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full);
    }
    // ---- the output rows ----
    if (n > 0) ok = ok && mbar_wait(o_full, (n - 1) & 1);
    __syncwarp();
    tc_fence_after();
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *dst = static_cast<uint16_t *>(p.out) +
                    (unsigned long long)(q.first + r / p.group) * p.ldo +
                    (unsigned long long)(head * p.group + r % p.group) * D;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
      uint32_t o[16];
      if (n > 0) {
        tmem_ld16_nowait(trow + kOCol + c, o);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = 0;
      }
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float a = __uint_as_float(o[2 * i]) * inv, b = __uint_as_float(o[2 * i + 1]) * inv;
        if (p.type == APX_DTYPE_BF16) {
          __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
          w[i] = *reinterpret_cast<uint32_t *>(&v);
        } else {
          w[i] = h2u(__floats2half2_rn(a, b));
        }
      }
      if (live) {
        *reinterpret_cast<uint4 *>(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
        *reinterpret_cast<uint4 *>(dst + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    // ---- unpacking: thread t has token t of K, and of tile t / 16 of V the dims 64 mq + 16 i + g
    // and + 8 (four i) with all 16 tokens ----
    const int t = tid - 128, tile = t / kKvTile, g = t % 8, mq = t / 8 % 2;
    const bool has_v = D == 128 || mq == 0;
    const Unpack un;
    constexpr int K16 = D / 32;  // 16-byte loads of a token's K
    uint4 kraw[K16], vraw[4], vsc[4];
    __half ksc[D / 32];
    int page = -1, page_next = -1;
    const int *table = p.table + (size_t)seq * p.max_pages;
    auto find = [&](int j) {  // the page of this thread's tile at step j
      const int key = key_of(j) + tile * kKvTile;
      if (j >= n || key >= end) return -1;
      const int pg = table[key >> p.page_shift];
      if (pg >= 0 && pg < p.n_pages) return pg;
      attn_refuse(p, seq, APX_ERR_INVALID_ARGUMENT);
      return -1;
    };
    auto source = [&](int j, int pg) {
      const int key = key_of(j) + tile * kKvTile;
      return p.pages + ((unsigned long long)pg * p.kv_heads + head) * p.page_bytes +
             (unsigned)((key & ((1 << p.page_shift) - 1)) / kKvTile) * kv4_tile_bytes(D);
    };
    auto load_k = [&](int j) {
      if (page < 0) return;
      const uint8_t *src = source(j, page);
#pragma unroll
      for (int i = 0; i < K16; i++)
        kraw[i] = __ldg(reinterpret_cast<const uint4 *>(src + t % kKvTile * (D / 2)) + i);
#pragma unroll
      for (int i = 0; i < D / 32; i++)
        ksc[i] = __ldg(reinterpret_cast<const __half *>(src + kv4_ks_off(D)) + i * kKvTile +
                       t % kKvTile);
    };
    auto load_v = [&](int j) {
      if (page < 0 || !has_v) return;
      const uint8_t *src = source(j, page);
#pragma unroll
      for (int i = 0; i < 4; i++)
        vraw[i] = __ldg(reinterpret_cast<const uint4 *>(src + kv4_v_off(D)) + mq * 32 + g * 4 + i);
#pragma unroll
      for (int i = 0; i < 4; i++)  // two groups of 32 dims, 16 tokens each
        vsc[i] = __ldg(reinterpret_cast<const uint4 *>(src + kv4_vs_off(D)) + mq * 4 + i);
    };
    page = find(0);
    load_k(0);
    load_v(0);
    for (int j = 0; j < n; j++) {
      const int key = key_of(j);
      page_next = find(j + 1);
      if (j > 0) ok = ok && mbar_wait(s_full, (j - 1) & 1);  // K's last readers are done
      {
        const bool have = page >= 0 && key + t < end;
#pragma unroll
        for (int i = 0; i < K16; i++) {
          const uint32_t w[4] = {kraw[i].x, kraw[i].y, kraw[i].z, kraw[i].w};
          const __half2 sc = __half2half2(ksc[i]);  // 32 dims: one group
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int chunk = 4 * i + c;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (have)
              v = make_uint4(un.low2(w[c], sc), un.high2(w[c], sc), un.low2(w[c] >> 8, sc),
                             un.high2(w[c] >> 8, sc));
            *reinterpret_cast<uint4 *>(smem + L::kK + chunk / 8 * (kKeys * 128) +
                                       swizzled(t, chunk % 8)) = v;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(k_full);
      const int page_now = page;
      page = page_next;
      load_k(j + 1);
      if (j > 0) ok = ok && mbar_wait(o_full, (j - 1) & 1);  // V's last readers are done
      if (has_v) {
        const int first = key + tile * kKvTile;
        const bool have = page_now >= 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {  // dims 64 mq + 16 i + g and + 8
          uint32_t a[2][8];            // dim; tokens 2 k and 2 k + 1
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t w = i == 0 ? vraw[k].x : i == 1 ? vraw[k].y : i == 2 ? vraw[k].z : vraw[k].w;
            const uint4 lo4 = vsc[i / 2 * 2], hi4 = vsc[i / 2 * 2 + 1];
            const uint32_t s0 = k == 0 ? lo4.x : k == 1 ? lo4.y : k == 2 ? lo4.z : lo4.w;
            const uint32_t s1 = k == 0 ? hi4.x : k == 1 ? hi4.y : k == 2 ? hi4.z : hi4.w;
            a[0][k] = un.low2(w, u2h(s0));
            a[1][k] = un.high2(w, u2h(s0));
            a[0][4 + k] = un.low2(w >> 8, u2h(s1));
            a[1][4 + k] = un.high2(w >> 8, u2h(s1));
          }
          if (!have || first + kKvTile > end) {  // tokens past the last key may hold anything
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
              for (int k = 0; k < 8; k++) {
                if (!have || first + 2 * k >= end) a[h][k] &= 0xFFFF0000u;
                if (!have || first + 2 * k + 1 >= end) a[h][k] &= 0x0000FFFFu;
              }
          }
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int d = 64 * mq + 16 * i + g + 8 * h;
#pragma unroll
            for (int k = 0; k < 2; k++) {  // tokens 8 k .. 8 k + 7 of the tile
              const int chunk = tile * 2 + k;
              *reinterpret_cast<uint4 *>(smem + L::kV + chunk / 8 * (D * 128) +
                                         swizzled(d, chunk % 8)) =
                  make_uint4(a[h][4 * k], a[h][4 * k + 1], a[h][4 * k + 2], a[h][4 * k + 3]);
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(v_full);
      load_v(j + 1);
    }
  } else if (lane == 0) {
    // ---- the products ----
    const uint64_t qd = kDesc | (smem_addr(smem + L::kQ) >> 4);
    const uint64_t kd = kDesc | (smem_addr(smem + L::kK) >> 4);
    const uint64_t vd = kDesc | (smem_addr(smem + L::kV) >> 4);
    for (int j = 0; ok && j < n; j++) {
      ok = ok && mbar_wait(k_full, j & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < D / 16; k++) {
        const uint64_t at = (uint64_t)(k / 4 * (kRows * 128 >> 4) + k % 4 * 2);
        mma_f16_ss(tmem, qd + at, kd + at, idesc_f16(kKeys), k > 0);
      }
      mma_commit(s_full);
      ok = ok && mbar_wait(v_full, j & 1) && mbar_wait(p_full, j & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int k = 0; k < kKeys / 16; k++)
        mma_f16_ts(tmem + kOCol, tmem + 8 * k, vd + (uint64_t)(k / 4 * (D * 128 >> 4) + k % 4 * 2),
                   idesc_f16(D), j > 0 || k > 0);
      mma_commit(o_full);
    }
  }
  if (!ok) attn_refuse(p, seq, APX_ERR_DEVICE_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
}

template <int D>
cudaError_t launch(const AttnArgs &p, int max_q, cudaStream_t stream) {
  auto kern = attn_tc_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Smem<D>::kBytes);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.n_seqs * p.kv_heads,
                     (unsigned)(((long long)max_q * p.group + kRows - 1) / kRows));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<D>::kBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_allowed() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

// Prompts in 16-bit numbers: enough rows for half a block.
bool attn_tc_serves(const AttnArgs &p, int dim, int max_q) {
  const long long rows = (long long)max_q * p.group;
  return p.type != APX_DTYPE_F32 && rows >= 64 && rows <= 65535ll * kRows &&
         (long long)p.n_seqs * p.kv_heads < (1ll << 31) && (dim == 64 || dim == 128);
}

cudaError_t launch_attn_tc(const AttnArgs &p, int dim, int max_q, cudaStream_t stream) {
  return dim == 128 ? launch<128>(p, max_q, stream) : launch<64>(p, max_q, stream);
}

}  // namespace apx
