// apx_attn_tc.cu — attention over the paged 4-bit cache for prompts: query rows 128 at a time on
// the tensor cores (apx_attn.cu serves few rows, and f32).
//
// A CTA holds two tiles of 128 query rows of one KV head (a token's group of heads are neighbouring
// rows) and takes its keys 128 at a time: S = Q K^T into TMEM, four softmax warps a tile turn S
// into probabilities in place (f16), O += P V with P read from TMEM.  A tile's first softmax warp
// issues its products.  The tiles' softmaxes take turns: while one is in its softmax the other's
// products run (left to themselves they fall into step and both wait for their products: two
// prompts of up to 2048 66 us against 60.5 with turns; now 59, 585 TFLOP/s of what they see).
// Both read the same keys and values, which eight warps unpack from the cache's pages to f16
// operands in shared memory (exact: d (c - 8) fits f16), two buffers each, registers holding the
// bytes in flight.
//
// What bounds it, per 128 x 128 step of a tile at D = 128: the products 1024 cycles, the
// exponentials 1024 (16 a cycle), shared memory 1024 (S reads both operands, P V one, the unpacked
// keys and values go in for both tiles).
//
// A block's keys are shared by a cluster of up to eight CTAs where the blocks are too few for the
// GPU; each turns its part of the steps into rows of O, m and l, and every CTA joins its share of the
// block's rows from what the others have stored into its shared memory (in the CTAs' order: the same
// bits every time).
//
// The running maximum is a stale one: O (in TMEM) and the row sum turn only when a row's maximum
// has grown by more than 2^8 since the last turn; probabilities are held at 2^6 e^(s - m), at most
// 2^14, and rounded to f16's 11 bits for the product with V (their sum is not): below what the
// output's rounding costs.  A row of q is scaled by a power of two to the top of f16's range: bf16
// and f16 both fit.
//
// K's dims are stored in the order the unpacking yields them (0 4 1 5 2 6 3 7 of every eight), Q's
// the same.
#include <cuda_bf16.h>

#include <atomic>

#include "apx_common.cuh"
#include "apx_kernels.h"
#include "apx_kv4.cuh"
#include "apx_pack.cuh"
#include "apx_tc.cuh"

namespace apx {

namespace {

constexpr int kTile = 128, kRows = 2 * kTile, kKeys = 128;
constexpr int kThreads = 512;     // 8 softmax warps, 8 unpacking warps
constexpr int kUnpack = 256;      // unpacking threads
// Registers of a softmax and of an unpacking thread: together what the CTA is launched with (128 a
// thread, the launch bounds' limit, which the build's resource table shows).
constexpr int kSoftmaxRegs = 176, kUnpackRegs = 80;
static_assert((kSoftmaxRegs + kUnpackRegs) * 256 <= 128 * kThreads, "the launch's registers");
constexpr float kStale = 8.0f;    // log2 of how far a row's maximum may outgrow the stale one
constexpr float kUnseen = -1e30f;  // an unseen key's score
constexpr float kOffset = 6.0f;   // probabilities are held at 2^6 e^(s - m)
constexpr int kMaxSplit = 8;      // CTAs a block's keys are shared by at most
constexpr int kTmemCols = 512;    // S (then P) of the tiles in columns 0-255, O from 256 on

// K-major operands in the 128-byte swizzle: rows of 64 f16, 8-row groups 1024 bytes apart.
constexpr uint64_t kDesc = ((uint64_t)(16 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
                           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
// kind::f16: D f32 (1) at bits 4-5, A and B f16 (0), N >> 3 at bits 17-22, M >> 4 at bits 24-28.
__host__ __device__ constexpr uint32_t idesc_f16(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// Warps' rows that a CTA of `split` joins at most.
__host__ __device__ constexpr int join_warps(int split) { return (8 + split - 1) / split; }

template <int D>
struct Smem {
  // operands in panels of 64 columns: Q (both tiles) and K by dims, V^T by keys
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kRows * D * 2;
  static constexpr int kOne = kKeys * D * 2;  // a buffer of K or V
  static constexpr int kV = kK + 2 * kOne;
  static constexpr int kCq = kV + 2 * kOne;
  static constexpr int kBars = kCq + kRows * 4;
  static constexpr int kBytes = kBars + 128 + 1024;  // and the base's alignment
  // the parts that a join by `split` CTAs holds fit the operands' place
  static constexpr bool joins(int split) {
    return (split - 1) * 32 * join_warps(split) * (D * 4 + 8) <= kCq;
  }
};

// 16-byte chunk c (of 8) of row r in a panel of 128-byte rows.
__device__ __forceinline__ int swizzled(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Two f32 at a time.
__device__ __forceinline__ uint64_t pack2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Named barriers over n threads, those that wait and those that only arrive.
__device__ __forceinline__ void bar_sync_n(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive_n(int id, int n) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory");
}

__device__ __forceinline__ float as_f(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ float as_f(float x) { return x; }
template <typename A, typename B, typename C>
__device__ __forceinline__ float max3(A a, B b, C c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(as_f(a)), "f"(as_f(b)), "f"(as_f(c)));
  return m;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnArgs p, const int ctas) {
  using L = Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint64_t *k_full = bars, *v_full = bars + 2, *k_free = bars + 4, *v_free = bars + 6;
  uint64_t *s_full = bars + 8, *o_full = bars + 10;  // per tile
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 12);
  float *s_cq = reinterpret_cast<float *>(smem + L::kCq);
  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid / 32, 0);  // the same in every lane, and known to be
  const int rank = (int)blockIdx.x % ctas, item = (int)blockIdx.x / ctas;  // of the cluster
  const int seq = item / p.kv_heads, head = item % p.kv_heads;

  pdl_launch_dependents();
  pdl_wait();
  SeqRows<kRows, kKeys> q;
  q.load(p, seq);
  if (q.bad && blockIdx.y == 0 && head == 0 && rank == 0 && tid == 0)
    attn_refuse(p, seq, APX_ERR_INVALID_ARGUMENT);
  const int blk = (int)(gridDim.y - 1 - blockIdx.y);  // the longest first
  if (blk >= q.nblk) return;  // with its whole cluster
  int end, sink, low;
  q.range(p, blk, end, sink, low);
  const int from = low / kKeys;
  // this CTA's share of the block's steps: [j0, j0 + n)
  const int all = sink + max(q.steps_to(end) - from, 0);
  const int split = all >= ctas ? ctas : 1;  // too few steps: all of them here
  if (rank >= split) return;
  const int j0 = (int)((long long)all * rank / split);
  const int n = (int)((long long)all * (rank + 1) / split) - j0;
  const int tiles = q.rows - blk * kRows > kTile ? 2 : 1;
  auto key_of = [&](int j) { return (j + j0 < sink ? j + j0 : j + j0 - sink + from) * kKeys; };

  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      mbar_init(k_full + i, kUnpack);
      mbar_init(v_full + i, kUnpack);
      mbar_init(k_free + i, tiles);
      mbar_init(v_free + i, tiles);
      mbar_init(s_full + i, 1);
      mbar_init(o_full + i, 1);
    }
  }
  {
    // ---- Q: two threads a row ----
    const int row = tid / 2, half = tid % 2;
    const int r = blk * kRows + row;
    uint4 x[D / 16];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; i++) x[i] = make_uint4(0, 0, 0, 0);
    if (r < q.rows) {
      const int tok = by_group(p, r);
      const uint4 *src = reinterpret_cast<const uint4 *>(
          static_cast<const uint16_t *>(p.q) + (unsigned long long)(q.first + tok) * p.ldq +
          (unsigned long long)(head * p.group + r - tok * p.group) * D + half * (D / 2));
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
    uint8_t *dst = smem + L::kQ + row / kTile * (kTile * D * 2);
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
      const float2 a = pair(x[i].x), b = pair(x[i].y), c = pair(x[i].z), d = pair(x[i].w);
      auto two = [&](float u, float v) { return h2u(__floats2half2_rn(u * up, v * up)); };
      const int chunk = half * (D / 16) + i;
      *reinterpret_cast<uint4 *>(dst + chunk / 8 * (kTile * 128) +
                                 swizzled(row % kTile, chunk % 8)) =
          make_uint4(two(a.x, c.x), two(a.y, c.y), two(b.x, d.x), two(b.y, d.y));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp < 8) {
    // ---- softmax: one row a thread, its 128 scores in registers ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int tile = warp / 4, row = tid, r = blk * kRows + row;
    const bool live = r < q.rows;
    const int tok = by_group(p, live ? r : 0), pos = q.p0 + tok;
    const int hi = live ? min(pos, end - 1) : -1, lo = window_start(p, pos);
    // keys that every live row of the tile sees
    const int r0 = blk * kRows + tile * kTile;
    const int all_hi = min(q.p0 + by_group(p, r0), end - 1);
    const int all_lo = window_start(p, q.p0 + by_group(p, min(r0 + kTile, q.rows) - 1));
    // below 1e-20 no score (they stay below 2^34) tells; at it an unseen one still counts as none
    const float cq = fmaxf(s_cq[row], 1e-20f);
    const uint32_t lanes = (uint32_t)(32 * (warp % 4)) << 16;
    const uint32_t ts = tmem + lanes + tile * 128, to = tmem + lanes + 256 + tile * D;
    float m = -INFINITY;
    uint64_t l2[2] = {0, 0};  // the row's sum in four parts
    const int steps = tile < tiles ? n : 0;
    const bool turns = tiles == 2;
    if (turns && tile == 1 && steps > 0) bar_arrive_n(3, 2 * kTile);  // the first turn is tile 0's
    const bool issues = warp % 4 == 0;  // this warp issues the tile's products
    const uint32_t leader = elect_leader();
    auto scores = [&](int j) {
      ok = ok && mbar_wait(k_full + (j & 1), j >> 1 & 1);
      if (!__all_sync(0xFFFFFFFFu, ok)) return;
      tc_fence_after();
      const uint64_t qd = (kDesc | (smem_addr(smem + L::kQ) >> 4)) +
                          (uint64_t)(tile * (kTile * D * 2 >> 4));
      const uint64_t kd = (kDesc | (smem_addr(smem + L::kK) >> 4)) +
                          (uint64_t)((j & 1) * (L::kOne >> 4));
#pragma unroll
      for (int k = 0; k < D / 16; k++) {
        const uint64_t at = (uint64_t)(k / 4 * (kTile * 128 >> 4) + k % 4 * 2);
        mma_f16_ss(leader, tmem + tile * 128, qd + at, kd + at, idesc_f16(kKeys), k > 0);
      }
      if (leader) {
        mma_commit(s_full + tile);
        mma_commit(k_free + (j & 1));
      }
      __syncwarp();
    };
    auto outputs = [&](int j) {
      ok = ok && mbar_wait(v_full + (j & 1), j >> 1 & 1);
      if (!__all_sync(0xFFFFFFFFu, ok)) return;
      tc_fence_after();
      const uint64_t vd = (kDesc | (smem_addr(smem + L::kV) >> 4)) +
                          (uint64_t)((j & 1) * (L::kOne >> 4));
#pragma unroll
      for (int k = 0; k < kKeys / 16; k++)
        mma_f16_ts(leader, tmem + 256 + tile * D, tmem + tile * 128 + 8 * k,
                   vd + (uint64_t)(k / 4 * (D * 128 >> 4) + k % 4 * 2), idesc_f16(D),
                   j > 0 || k > 0);
      if (leader) mma_commit(v_free + (j & 1));
      __syncwarp();
    };
    if (issues && steps > 0) {
      scores(0);
    }
    __syncwarp();
#pragma unroll 1
    for (int j = 0; j < steps; j++) {
      const int key = key_of(j);
      ok = ok && mbar_wait(s_full + tile, j & 1);
      __syncwarp();
      tc_fence_after();
      const bool masked = key + kKeys - 1 > all_hi || (key < all_lo && key + kKeys > p.sinks);
      if (turns) bar_sync_n(3 + tile, 2 * kTile);  // the other tile's softmax is over
      tc_fence_after();
      uint32_t s[4][32];  // the row's scores
#pragma unroll
      for (int c = 0; c < 4; c++) tmem_ld32_nowait(ts + 32 * c, s[c]);
      tmem_wait_ld();
      if (masked) {  // unseen keys' scores to where they cost the exponential nothing
        auto below = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u; };
#pragma unroll
        for (int c = 0; c < 4; c++) {
          const int k0 = key + 32 * c;
          const uint32_t bits = below(hi + 1 - k0) & (~below(lo - k0) | below(p.sinks - k0));
#pragma unroll
          for (int i = 0; i < 32; i++)
            if (!(bits >> i & 1)) s[c][i] = __float_as_uint(kUnseen);
        }
      }
      float t4[4];
#pragma unroll
      for (int c = 0; c < 4; c++) {
        t4[c] = max3(s[c][0], s[c][1], s[c][2]);
#pragma unroll
        for (int i = 3; i < 31; i += 2) t4[c] = max3(t4[c], s[c][i], s[c][i + 1]);
        t4[c] = fmaxf(t4[c], __uint_as_float(s[c][31]));
      }
      const float top = fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]);
      const float now = top <= kUnseen ? -INFINITY : top * cq;
      const bool grew = now > m + kStale || (m == -INFINITY && now > -INFINITY);
      if (__any_sync(0xFFFFFFFFu, grew)) {
        // the tile's products so far are complete: O may be read and written
        float f = 1.0f;
        if (grew) {
          f = m == -INFINITY ? 0.0f : ex2(m - now);
          m = now;
          const float2 a = unpack2(l2[0]), b = unpack2(l2[1]);
          l2[0] = pack2(a.x * f, a.y * f);
          l2[1] = pack2(b.x * f, b.y * f);
        }
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16_nowait(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st16(to + c, o);
          }
        }
      }
      const float base = kOffset - (m == -INFINITY ? 0.0f : m);
      const uint64_t cq2 = pack2(cq, cq), base2 = pack2(base, base);
#pragma unroll
      for (int c = 0; c < 4; c++) {
        uint32_t h[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
          const float2 x = unpack2(fma2(pack2(__uint_as_float(s[c][2 * i]),
                                              __uint_as_float(s[c][2 * i + 1])),
                                        cq2, base2));
          const float e0 = ex2(x.x), e1 = ex2(x.y);
          l2[i & 1] = add2(l2[i & 1], pack2(e0, e1));
          h[i] = h2u(__floats2half2_rn(e0, e1));
        }
        tmem_st16(ts + 16 * c, h);
      }
      tmem_wait_st();
      tc_fence_before();
      if (turns && (tile == 0 || j + 1 < steps)) bar_arrive_n(3 + (tile ^ 1), 2 * kTile);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + tile), "n"(kTile) : "memory");  // the tile's threads
      if (issues) {
        outputs(j);
        if (j + 1 < steps) scores(j + 1);
        else if (leader) mma_commit(o_full + tile);
      }
      __syncwarp();
    }
    // ---- the output rows ----
    // (after a wait that gave up, too: tensor memory is given back once its products are done)
    if (steps > 0) ok = mbar_wait(o_full + tile, 0) && ok;
    __syncwarp();
    tc_fence_after();
    const float2 la = unpack2(l2[0]), lb = unpack2(l2[1]);
    float l = (la.x + la.y) + (lb.x + lb.y);
    // The rows of a split block are joined by the CTAs in warps' rows, as even as they go: warp w's by
    // CTA w split / 8, in whose shared memory the parts from the others take the operands' place,
    // [split - 1][per] rows of D (chunks of a row turned by its number: no bank twice), then as many
    // (m, l).
    const int per = 32 * join_warps(split), to_rank = warp * split / 8;
    const int rl = row - 32 * ((8 * to_rank + split - 1) / split);
    auto part = [&](int slot) { return smem + (size_t)(slot * per + rl) * (D * 4); };
    auto part_ml = [&](int slot) {
      return smem + (size_t)(split - 1) * per * (D * 4) + (slot * per + rl) * 8;
    };
    auto turned = [&](int chunk) { return (chunk ^ (rl & (D / 4 - 1))) << 4; };
    float own = steps > 0 && m > -INFINITY ? 1.0f : 0.0f, top = m;  // this CTA's factor
    if (split > 1) {
      cluster_arrive_release();  // every CTA is done with its operands
      cluster_wait_acquire();
      if (to_rank != rank) {
        const int slot = rank < to_rank ? rank : rank - 1;
        const uint32_t dst = cluster_map(part(slot), to_rank);
        if (steps > 0)
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tmem_ld16_nowait(to + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; i++)
              asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                               dst + turned(c / 4 + i)),
                           "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]), "r"(o[4 * i + 3])
                           : "memory");
          }
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(
                         cluster_map(part_ml(slot), to_rank)),
                     "f"(own == 0.0f ? -INFINITY : m), "f"(l)
                     : "memory");
      }
      __syncwarp();
      cluster_arrive_release();
      cluster_wait_acquire();
      if (to_rank == rank) {
        for (int i = 0; i < split - 1; i++)
          top = fmaxf(top, *reinterpret_cast<const float *>(part_ml(i)));
        if (own != 0.0f) own = ex2(m - top);
        l *= own;
        for (int i = 0; i < split - 1; i++) {
          const float2 ml = *reinterpret_cast<const float2 *>(part_ml(i));
          if (ml.x > -INFINITY) l = fmaf(ex2(ml.x - top), ml.y, l);
        }
      }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *dst = static_cast<uint16_t *>(p.out) +
                    (unsigned long long)(q.first + tok) * p.ldo +
                    (unsigned long long)(head * p.group + (live ? r : 0) - tok * p.group) * D;
#pragma unroll 1
    for (int c = 0; c < (to_rank == rank ? D : 0); c += 16) {
      uint32_t o[16];
      if (steps > 0) {
        tmem_ld16_nowait(to + c, o);
        tmem_wait_ld();
      }
      if (own != 1.0f)
#pragma unroll
        for (int i = 0; i < 16; i++)
          o[i] = own == 0.0f ? 0 : __float_as_uint(__uint_as_float(o[i]) * own);
#pragma unroll 1
      for (int k = 0; k < split - 1; k++) {
        const float ms = *reinterpret_cast<const float *>(part_ml(k));
        if (ms == -INFINITY) continue;
        const float f = ex2(ms - top);
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4 x = *reinterpret_cast<const float4 *>(part(k) + turned(c / 4 + i));
          o[4 * i] = __float_as_uint(fmaf(f, x.x, __uint_as_float(o[4 * i])));
          o[4 * i + 1] = __float_as_uint(fmaf(f, x.y, __uint_as_float(o[4 * i + 1])));
          o[4 * i + 2] = __float_as_uint(fmaf(f, x.z, __uint_as_float(o[4 * i + 2])));
          o[4 * i + 3] = __float_as_uint(fmaf(f, x.w, __uint_as_float(o[4 * i + 3])));
        }
      }
      __syncwarp();
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
  } else {
    // ---- unpacking: a warp has 16 keys, a thread half `part` of one's K; and of V dims
    // 64 mq + 32 part + 16 i + g and + 8 (i < 2) of all 16.  Neighbours have rows of different
    // swizzle: their stores meet no bank twice ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
    const int t = tid - 256, tile = t / 32;
    const int tok = t % kKvTile, g = t % 8, mq = t / 8 % 2, part = t / 16 % 2;
    const bool has_v = D == 128 || mq == 0;
    const Unpack un;
    constexpr int K16 = D / 64;  // 16-byte loads of half a token's K
    uint4 kraw[K16], vsc[2];
    uint2 vraw[4];
    __half ksc[K16];
    int page = -1;
    const int *table = p.table + (size_t)seq * p.max_pages;
    auto find = [&](int j) {  // the page of this thread's tile at step j
      const int key = key_of(j) + tile * kKvTile;
      if (j >= n || key >= end || unseen(p, key, kKvTile, low)) return -1;
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
    // plain loads: the kernel that writes the pages may still run when this one starts, and the
    // read-only path promises nothing then
    auto load_k = [&](int j) {
      if (page < 0) return;
      const uint8_t *src = source(j, page);
#pragma unroll
      for (int i = 0; i < K16; i++) {
        kraw[i] = reinterpret_cast<const uint4 *>(src + tok * (D / 2) + part * (D / 4))[i];
        ksc[i] = reinterpret_cast<const __half *>(
            src + kv4_ks_off(D))[(part * K16 + i) * kKvTile + tok];
      }
    };
    auto load_v = [&](int j) {
      if (page < 0 || !has_v) return;
      const uint8_t *src = source(j, page);
#pragma unroll
      for (int i = 0; i < 4; i++)
        vraw[i] = reinterpret_cast<const uint2 *>(
            src + kv4_v_off(D))[(mq * 32 + g * 4 + i) * 2 + part];
#pragma unroll
      for (int i = 0; i < 2; i++)  // a group of 32 dims, 16 tokens
        vsc[i] = reinterpret_cast<const uint4 *>(src + kv4_vs_off(D))[(mq * 2 + part) * 2 + i];
    };
    page = find(0);
    load_k(0);
    load_v(0);
#pragma unroll 1
    for (int j = 0; j < n; j++) {
      const int key = key_of(j), buf = j & 1;
      const int page_now = page, page_next = find(j + 1);
      if (j > 1) ok = ok && mbar_wait(k_free + buf, ((j >> 1) - 1) & 1);
      {
        const bool have = page_now >= 0 && key + tile * kKvTile + tok < end;
        uint8_t *dst = smem + L::kK + buf * L::kOne;
        const int row = tile * kKvTile + tok;
#pragma unroll
        for (int i = 0; i < K16; i++) {
          const uint32_t w[4] = {kraw[i].x, kraw[i].y, kraw[i].z, kraw[i].w};
          const __half2 sc = __half2half2(ksc[i]);  // 32 dims: one group
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const int chunk = part * (D / 16) + 4 * i + c;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (have)
              v = make_uint4(un.low2(w[c], sc), un.high2(w[c], sc), un.low2(w[c] >> 8, sc),
                             un.high2(w[c] >> 8, sc));
            *reinterpret_cast<uint4 *>(dst + chunk / 8 * (kKeys * 128) +
                                       swizzled(row, chunk % 8)) = v;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(k_full + buf);
      page = page_next;
      load_k(j + 1);
      if (j > 1) ok = ok && mbar_wait(v_free + buf, ((j >> 1) - 1) & 1);
      if (has_v) {
        const int first = key + tile * kKvTile;
        const bool have = page_now >= 0;
        uint8_t *dst = smem + L::kV + buf * L::kOne;
#pragma unroll
        for (int i = 0; i < 2; i++) {  // dims 64 mq + 32 part + 16 i + g and + 8
          uint32_t a[2][8];            // dim; tokens 2 k and 2 k + 1
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t w = i == 0 ? vraw[k].x : vraw[k].y;
            const uint32_t s0 = k == 0 ? vsc[0].x : k == 1 ? vsc[0].y : k == 2 ? vsc[0].z : vsc[0].w;
            const uint32_t s1 = k == 0 ? vsc[1].x : k == 1 ? vsc[1].y : k == 2 ? vsc[1].z : vsc[1].w;
            a[0][k] = un.low2(w, u2h(s0));
            a[1][k] = un.high2(w, u2h(s0));
            a[0][4 + k] = un.low2(w >> 8, u2h(s1));
            a[1][4 + k] = un.high2(w >> 8, u2h(s1));
          }
          if (!have || first + kKvTile > end || first < low) {
            // tokens past the last key or behind the window may hold anything
            auto gone = [&](int key) { return !have || key >= end || unseen(p, key, 1, low); };
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
              for (int k = 0; k < 8; k++) {
                if (gone(first + 2 * k)) a[h][k] &= 0xFFFF0000u;
                if (gone(first + 2 * k + 1)) a[h][k] &= 0x0000FFFFu;
              }
          }
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int d = 64 * mq + 32 * part + 16 * i + g + 8 * h;
#pragma unroll
            for (int k = 0; k < 2; k++) {  // tokens 8 k .. 8 k + 7 of the tile
              const int chunk = tile * 2 + k;
              *reinterpret_cast<uint4 *>(dst + chunk / 8 * (D * 128) + swizzled(d, chunk % 8)) =
                  make_uint4(a[h][4 * k], a[h][4 * k + 1], a[h][4 * k + 2], a[h][4 * k + 3]);
            }
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(v_full + buf);
      load_v(j + 1);
    }
    if (split > 1) {  // the softmax threads' two
      __syncwarp();
      cluster_arrive_release();
      cluster_wait_acquire();
      cluster_arrive_release();
      cluster_wait_acquire();
    }
  }
  if (!ok) attn_refuse(p, seq, APX_ERR_DEVICE_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 15) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// Clusters of `split` CTAs that the current device holds at once (found once a device).
template <int D>
int resident(int split, cudaLaunchConfig_t cfg) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMaxSplit + 1];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kDevices) return 0;
  std::atomic<int> &k = known[dev][split];
  n = k.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)split, 1, 1};
    cfg.gridDim = dim3((unsigned)split, 1);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, attn_tc_kernel<D>, &cfg) != cudaSuccess) {
      cudaGetLastError();
      return 0;
    }
    k.store(n, std::memory_order_relaxed);
  }
  return n;
}

template <int D>
cudaError_t launch(const AttnArgs &p, int max_q, cudaStream_t stream) {
  auto kern = attn_tc_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Smem<D>::kBytes);
  if (e != cudaSuccess) return e;
  const long long blocks = ((long long)max_q * p.group + kRows - 1) / kRows;
  const long long items = (long long)p.n_seqs * p.kv_heads * blocks;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Smem<D>::kBytes;
  cfg.stream = stream;
  // A block's keys to as many CTAs as let all of them run at once (heads of 128; 64 tokens over 60000
  // keys, 64 / 8 heads: one CTA a block 1190 us, four 338, six 237; 128 over 8000, 64 / 8 heads: 158,
  // four 59, and 12 / 2 heads: 157, four 57, eight 43; 100 over 30000, 12 / 2 heads: 552, four 157,
  // eight 94).  Past that it costs: two rounds of short CTAs are slower than one of long ones (two
  // prompts of up to 2048, 192 blocks: 64 us, in pairs 95).
  int split = kMaxSplit;
  while (split > 1 && !(Smem<D>::joins(split) && items <= resident<D>(split, cfg))) split--;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_allowed() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)split, 1, 1};
  cfg.gridDim = dim3((unsigned)(p.n_seqs * p.kv_heads * split), (unsigned)blocks);
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p, split);
}

}  // namespace

// Prompts in 16-bit numbers, from three quarters of a tile's rows on: a tile costs the same
// however many of its rows are there.  One request over 30000 keys, 8 KV heads of 128: 87 us here
// for any of 64 to 128 rows, apx_attn.cu's kernel 60 for 64, 77 for 80 and 96, 98 for 112 and 128;
// 32 requests over 100 to 4000: 155 to 159, and 139 for 64, 203 for 96, 262 for 128.  Where one
// request has two KV heads of 64 the other kernel stays ahead for longer (96 rows over 30000 keys:
// 62 and 28).
bool attn_tc_serves(const AttnArgs &p, int dim, int max_q) {
  const long long rows = (long long)max_q * p.group;
  return p.type != APX_DTYPE_F32 && rows >= 96 && rows <= 65535ll * kRows &&
         (long long)p.n_seqs * p.kv_heads < (1ll << 31) && (dim == 64 || dim == 128);
}

cudaError_t launch_attn_tc(const AttnArgs &p, int dim, int max_q, cudaStream_t stream) {
  return dim == 128 ? launch<128>(p, max_q, stream) : launch<64>(p, max_q, stream);
}

}  // namespace apx
