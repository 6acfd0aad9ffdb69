// apx_attn.cu — attention over the paged 4-bit cache (layout: apx_kv4.cuh): the kernel for few
// query rows and for f32.
//
// out_i = sum_j p_ij v_j, p = softmax over the visible keys of scale q_i.k_j, in one pass over
// the keys with a running maximum m and sum l: keys with scores s_j turn (m, l, o) into
// m' = max(m, max s_j), l' = l e^(m-m') + sum e^(s_j-m'), o' = o e^(m-m') + sum e^(s_j-m') v_j.
//
// What bounds it: a decoded token reads every visible key once (D * 1.125 bytes a token and KV
// head) and its group's query heads share the read, so the cache's bytes are the floor.  What a
// byte costs in instructions decides how near it comes: a key's D dims unpack to f16 (three
// instructions for two values) and go through the matrix unit as the 16-row operand, S^T = K Q^T
// and O^T = V^T P, with 8 query rows per column tile.  mma.sync, not tcgen05: with 8 rows the
// unpacked keys would cross shared memory and tensor memory for an 8th of a 64-row tile; from
// registers they go straight in.
//
// Numbers.  d (c - 8) is exact in f16 (the append's d has 8 significant bits).  A query row is
// scaled by a power of two to the top of f16's range and, for f32, split in two halves of 11 bits
// each; so are the probabilities, taken at 2^13 e^(s - m): 22 bits down to 2^-38 of the largest.
// With 16-bit q the probabilities go to the product in one half of 11 bits (their sum keeps f32):
// below what the output's rounding costs, and half of the products (against 64 bits, relative:
// bf16 1.7e-3 as the plain form in f32, f16 2.1e-4 against the plain form's 2.0e-4).
// The unit's f32 accumulation is cut into short chains joined by f32 additions.
//
// Split.  Work is counted in steps of 32 keys of one item (sequence, KV head, block of query
// rows), in that order; every warp of the grid takes the same number of consecutive steps, so
// ragged lengths and one long context balance alike.  Where an item spans warps of a CTA they
// join in shared memory, where it spans CTAs through a workspace, joined by the last to arrive in
// the items' order (not in the order of arrival: the same bits every time).  Blocks of a prompt's
// rows pair first with last, so that the causal halves fill up to equal work.
//
// Copies: each warp has its own ring of slots in shared memory, two tiles (32 keys) each, filled
// by bulk copies a ring ahead; nothing in the loop waits for another warp.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "apx_attn_items.cuh"
#include "apx_common.cuh"
#include "apx_kv4.cuh"
#include "apx_pack.cuh"
#include "apx_kernels.h"
#include "apx_step.h"

namespace apx {

// apx_attn_tc.cu
bool attn_tc_serves(const AttnArgs &p, int dim, int max_q);
cudaError_t launch_attn_tc(const AttnArgs &p, int dim, int max_q, cudaStream_t stream);

namespace {

// Probabilities are held at 2^13 e^(s - m), where m is a stale maximum: it moves when a score
// outgrows it by more than 2^2.
constexpr float kTopExp = 13.0f, kStale = 2.0f;

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = h2u(h);
  lo = h2u(__floats2half2_rn(x - f.x, y - f.y));
}

template <int TYPE>
__device__ __forceinline__ void store4(void *o, unsigned long long i, const float4 v) {
  if (TYPE == APX_DTYPE_F32) {
    *reinterpret_cast<float4 *>(static_cast<float *>(o) + i) = v;
  } else {
    uint2 w;
    if (TYPE == APX_DTYPE_BF16) {
      __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
      w = make_uint2(*reinterpret_cast<uint32_t *>(&x), *reinterpret_cast<uint32_t *>(&y));
    } else {
      w = make_uint2(h2u(__floats2half2_rn(v.x, v.y)), h2u(__floats2half2_rn(v.z, v.w)));
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(o) + i) = w;
  }
}
template <int TYPE>
__device__ __forceinline__ void store_out(void *o, unsigned long long i, float v) {
  if (TYPE == APX_DTYPE_F32) static_cast<float *>(o)[i] = v;
  else if (TYPE == APX_DTYPE_F16) static_cast<__half *>(o)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16 *>(o)[i] = __float2bfloat16_rn(v);
}

template <int D, int NT>
struct Cfg {
  static constexpr int kWarps = NT == 1 ? 16 : 8;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRows = 8 * NT;
  static constexpr int kTile = kv4_tile_bytes(D);
  static constexpr int kSlot = 2 * kTile;
  static constexpr int kSlots = (D == 128 ? 2 : 4) * (NT == 1 ? 1 : 2);  // a power of two
  static constexpr int kRing = kSlots * kSlot;
  // a partial item: O (rows x D), then m and l of each row, all f32
  static constexpr int kPart = kRows * D + 2 * kRows;
  static constexpr int kWarpSmem = kRing + kPart * 4;
  static constexpr int kSmem = kWarps * kWarpSmem;
  static_assert(kPart * 4 <= kRing, "a partial item fits the ring");
  static_assert(kSmem <= 227 * 1024 - 13 * 1024, "shared memory");
};

// The item of step g, the same g in every lane.  pre: the steps of the call up to the end of each
// thread's `per` sequences.
template <int R, bool ONE, int THREADS, typename S>
__device__ __noinline__ Item<S> find_item(const AttnArgs &p, const S *pre, int per, S g) {
  constexpr int N = THREADS / 32;
  const int lane = threadIdx.x % 32;
  int at = __ffs(__ballot_sync(0xFFFFFFFFu, pre[lane * N + N - 1] > g)) - 1;
  at = at * N + __ffs(__ballot_sync(0xFFFFFFFFu, lane < N && pre[at * N + lane % N] > g)) - 1;
  return item_from<R, ONE, S>(p, at * per, at ? pre[at - 1] : 0, g);
}

// Where a wait has given up, a CTA has no parts to give, yet each item that crosses its ends counts it:
// these stand for what its warps would have kept (the parts behind them may hold anything: the
// status has the call as refused), so that the counters are zero again at the end of the call.
template <int R, bool ONE, int W, typename S>
__device__ __noinline__ void keep_owed(const AttnArgs &p, S e0, S e1, Edge<S> (*edge)[2]) {
  for (int w = 0; w < W; w++) edge[w][0].used = edge[w][1].used = 0;
  Edge<S> from_before, goes_on;
  const int owes = owed<R, ONE, S>(p, e0, e1, from_before, goes_on);
  if (owes & 1) edge[0][0] = from_before;
  if (owes & 2) edge[W - 1][1] = goes_on;
}

// After a wait has given up: copies [from, to) may still be on their way into shared memory.
__device__ __noinline__ void drain(uint64_t *bar, int slots, int from, int to) {
  for (int i = from; i < to; i++) mbar_wait(bar + i % slots, i / slots & 1);
}

template <int D, int NT, int TYPE, typename S>
__global__ void __launch_bounds__(Cfg<D, NT>::kThreads, 1) attn_split_kernel(const __grid_constant__ AttnArgs p) {
  using C = Cfg<D, NT>;
  constexpr int SPLIT = TYPE == APX_DTYPE_F32 ? 2 : 1;
  constexpr int W = C::kWarps, R = C::kRows, K4 = D / 32;  // words of K per thread and row
  constexpr bool ONE = NT == 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ S s_pre[C::kThreads], s_warp[W];
  __shared__ __align__(8) uint64_t s_bar[W * C::kSlots];
  __shared__ Edge<S> s_edge[W][2];
  __shared__ int s_last[2], s_most[W];
  __shared__ float s_inv[R];

  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, gid = lane / 4, tig = lane % 4;
  pdl_launch_dependents();
  uint8_t *ring = smem + warp * C::kWarpSmem;
  uint64_t *bar = s_bar + warp * C::kSlots;
  if (lane == 0)
    for (int i = 0; i < C::kSlots; i++) mbar_init(bar + i, 1);
  if (lane < 2) s_edge[warp][lane].used = 0;
  pdl_wait();

  // ---- the call's steps, summed over the sequences before each thread's share of them ----
  const int per = (p.n_seqs + C::kThreads - 1) / C::kThreads;
  S total;
  int longest = 0;
  {
    S run = 0;
    int most = 0;
#pragma unroll 1
    for (int i = 0; i < per; i++) {
      const int s = tid * per + i;
      if (s >= p.n_seqs) break;
      SeqShape<R, ONE> q;
      q.load(p, s);
      if (q.bad && blockIdx.x == 0) attn_refuse(p, s, APX_ERR_INVALID_ARGUMENT);
      most = max(most, q.pair);
      run += q.template all<S>(p);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const S u = __shfl_up_sync(0xFFFFFFFFu, run, o);
      if (lane >= o) run += u;
    }
    if (ONE) most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 31) s_warp[warp] = run, s_most[warp] = most;
    __syncthreads();
    S before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < W; i++) {
      all += s_warp[i];
      longest = max(longest, s_most[i]);
      if (i < warp) before += s_warp[i];
    }
    s_pre[tid] = before + run;  // inclusive
    total = all;
    __syncthreads();
  }
  // Equal shares for every warp of the grid, the first `rem` one step more.  Or, while there are
  // CTAs for all items and the longest costs a warp four steps at most: an item per CTA, which
  // saves the join through the workspace (0.5B shape, 777 keys: 13.5 -> 9.3 us).
  const int items = ONE ? p.n_seqs * p.kv_heads : 0;
  const bool whole_items = ONE && items <= (int)gridDim.x && longest <= 4 * W + kItemCost;
  const unsigned nwarps =
      whole_items ? W : (unsigned)min((S)(gridDim.x * W), max(total, (S)1));
  S c0 = 0, c1 = total;
  if (whole_items) {
    if ((int)blockIdx.x >= items) return;
    const int s = blockIdx.x / p.kv_heads, h = blockIdx.x - s * p.kv_heads;
    const S s0 = s ? s_pre[s - 1] : 0, n = (s_pre[s] - s0) / (unsigned)p.kv_heads;
    c0 = s0 + h * n;
    c1 = c0 + (n ? n - kItemCost : 0);
  }
  const Shares<W, S> share(c0, c1, nwarps);
  const unsigned w0 = whole_items ? 0 : blockIdx.x * W;  // this CTA's first warp
  const S u0 = share.bound(w0 + warp), u1 = share.bound(w0 + warp + 1);

  // ---- copies: step u0 + i into slot i of the ring, through every item of this warp ----
  const uint8_t *src = nullptr;  // lane i: tile i % 2 of step u0 + batch + i / 2; null: no such
  unsigned there = 0;            // which lanes' tiles are
  int batch = -16;
  const uint64_t policy = stream_policy();
  auto look_ahead = [&](int i, Item<S> c) {  // c: the item of step u0 + i, or one before
    batch = i;
    src = nullptr;
    const S g0 = u0 + i, g = g0 + lane / 2;
    while (true) {
      if (c.real && g >= c.i0 && g < min(c.i1, u1)) {
        const int key = c.key_of((int)(g - c.i0)) + lane % 2 * kKvTile;
        if (key < c.end && !unseen(p, key, kKvTile, c.low)) {
          const int page = p.table[(size_t)c.seq * p.max_pages + (key >> p.page_shift)];
          if (page >= 0 && page < p.n_pages)
            src = p.pages + ((unsigned long long)page * p.kv_heads + c.head) * p.page_bytes +
                  (unsigned)((key & ((1 << p.page_shift) - 1)) / kKvTile) * C::kTile;
          else
            attn_refuse(p, c.seq, APX_ERR_INVALID_ARGUMENT);
        }
      }
      if (c.i1 >= min(g0 + 16, u1)) break;
      c = find_item<R, ONE, C::kThreads, S>(p, s_pre, per, c.i1);
    }
    there = __ballot_sync(0xFFFFFFFFu, src != nullptr);
  };
  auto start = [&](int i) {  // i < batch + 16
    const int sl = i & (C::kSlots - 1), owner = 2 * (i - batch);
    if (lane == owner)
      mbar_expect_tx(bar + sl, (uint32_t)__popc(there >> owner & 3u) * C::kTile);
    if ((lane & ~1) == owner && src != nullptr)
      bulk_g2s_policy(ring + sl * C::kSlot + (lane & 1) * C::kTile, src, C::kTile, bar + sl,
                      policy);
  };
  const int mine = (int)(u1 - u0);  // steps of this warp
  int at = 0;                       // of them, done
  bool alive = true;                // no wait has given up; between steps the same in every lane
  auto arrived = [&](int i) {
    const int sl = i & (C::kSlots - 1);
    const unsigned parity = (unsigned)i / C::kSlots & 1;
    if (!mbar_try(bar + sl, parity)) alive = mbar_wait_more(bar + sl, parity);
  };

  // ---- this warp's steps, item by item ----
  const Unpack un;
#pragma unroll 1
  while (at < mine && alive) {
    const Item<S> it = find_item<R, ONE, C::kThreads, S>(p, s_pre, per, u0 + at);
    const int stop = (int)(min(it.i1, u1) - u0), before = (int)(u0 - it.i0);
    // the block's query rows, asked for before the first copies
    constexpr int QV = SPLIT == 2 ? D / 16 : D / 32;  // 16-byte loads a row and thread
    uint4 qraw[NT][QV];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int r = it.row0 + 8 * n + gid;
#pragma unroll
      for (int i = 0; i < QV; i++) qraw[n][i] = make_uint4(0, 0, 0, 0);
      if (it.real && r < it.rows) {
        const int tok = by_group(p, r);
        const unsigned long long e =
            (unsigned long long)(it.first + tok) * p.ldq +
            (unsigned long long)(it.head * p.group + r - tok * p.group) * D + tig * (D / 4);
        const uint4 *src4 = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p.q) +
                                                            e * (SPLIT == 2 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < QV; i++) qraw[n][i] = src4[i];
      }
    }
    if (at == 0) {
      look_ahead(0, it);
      for (int i = 0; i < min(mine, C::kSlots); i++) start(i);
    }
    const int end = it.end;

    // ---- the rows as the second operand ----
    uint32_t qh[NT][2 * K4][2], ql[SPLIT == 2 ? NT : 1][2 * K4][2];
    float cq[NT][2];  // of columns 2 tig, 2 tig + 1: score units per product unit, times log2 e
    int vis_lo[NT][2], vis_hi[NT][2];
    int all_lo = 0, all_hi = 1 << 30;  // keys that every row of the block sees
#pragma unroll
    for (int n = 0; n < NT; n++) {
      // matrix steps 2 w and 2 w + 1 take dims (0,4),(1,5) and (2,6),(3,7) of word w
      float v[2 * K4][4];
      auto put = [&v](int i, float x) { v[2 * (i / 8) + i % 4 / 2][2 * (i % 2) + i % 8 / 4] = x; };
#pragma unroll
      for (int i = 0; i < QV; i++) {
        const uint32_t w[4] = {qraw[n][i].x, qraw[n][i].y, qraw[n][i].z, qraw[n][i].w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (TYPE == APX_DTYPE_F32) {
            put(4 * i + j, __uint_as_float(w[j]));
          } else if (TYPE == APX_DTYPE_BF16) {
            put(8 * i + 2 * j, __uint_as_float(w[j] << 16));
            put(8 * i + 2 * j + 1, __uint_as_float(w[j] & 0xFFFF0000u));
          } else {
            const float2 f = __half22float2(u2h(w[j]));
            put(8 * i + 2 * j, f.x);
            put(8 * i + 2 * j + 1, f.y);
          }
        }
      }
      float top = 0.0f;
#pragma unroll
      for (int w = 0; w < 2 * K4; w++)
#pragma unroll
        for (int j = 0; j < 4; j++) top = fmaxf(top, fabsf(v[w][j]));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      const int e = row_exponent(top);
      const float up = pow2(9 - e);
#pragma unroll
      for (int w = 0; w < 2 * K4; w++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          if (SPLIT == 2)
            split2(v[w][2 * j] * up, v[w][2 * j + 1] * up, qh[n][w][j],
                   ql[SPLIT == 2 ? n : 0][w][j]);
          else
            qh[n][w][j] = h2u(__floats2half2_rn(v[w][2 * j] * up, v[w][2 * j + 1] * up));
        }
      const float c = p.scale * 1.44269504088896341f * pow2(e - 9);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        cq[n][j] = __shfl_sync(0xFFFFFFFFu, c, (2 * tig + j) * 4);
        const int col = it.row0 + 8 * n + 2 * tig + j;
        const int pos = it.p0 + by_group(p, col);
        const bool live = col < it.rows;
        vis_hi[n][j] = live ? min(pos, end - 1) : -1;
        vis_lo[n][j] = window_start(p, pos);
        if (live) {
          all_hi = min(all_hi, vis_hi[n][j]);
          all_lo = max(all_lo, vis_lo[n][j]);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      all_hi = min(all_hi, __shfl_xor_sync(0xFFFFFFFFu, all_hi, o));
      all_lo = max(all_lo, __shfl_xor_sync(0xFFFFFFFFu, all_lo, o));
    }

    float o[NT][D / 16][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < D / 16; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) o[n][i][j] = 0.0f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }
    const bool from_start = u0 + at == it.i0;

#pragma unroll 1
    for (; at < stop && alive; at++) {
      arrived(at);
      uint8_t *tile = ring + (at & (C::kSlots - 1)) * C::kSlot;
      if (it.real) {  // not filling, which has no keys
      const int key = it.key_of(at + before);
      const bool behind = key < all_lo && key + kStepKeys > p.sinks;  // some row's window
      if (key + kStepKeys > end || behind) {
        // tokens past the last key or behind the window may hold anything: V's scales there count
        // as zero (K's are masked)
        __syncwarp();
        if (key + lane >= end || unseen(p, key + lane, 1, it.low))
#pragma unroll
          for (int g = 0; g < D / kKvGroup; g++)
            *reinterpret_cast<uint16_t *>(tile + lane / kKvTile * C::kTile + kv4_vs_off(D) +
                                          (g * kKvTile + lane % kKvTile) * 2) = 0;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the slot's next copy
        __syncwarp();
      }

      // scores of 32 keys, S^T = K Q^T: rows gid and gid + 8 of two tiles
      float s[2][NT][4];
      {
        uint32_t kw[2][2][K4];
        __half2 ks[2][2];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            const uint8_t *k = tile + t * C::kTile + (gid + 8 * r) * (D / 2) + tig * (D / 8);
            if (D == 128) {
              const uint4 x = *reinterpret_cast<const uint4 *>(k);
              kw[t][r][0] = x.x, kw[t][r][1] = x.y;
              kw[t][r][2 % K4] = x.z, kw[t][r][3 % K4] = x.w;
            } else {
              const uint2 x = *reinterpret_cast<const uint2 *>(k);
              kw[t][r][0] = x.x, kw[t][r][1] = x.y;
            }
            const int g = tig * (D / 4) / kKvGroup;
            ks[t][r] = __half2half2(*reinterpret_cast<const __half *>(
                tile + t * C::kTile + kv4_ks_off(D) + (g * kKvTile + gid + 8 * r) * 2));
          }
        float lo[2][NT][4];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) s[t][n][j] = lo[t][n][j] = 0.0f;
#pragma unroll
        for (int w = 0; w < K4; w++)
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const uint32_t x = kw[t][0][w], y = kw[t][1][w];
            const uint32_t a[4] = {un.low2(x, ks[t][0]), un.low2(y, ks[t][1]), un.high2(x, ks[t][0]),
                                   un.high2(y, ks[t][1])};
            const uint32_t b[4] = {un.low2(x >> 8, ks[t][0]), un.low2(y >> 8, ks[t][1]),
                                   un.high2(x >> 8, ks[t][0]), un.high2(y >> 8, ks[t][1])};
#pragma unroll
            for (int n = 0; n < NT; n++) {
              mma_f16(s[t][n], a, qh[n][2 * w][0], qh[n][2 * w][1]);
              mma_f16(s[t][n], b, qh[n][2 * w + 1][0], qh[n][2 * w + 1][1]);
              if (SPLIT == 2) {
                mma_f16(lo[t][n], a, ql[SPLIT == 2 ? n : 0][2 * w][0],
                        ql[SPLIT == 2 ? n : 0][2 * w][1]);
                mma_f16(lo[t][n], b, ql[SPLIT == 2 ? n : 0][2 * w + 1][0],
                        ql[SPLIT == 2 ? n : 0][2 * w + 1][1]);
              }
            }
          }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++)
              s[t][n][j] = (SPLIT == 2 ? s[t][n][j] + lo[t][n][j] : s[t][n][j]) * cq[n][j & 1];
      }
      // masks, where some row does not see all 32 keys
      if (key + kStepKeys - 1 > all_hi || behind) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int k = key + kKvTile * t + gid + 8 * (j / 2);
              const bool seen =
                  k <= vis_hi[n][j & 1] && (k >= vis_lo[n][j & 1] || k < p.sinks);
              if (!seen) s[t][n][j] = -INFINITY;
            }
      }
      // the sums and outputs turn only when some score has outgrown its maximum
      bool grew = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          top[n][j] = fmaxf(fmaxf(s[0][n][j], s[0][n][j + 2]), fmaxf(s[1][n][j], s[1][n][j + 2]));
          grew |= top[n][j] > m[n][j] + kStale;
        }
      if (__any_sync(0xFFFFFFFFu, grew)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int sh = 4; sh < 32; sh <<= 1)
              top[n][j] = fmaxf(top[n][j], __shfl_xor_sync(0xFFFFFFFFu, top[n][j], sh));
            const float mn = fmaxf(m[n][j], top[n][j]);
            f[j] = m[n][j] == -INFINITY ? 0.0f : ex2(m[n][j] - mn);
            l[n][j] *= f[j];
            m[n][j] = mn;
          }
#pragma unroll
          for (int d = 0; d < D / 16; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[n][d][j] *= f[j & 1];
        }
      }
      // probabilities, turned into the second operand of O^T = V^T P
      uint32_t ph[2][NT][2], pl[2][SPLIT == 2 ? NT : 1][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float base[2];
#pragma unroll
        for (int j = 0; j < 2; j++) base[j] = kTopExp - (m[n][j] == -INFINITY ? 0.0f : m[n][j]);
#pragma unroll
        for (int t = 0; t < 2; t++) {
          float e[4];
#pragma unroll
          for (int j = 0; j < 4; j++) {
            e[j] = ex2(s[t][n][j] + base[j & 1]);
            l[n][j & 1] += e[j];
          }
#pragma unroll
          for (int r = 0; r < 2; r++) {
            uint32_t hi, lo;
            if (SPLIT == 2) {
              split2(e[2 * r], e[2 * r + 1], hi, lo);
              pl[t][SPLIT == 2 ? n : 0][r] = transpose8(lo);
            } else {
              hi = h2u(__floats2half2_rn(e[2 * r], e[2 * r + 1]));
            }
            ph[t][n][r] = transpose8(hi);
          }
        }
      }
#pragma unroll
      for (int mq = 0; mq < D / 64; mq++) {
        uint32_t vw[2][4];
        uint32_t vs[2][2][2];  // tile, group of 32 dims, token half
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const uint4 x = *reinterpret_cast<const uint4 *>(tile + t * C::kTile + kv4_v_off(D) +
                                                           (mq * 32 + lane) * 16);
          vw[t][0] = x.x, vw[t][1] = x.y, vw[t][2] = x.z, vw[t][3] = x.w;
#pragma unroll
          for (int g = 0; g < 2; g++)
#pragma unroll
            for (int h = 0; h < 2; h++)
              vs[t][g][h] = *reinterpret_cast<const uint32_t *>(
                  tile + t * C::kTile + kv4_vs_off(D) +
                  ((2 * mq + g) * kKvTile + 8 * h + 2 * tig) * 2);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const int d = 4 * mq + j;
          uint32_t a[2][4];
#pragma unroll
          for (int t = 0; t < 2; t++) {
            const uint32_t x = vw[t][j];
            const __half2 s0 = u2h(vs[t][j / 2][0]), s1 = u2h(vs[t][j / 2][1]);
            a[t][0] = un.low2(x, s0);
            a[t][1] = un.high2(x, s0);
            a[t][2] = un.low2(x >> 8, s1);
            a[t][3] = un.high2(x >> 8, s1);
          }
#pragma unroll
          for (int n = 0; n < NT; n++) {
            if (SPLIT == 2) {
              float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int t = 0; t < 2; t++) {
                mma_f16(acc, a[t], pl[t][SPLIT == 2 ? n : 0][0], pl[t][SPLIT == 2 ? n : 0][1]);
                mma_f16(acc, a[t], ph[t][n][0], ph[t][n][1]);
              }
#pragma unroll
              for (int c = 0; c < 4; c++) o[n][d][c] += acc[c];
            } else {
#pragma unroll
              for (int t = 0; t < 2; t++) mma_f16(o[n][d], a[t], ph[t][n][0], ph[t][n][1]);
            }
          }
        }
      }
      }
      alive = __all_sync(0xFFFFFFFFu, alive);  // and every lane has read the slot
      if (alive && at + C::kSlots < mine) {
        if (at + C::kSlots - batch >= 16) look_ahead(at + C::kSlots, it);
        start(at + C::kSlots);
      }
    }
    if (!it.real || !alive) continue;

    // ---- the item's rows of this warp ----
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int sh = 4; sh < 32; sh <<= 1)
          l[n][j] += __shfl_xor_sync(0xFFFFFFFFu, l[n][j], sh);
    if (from_start && u0 + at == it.i1) {  // the whole item
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int r = it.row0 + 8 * n + 2 * tig + j;
          if (r >= it.rows) continue;
          const float inv = l[n][j] == 0.0f ? 0.0f : 1.0f / l[n][j];
          const int tok = by_group(p, r);
          const unsigned long long to =
              (unsigned long long)(it.first + tok) * p.ldo +
              (unsigned long long)(it.head * p.group + r - tok * p.group) * D + gid;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            store_out<TYPE>(p.out, to + 16 * d, o[n][d][j] * inv);
            store_out<TYPE>(p.out, to + 16 * d + 8, o[n][d][j + 2] * inv);
          }
        }
    } else {
      // kept for the join at the end: an item that began before this warp, behind the ring; one
      // that goes on after it (its last), in the ring, whose copies have all arrived
      const int e = from_start ? 1 : 0;
      float *part = reinterpret_cast<float *>(e ? ring : ring + C::kRing);
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const int r = 8 * n + 2 * tig + j;
#pragma unroll
          for (int d = 0; d < D / 16; d++) {
            part[r * D + 16 * d + gid] = o[n][d][j];
            part[r * D + 16 * d + gid + 8] = o[n][d][j + 2];
          }
          if (gid == 0) {
            part[R * D + r] = m[n][j];
            part[R * D + R + r] = l[n][j];
          }
        }
      if (lane == 0) s_edge[warp][e] = edge_of(it);
    }
  }
  if (!alive) {
    if (lane == 0) attn_refuse(p, 0, APX_ERR_DEVICE_TIMEOUT);
    drain(bar, C::kSlots, at - 1, min(at - 1 + C::kSlots, mine));
  }

  // ---- the join: items that cross warps, each by the warp that has its first part ----
  const S e0 = share.bound(w0), e1 = share.bound(w0 + W);  // this CTA's steps
  if (__syncthreads_or(!alive)) {
    if (whole_items) return;
    if (tid == 0) keep_owed<R, ONE, W, S>(p, e0, e1, s_edge);
    __syncthreads();
  }
  constexpr int E = R * D / 4, Q = D / 4;             // quads of an item's rows, of a row
  auto part_of = [&](int w, int e) {
    return reinterpret_cast<const float *>(smem + w * C::kWarpSmem + (e ? 0 : C::kRing));
  };
  auto add4 = [](float4 &v, float f, const float4 x) {
    v = make_float4(fmaf(f, x.x, v.x), fmaf(f, x.y, v.y), fmaf(f, x.z, v.z), fmaf(f, x.w, v.w));
  };
  auto write4 = [&](const Edge<S> &ed, int r, int d, const float4 v, float inv) {
    const int row = ed.row0 + r;
    if (row >= ed.rows) return;
    const int tok = by_group(p, row);
    store4<TYPE>(p.out,
                 (unsigned long long)(ed.first + tok) * p.ldo +
                     (unsigned long long)(ed.head * p.group + row - tok * p.group) * D + d,
                 make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
  };
  {
    // a bit per warp: whose first edge, whose last edge is used
    const bool used = lane < W && s_edge[lane % W][0].used;
    const S begin = s_edge[lane % W][0].begin;
    const unsigned firsts = __ballot_sync(0xFFFFFFFFu, used);
    unsigned starts = __ballot_sync(0xFFFFFFFFu, lane < W && s_edge[lane % W][1].used);
    // items here: the one that began before this CTA or at its first warp's first step, and each
    // warp's last; their rows go round the warps, one at a time, of prompts eight
    constexpr int U = ONE ? 1 : 8, UNITS = R / U;
    const int items_here = (int)(firsts & 1) + __popc(starts);
    int item = 0;
#pragma unroll 1
    for (int j = warp; j < items_here * UNITS; j += W) {
      while (item < j / UNITS - (int)(firsts & 1)) {
        starts &= starts - 1;
        item++;
      }
      const bool head = (firsts & 1) && j < UNITS;
      const int w = head ? 0 : __ffs(starts) - 1, r = j % UNITS * U;
      const Edge<S> &ed = s_edge[w][head ? 0 : 1];
      // its parts: this one and the first edges of the warps that follow
      const int n =
          __popc(__ballot_sync(0xFFFFFFFFu, used && lane > w && begin == ed.begin)) + 1;
      const float *first = part_of(w, head ? 0 : 1), *rest = part_of(w, 0);
      constexpr int kNext = C::kWarpSmem / 4;  // from a warp's part to the next one's
      if constexpr (!ONE) {
        // lane: row r + lane % U, parts lane / U + i KG
        constexpr int KG = 32 / U, KR = (W + KG - 1) / KG;
        float m[KR], l[KR], f[KR], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < KR; i++) {
          const int k = lane / U + i * KG;
          const float *mine = (k ? rest + min(k, n - 1) * kNext : first) + R * D + r + lane % U;
          m[i] = k < n ? mine[0] : -INFINITY, l[i] = k < n ? mine[R] : 0.0f;
          top = fmaxf(top, m[i]);
        }
#pragma unroll
        for (int o = U; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
#pragma unroll
        for (int i = 0; i < KR; i++) {
          f[i] = m[i] == -INFINITY ? 0.0f : ex2(m[i] - top);
          sum = fmaf(f[i], l[i], sum);
        }
#pragma unroll
        for (int o = U; o < 32; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const bool whole = ed.begin >= e0 && ed.end <= e1;
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        float *dst = p.part + ((size_t)blockIdx.x * 2 + (ed.begin >= e0 ? 1 : 0)) * C::kPart;
        if (!whole && lane < U) {
          dst[R * D + r + lane] = top;
          dst[R * D + R + r + lane] = sum;
        }
#pragma unroll 2
        for (int i = lane; i < U * Q; i += 32) {
          const int u = i / Q, d = 4 * (i % Q);
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          add4(v, __shfl_sync(0xFFFFFFFFu, f[0], u),
               *reinterpret_cast<const float4 *>(first + (r + u) * D + d));
#pragma unroll
          for (int k = 1; k < W; k++) {
            if (k >= n) break;
            add4(v, __shfl_sync(0xFFFFFFFFu, f[k / KG], u + U * (k % KG)),
                 *reinterpret_cast<const float4 *>(rest + k * kNext + (r + u) * D + d));
          }
          const float inv = __shfl_sync(0xFFFFFFFFu, scale, u);
          if (whole) write4(ed, r + u, d, v, inv);
          else *reinterpret_cast<float4 *>(dst + (r + u) * D + d) = v;
        }
        continue;
      }
      const float *mine = (lane ? rest + min(lane, n - 1) * kNext : first) + R * D + r;
      const float m = lane < n ? mine[0] : -INFINITY, l = lane < n ? mine[R] : 0.0f;
      float top = m;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      const float f = m == -INFINITY ? 0.0f : ex2(m - top);
      float sum = f * l;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      top = __shfl_sync(0xFFFFFFFFu, top, 0);
      sum = __shfl_sync(0xFFFFFFFFu, sum, 0);
      const int d = 4 * (lane % Q);  // half the warp idles at D = 64
      const float f0 = __shfl_sync(0xFFFFFFFFu, f, 0);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      add4(v, f0, *reinterpret_cast<const float4 *>(first + r * D + d));
#pragma unroll 4
      for (int k = 1; k < n; k++)
        add4(v, __shfl_sync(0xFFFFFFFFu, f, k),
             *reinterpret_cast<const float4 *>(rest + k * kNext + r * D + d));
      if (lane >= Q) continue;
      if (ed.begin >= e0 && ed.end <= e1) {
        write4(ed, r, d, v, sum == 0.0f ? 0.0f : 1.0f / sum);
      } else {
        float *dst = p.part + ((size_t)blockIdx.x * 2 + (ed.begin >= e0 ? 1 : 0)) * C::kPart;
        *reinterpret_cast<float4 *>(dst + r * D + d) = v;
        if (lane == 0) {
          dst[R * D + r] = top;
          dst[R * D + R + r] = sum;
        }
      }
    }
  }
  // ---- items that cross CTAs: the CTA that arrives last joins their parts, in their order ----
  if (whole_items) return;
  int out_of_cta = 0;  // bit 0: an item began before this CTA; bit 1: one goes on after it
  Edge<S> edge0 = s_edge[0][0], edge1;
  if (edge0.used && edge0.begin < e0) out_of_cta = 1;
  {
    const unsigned any = __ballot_sync(0xFFFFFFFFu, lane < W && (s_edge[lane % W][0].used ||
                                                                 s_edge[lane % W][1].used));
    if (!any) return;
    const int last = 31 - __clz(any);
    edge1 = s_edge[last][s_edge[last][1].used ? 1 : 0];
    if (edge1.end > e1 && edge1.begin >= e0) out_of_cta |= 2;
  }
  if (!out_of_cta) return;  // the same in every thread
  // An item's CTAs: the first holds it as its last item, the others as the one from before.
  fence_acq_rel_gpu();
  __syncthreads();
  if (tid < 2) {
    int n = 0;
    if (out_of_cta >> tid & 1) {
      const S begin = tid ? edge1.begin : edge0.begin;
      const S end = tid ? edge1.end : edge0.end;
      const int a = share.cta_of(begin), all = share.cta_of(end - 1) - a + 1;
      if (atomicAdd(p.count + a, 1u) == (unsigned)all - 1) {
        n = all;
        p.count[a] = 0;  // for the next call
      }
      fence_acq_rel_gpu();
    }
    s_last[tid] = n;
  }
  __syncthreads();
#pragma unroll 1
  for (int e = 0; e < 2; e++) {
    const int n = s_last[e];
    if (!n) continue;
    const Edge<S> ed = e ? edge1 : edge0;
    const float *first = p.part + ((size_t)share.cta_of(ed.begin) * 2 + 1) * C::kPart;
    auto src_of = [&](int k) { return first + (k ? (size_t)(2 * k - 1) * C::kPart : 0); };
    // the parts' factors, then their sum by groups of threads, each a share of the parts; a
    // thread's first eight quads are on their way meanwhile
    constexpr int G = C::kThreads >= E ? C::kThreads / E : 1;
    constexpr int PER = E * G / C::kThreads;  // quads of the rows a thread has
    float *f = reinterpret_cast<float *>(smem), *fl = f + n * R;
    float4 *red = reinterpret_cast<float4 *>(smem + ((n * R * 8 + 15) & ~15));
    float4 x[PER][8 / PER];
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int i = tid + j * C::kThreads, q4 = i % E;
#pragma unroll
      for (int k = 0; k < 8 / PER; k++)
        if (i / E + k * G < n)
          x[j][k] = __ldcg(reinterpret_cast<const float4 *>(src_of(i / E + k * G) + 4 * q4));
    }
    for (int i = tid; i < n * R; i += C::kThreads) {
      const float *part = src_of(i / R) + R * D + i % R;
      f[i] = __ldcg(part);
      fl[i] = __ldcg(part + R);
    }
    __syncthreads();
    for (int r = warp; r < R; r += W) {
      float top = -INFINITY, sum = 0.0f;
      for (int k = lane; k < n; k += 32) top = fmaxf(top, f[k * R + r]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
      for (int k = lane; k < n; k += 32) {
        const float m = f[k * R + r], g = m == -INFINITY ? 0.0f : ex2(m - top);
        f[k * R + r] = g;
        sum += g * fl[k * R + r];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
      if (lane == 0) s_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; j++) {
      const int i = tid + j * C::kThreads, q4 = i % E, r = q4 / Q;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int k = 0; k < 8 / PER; k++)
        if (i / E + k * G < n) add4(v, f[(i / E + k * G) * R + r], x[j][k]);
#pragma unroll 4
      for (int k = i / E + 8 / PER * G; k < n; k += G)
        add4(v, f[k * R + r], __ldcg(reinterpret_cast<const float4 *>(src_of(k) + 4 * q4)));
      if (G == 1) write4(ed, r, q4 % Q * 4, v, s_inv[r]);
      else red[i] = v;
    }
    if (G > 1) {
      __syncthreads();
      for (int i = tid; i < E; i += C::kThreads) {
        float4 v = red[i];
#pragma unroll
        for (int g = 1; g < G; g++) add4(v, 1.0f, red[g * E + i]);
        write4(ed, i / Q, i % Q * 4, v, s_inv[i / Q]);
      }
    }
    __syncthreads();
  }
}

template <int D, int NT, typename S, int TYPE>
cudaError_t launch_split(const AttnArgs &p, int grid, cudaStream_t stream) {
  using C = Cfg<D, NT>;
  auto kern = attn_split_kernel<D, NT, TYPE, S>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_allowed() ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <int D, int NT, typename S>
cudaError_t launch_type(const AttnArgs &p, int grid, cudaStream_t stream) {
  if (p.type == APX_DTYPE_F32) return launch_split<D, NT, S, APX_DTYPE_F32>(p, grid, stream);
  if (p.type == APX_DTYPE_F16) return launch_split<D, NT, S, APX_DTYPE_F16>(p, grid, stream);
  return launch_split<D, NT, S, APX_DTYPE_BF16>(p, grid, stream);
}

template <int D>
cudaError_t launch_rows(const AttnArgs &p, int grid, cudaStream_t stream) {
  if ((long long)p.max_q * p.group <= Cfg<D, 1>::kRows && steps_fit<Cfg<D, 1>::kRows, true>(p))
    return launch_type<D, 1, unsigned>(p, grid, stream);
  if (steps_fit<Cfg<D, 2>::kRows, false>(p)) return launch_type<D, 2, unsigned>(p, grid, stream);
  return launch_type<D, 2, unsigned long long>(p, grid, stream);
}

}  // namespace

// Two partial items per CTA of the largest block, and the arrival counters before them.
constexpr int kCountBytes = 4096;
size_t attn_work_bytes(int sms) {
  return kCountBytes + (size_t)sms * 2 * Cfg<128, 2>::kPart * sizeof(float);
}

cudaError_t launch_attn_kv4(const apx_attn_args &a, const apx_kv4_cache &c,
                            const apx_seq_batch &b, void *work, int sms, cudaStream_t stream) {
  AttnArgs p;
  p.q = a.d_q;
  p.out = a.d_out;
  p.pages = static_cast<const uint8_t *>(c.d_pages);
  p.cu = b.d_cu;
  p.kv_len = b.d_kv_len;
  p.table = b.d_table;
  p.status = a.d_status ? &a.d_status->first : nullptr;
  p.ldq = a.ldq;
  p.ldo = a.ldo;
  p.page_bytes = apx_kv4_page_bytes(c.head_dim, c.page_tokens);
  p.count = static_cast<unsigned *>(work);
  p.part = reinterpret_cast<float *>(static_cast<uint8_t *>(work) + kCountBytes);
  p.n_pages = (int)c.n_pages;
  p.n_seqs = b.n_seqs;
  p.n_tokens = (int)b.n_tokens;
  p.max_q = b.max_q;
  p.max_pages = b.max_pages;
  p.kv_heads = c.n_kv_heads;
  p.group = a.n_heads / c.n_kv_heads;
  p.page_shift = 0;
  while (1 << p.page_shift < c.page_tokens) p.page_shift++;
  // a window with room for all that the table can hold hides no key
  const long long room = (long long)b.max_pages * c.page_tokens;
  p.window = a.window < room ? a.window : 0;
  p.sinks = p.window ? a.sinks : 0;
  p.type = a.type;
  p.scale = a.scale;
  p.group_mul = (unsigned)(0x100000000ull / (unsigned)p.group + 1);
  const int grid = std::min(sms, kCountBytes / 4);
  if (attn_tc_serves(p, c.head_dim, b.max_q)) return launch_attn_tc(p, c.head_dim, b.max_q, stream);
  return c.head_dim == 128 ? launch_rows<128>(p, grid, stream) : launch_rows<64>(p, grid, stream);
}

}  // namespace apx
