// apx_attn_items.cuh — how apx_attn.cu's kernel deals a call's work: steps of 32 keys, the items
// that they belong to, each warp's share of them, and the parts of an item that CTAs owe each other.
//
// Plain integer arithmetic of the call's lengths, the same on the host (where it is tested).
#pragma once

#include "apx_kv4.cuh"

namespace apx {

// S, throughout: the type of a step's number in its call (steps_fit).
constexpr int kStepKeys = 32;
// What a warp loses at an item's end (its rows to keep or write, the next one's to read), in steps:
// items of single tokens carry as many steps without keys, so that warps with a boundary get fewer
// keys (without, at 2, 5 and 8: 64 requests of 100-4096 keys, 64 / 8 heads of 128 53.6 51.1 48.0 49.9
// us; 32 of up to 8000, 12 / 2 of 128 23.4 22.8 21.6 21.2; 48 of 1000, 32 / 4 of 128 20.3 19.6 19.3
// 19.6; 64 of 200-600, 16 / 16 of 64 24.4 25.1 23.7 25.2; prompts lose by it).
constexpr int kItemCost = 5;

// A sequence's steps.  Its blocks of rows pair first with last: a pair has `pair` steps, the
// first block's, then the second's, then filling, steps without keys.  ONE: every sequence has one
// block at most.
template <int R, bool ONE>
struct SeqShape : SeqRows<R, kStepKeys> {
  using Base = SeqRows<R, kStepKeys>;
  int pair;

  __host__ __device__ __forceinline__ void load(const AttnArgs &p, int s) {
    Base::load(p, s);
    const int n = this->nblk;
    if (n <= 0) pair = 0;
    else if (ONE || n == 1) pair = steps(p, 0) + kItemCost;
    else if (!p.window) pair = steps(p, 0) + steps(p, n - 1) + 2;
    else {
      // a window's keys: what the block's positions span, in whole steps
      const int most =
          (int)min((long long)p.window + (R - 1) / p.group + 1, (long long)this->kv);
      pair = 2 * (min(most / kStepKeys + 2 + Base::steps_to(min(p.sinks, this->kv)),
                      Base::steps_to(this->kv)) + 1);
    }
  }
  __host__ __device__ __forceinline__ int steps(const AttnArgs &p, int b) const {
    int end, sink, low;
    this->range(p, b, end, sink, low);
    return max(sink + max(Base::steps_to(end) - low / kStepKeys, 0), 1);  // one writes unseeing rows' zeros
  }
  __host__ __device__ __forceinline__ int pairs() const {
    return ONE ? (this->nblk > 0 ? 1 : 0) : (this->nblk + 1) / 2;
  }
  template <typename S>
  __host__ __device__ __forceinline__ S all(const AttnArgs &p) const {
    return (S)pairs() * (unsigned)pair * (unsigned)p.kv_heads;
  }
};

// One item: the steps [i0, i1) of a block of query rows of a KV head.  `real` is false for a pair's
// filling, steps without keys.
template <typename S>
struct Item {
  S i0, i1;
  int seq, first, rows, p0;  // of its sequence: first query token, rows, position of row 0
  int head, row0;            // its KV head and first row
  int end, sink, low;        // its keys (SeqRows::range)
  bool real;
  __host__ __device__ __forceinline__ int key_of(int st) const {  // its step st
    return (st < sink ? st : st - sink + (int)((unsigned)low / kStepKeys)) * kStepKeys;
  }
};

// The item of step g, which is a step of sequence `seq` or of one behind it; seq0: the steps of the
// call before that sequence.
template <int R, bool ONE, typename S>
__host__ __device__ __forceinline__ Item<S> item_from(const AttnArgs &p, int seq, S seq0, S g) {
  S seq1 = seq0;
  SeqShape<R, ONE> q;
  Item<S> it;
  it.seq = seq - 1;
  do {
    seq0 = seq1;
    q.load(p, ++it.seq);
    seq1 = seq0 + q.template all<S>(p);
  } while (g >= seq1);
  const unsigned nth = (unsigned)((g - seq0) / (unsigned)q.pair), n = q.pairs();
  it.head = (int)(ONE ? nth : nth / n);
  int blk = ONE ? 0 : (int)(nth - it.head * n);
  it.i0 = seq0 + (S)nth * q.pair;
  const S end = it.i0 + q.pair;
  it.i1 = it.i0 + q.steps(p, blk);
  if (!ONE && g >= it.i1 && blk != q.nblk - 1 - blk) {
    blk = q.nblk - 1 - blk;
    it.i0 = it.i1;
    it.i1 = it.i0 + q.steps(p, blk);
  }
  it.real = g < it.i1;
  if (!it.real) it.i1 = end;
  it.first = q.first;
  it.rows = q.rows;
  it.p0 = q.p0;
  it.row0 = blk * R;
  q.range(p, blk, it.end, it.sink, it.low);
  return it;
}

// The steps [c0, c1) dealt to `warps` warps of CTAs of W, in equal shares of `base`, the first
// `rem` one more.
template <int W, typename S>
struct Shares {
  S c0, base;
  unsigned warps, rem;

  __host__ __device__ __forceinline__ Shares(S c0, S c1, unsigned warps)
      : c0(c0), base((c1 - c0) / warps), warps(warps), rem((unsigned)((c1 - c0) - base * warps)) {}
  __host__ __device__ __forceinline__ S bound(unsigned w) const {
    return c0 + min(w, warps) * base + min(w, rem);
  }
  // The CTA that has `step`, where c0 is 0.
  __host__ __device__ __forceinline__ int cta_of(S step) const {
    const S wide = rem * (base + 1);
    return (int)((step < wide ? step / (base + 1) : rem + (step - wide) / base) / W);
  }
};

// One item that crosses a warp's boundary, kept for the join at the end of the CTA.
template <typename S>
struct Edge {
  S begin, end;                 // the item's steps, numbered over the whole call
  int first, rows, head, row0;  // its sequence's first token and rows, its KV head and first row
  int used;
};
template <typename S>
__host__ __device__ __forceinline__ Edge<S> edge_of(const Item<S> &it) {
  return Edge<S>{it.i0, it.i1, it.first, it.rows, it.head, it.row0, 1};
}

// Whether a call's steps, in blocks of R rows (ONE: one a sequence at most), stay below 2^32 whatever
// its lengths are.  A prompt of a quarter of a million tokens with 8 KV heads of 8 query heads each
// does not; with 64-bit numbers the windowed chunks in f32 take 50.2 us in place of 48.9.
template <int R, bool ONE>
inline bool steps_fit(const AttnArgs &p) {
  const double room = (double)p.max_pages * (1 << p.page_shift);
  const double blocks = ONE ? p.n_seqs : (double)p.n_tokens * p.group / R + 2.0 * p.n_seqs;
  return blocks * p.kv_heads * (room / kStepKeys + 3 + kItemCost) < 4294967296.0;
}

// What the CTA of steps [e0, e1) owes to items that cross its ends, from the lengths alone: bit 0
// for one that began before it (edge0), bit 1 for one that begins in it and goes on after (edge1).
template <int R, bool ONE, typename S>
__host__ __device__ inline int owed(const AttnArgs &p, S e0, S e1, Edge<S> &edge0, Edge<S> &edge1) {
  const Item<S> a = item_from<R, ONE, S>(p, 0, 0, e0), b = item_from<R, ONE, S>(p, 0, 0, e1 - 1);
  edge0 = edge_of(a);
  edge1 = edge_of(b);
  return (a.real && a.i0 < e0 ? 1 : 0) | (b.real && b.i0 >= e0 && b.i1 > e1 ? 2 : 0);
}

}  // namespace apx
