// apx_attn_items.cuh — how apx_attn.cu's kernel deals a call's work: steps of 32 keys, the items
// that they belong to, each warp's share of them, and the parts of an item that CTAs owe each other.
//
// Plain integer arithmetic of the call's lengths, the same on the host (where it is tested).
#pragma once

#include "apx_kv4.cuh"

namespace apx {

constexpr int kStepKeys = 32;
// What a warp loses at an item's end (its rows to keep or write, the next one's to read), in steps:
// items of single tokens carry as many steps without keys, so that warps with a boundary get fewer
// keys (64 ragged requests: 53.2 us without, 51.4 at 2, 48.7 at 5; prompts lose by it).
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
    int end, sink, from;
    this->range(p, b, end, sink, from);
    return max(sink + max(Base::steps_to(end) - from, 0), 1);  // one writes unseeing rows' zeros
  }
  __host__ __device__ __forceinline__ int pairs() const {
    return ONE ? (this->nblk > 0 ? 1 : 0) : (this->nblk + 1) / 2;
  }
};

// One item: the steps [i0, i1) of a block of query rows of a KV head.  `real` is false for a pair's
// filling, steps without keys.
struct Item {
  unsigned i0, i1;
  int seq, first, rows, p0;  // of its sequence: first query token, rows, position of row 0
  int head, row0;            // its KV head and first row
  int end, sink, from;       // its keys (SeqRows::range)
  bool real;
  __host__ __device__ __forceinline__ int key_of(unsigned step) const {
    const int st = (int)(step - i0);
    return (st < sink ? st : st - sink + from) * kStepKeys;
  }
};

// The item of step g, which is a step of sequence `seq` or of one behind it; seq0: the steps of the
// call before that sequence.
template <int R, bool ONE>
__host__ __device__ __forceinline__ Item item_from(const AttnArgs &p, int seq, unsigned seq0,
                                                   unsigned g) {
  unsigned seq1 = seq0;
  SeqShape<R, ONE> q;
  Item it;
  it.seq = seq - 1;
  do {
    seq0 = seq1;
    q.load(p, ++it.seq);
    seq1 = seq0 + (unsigned)q.pairs() * q.pair * p.kv_heads;
  } while (g >= seq1);
  const unsigned nth = (g - seq0) / (unsigned)q.pair, n = q.pairs();
  it.head = (int)(ONE ? nth : nth / n);
  int blk = ONE ? 0 : (int)(nth - it.head * n);
  it.i0 = seq0 + nth * q.pair;
  const unsigned end = it.i0 + q.pair;
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
  q.range(p, blk, it.end, it.sink, it.from);
  return it;
}

// The steps [c0, c1) dealt to `warps` warps of CTAs of W, in equal shares of `base`, the first
// `rem` one more.
template <int W>
struct Shares {
  unsigned c0, warps, base, rem;

  __host__ __device__ __forceinline__ Shares(unsigned c0, unsigned c1, unsigned warps)
      : c0(c0), warps(warps), base((c1 - c0) / warps), rem((c1 - c0) - base * warps) {}
  __host__ __device__ __forceinline__ unsigned bound(unsigned w) const {
    return c0 + min(w, warps) * base + min(w, rem);
  }
  // The CTA that has `step`, where c0 is 0.
  __host__ __device__ __forceinline__ int cta_of(unsigned step) const {
    const unsigned wide = rem * (base + 1);
    return (int)((step < wide ? step / (base + 1) : rem + (step - wide) / base) / W);
  }
};

// One item that crosses a warp's boundary, kept for the join at the end of the CTA.
struct Edge {
  unsigned begin, end;          // the item's steps, numbered over the whole call
  int first, rows, head, row0;  // its sequence's first token and rows, its KV head and first row
  int used;
};
__host__ __device__ __forceinline__ Edge edge_of(const Item &it) {
  return Edge{it.i0, it.i1, it.first, it.rows, it.head, it.row0, 1};
}

// What the CTA of steps [e0, e1) owes to items that cross its ends, from the lengths alone: bit 0
// for one that began before it (edge0), bit 1 for one that begins in it and goes on after (edge1).
template <int R, bool ONE>
__host__ __device__ inline int owed(const AttnArgs &p, unsigned e0, unsigned e1, Edge &edge0,
                                    Edge &edge1) {
  const Item a = item_from<R, ONE>(p, 0, 0, e0), b = item_from<R, ONE>(p, 0, 0, e1 - 1);
  edge0 = edge_of(a);
  edge1 = edge_of(b);
  return (a.real && a.i0 < e0 ? 1 : 0) | (b.real && b.i0 >= e0 && b.i1 > e1 ? 2 : 0);
}

}  // namespace apx
