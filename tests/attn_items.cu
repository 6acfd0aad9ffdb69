// How the attention over the 4-bit cache deals its work (apeiron_b200/csrc/apx_attn_items.cuh), on
// the host: random batches, every CTA's parts walked as its warps walk them.
#include <cstdio>
#include <map>
#include <random>
#include <vector>

#include "apx_attn_items.cuh"

using namespace apx;

static int failures = 0;
static void fail(const char *what, int round, long long a, long long b) {
  if (failures++ < 10) std::printf("round %d: %s (%lld, %lld)\n", round, what, a, b);
}

struct Call {
  std::vector<int> cu{0}, kv;
  AttnArgs p = {};

  void finish(int group, int kv_heads, int page_shift) {
    int most = 0;
    p.max_q = 1;
    for (size_t s = 0; s < kv.size(); s++) {
      most = std::max(most, kv[s]);
      p.max_q = std::max(p.max_q, cu[s + 1] - cu[s]);
    }
    p.n_seqs = (int)kv.size();
    p.n_tokens = cu.back();
    p.group = group;
    p.group_mul = (unsigned)(0x100000000ull / (unsigned)group + 1);
    p.kv_heads = kv_heads;
    p.page_shift = page_shift;
    p.max_pages = (most >> page_shift) + 1;
    p.cu = cu.data();
    p.kv_len = kv.data();
  }
};

template <int R, bool ONE>
static long long steps_of(const AttnArgs &p) {
  unsigned long long n = 0;
  for (int s = 0; s < p.n_seqs; s++) {
    SeqShape<R, ONE> q;
    q.load(p, s);
    n += q.template all<unsigned long long>(p);
  }
  return (long long)n;
}

// Every step belongs to one item, items follow each other, and a real one has its block's steps.
template <int R, bool ONE>
static void check_items(const AttnArgs &p, int round) {
  const long long total = steps_of<R, ONE>(p);
  std::map<std::vector<long long>, int> seen;
  for (long long at = 0; at < total;) {
    const auto it = item_from<R, ONE, unsigned>(p, 0, 0, at);
    if ((long long)it.i0 > at || (long long)it.i1 <= at) return fail("an item's steps", round, it.i0, at);
    if (it.real && (long long)it.i0 != at) fail("a gap before an item", round, it.i0, at);
    if (it.real && seen[{it.seq, it.head, it.row0}]++) fail("an item twice", round, it.seq, it.row0);
    at = it.i1;
  }
  long long items = 0;
  for (int s = 0; s < p.n_seqs; s++) {
    SeqShape<R, ONE> q;
    q.load(p, s);
    items += (long long)q.nblk * p.kv_heads;
  }
  if (items != (long long)seen.size()) fail("items", round, items, (long long)seen.size());
}

// What a CTA's warps keep for items that they do not have whole, and what follows from it for the
// CTA, against owed(); and that each item's counter sees as many CTAs as the joining one waits for.
template <int R, bool ONE, int W>
static void check_owed(const AttnArgs &p, int grid, int round) {
  const long long total = steps_of<R, ONE>(p);
  if (total == 0) return;
  const Shares<W, unsigned> share(0, total, std::min<long long>((long long)grid * W, total));
  std::map<int, std::map<long long, int>> arrivals;  // counter: of which item, how many
  std::map<long long, long long> end_of;
  for (int cta = 0; cta < grid; cta++) {
    const long long e0 = share.bound(cta * W), e1 = share.bound(cta * W + W);
    if (e0 == e1) continue;
    int kept = 0;
    Edge<unsigned> first = {}, last = {};
    for (int w = 0; w < W; w++) {
      const long long u0 = share.bound(cta * W + w), u1 = share.bound(cta * W + w + 1);
      for (long long at = u0; at < u1;) {
        const auto it = item_from<R, ONE, unsigned>(p, 0, 0, at);
        const long long stop = std::min<long long>(it.i1, u1);
        const bool whole = at == (long long)it.i0 && stop == (long long)it.i1;
        if (it.real && !whole) {
          if (w == 0 && at != (long long)it.i0) first = edge_of(it);
          last = edge_of(it);
        }
        at = stop;
      }
    }
    if (first.used && (long long)first.begin < e0) kept |= 1;
    if (last.used && (long long)last.end > e1 && (long long)last.begin >= e0) kept |= 2;
    Edge<unsigned> edge0, edge1;
    const int owes = owed<R, ONE, unsigned>(p, e0, e1, edge0, edge1);
    if (owes != kept) fail("owed", round, owes, kept);
    if (owes & 1 && (edge0.begin != first.begin || edge0.end != first.end || edge0.head != first.head))
      fail("the item from before", round, edge0.begin, first.begin);
    if (owes & 2 && (edge1.begin != last.begin || edge1.end != last.end || edge1.row0 != last.row0))
      fail("the item that goes on", round, edge1.begin, last.begin);
    for (int e = 0; e < 2; e++)
      if (owes >> e & 1) {
        const auto &ed = e ? edge1 : edge0;
        arrivals[share.cta_of(ed.begin)][ed.begin]++;
        end_of[ed.begin] = ed.end;
      }
  }
  for (auto &[counter, of] : arrivals) {
    if (of.size() != 1) fail("two items at a counter", round, counter, (long long)of.size());
    for (auto &[begin, n] : of) {
      const int all = share.cta_of(end_of[begin] - 1) - share.cta_of(begin) + 1;
      if (n != all) fail("arrivals", round, n, all);
    }
  }
}

// Calls whose steps pass 32 bits: they are known for it, the shares cover them in order, and items
// are found on both sides of 2^32.
static void check_long_calls() {
  Call c;
  for (int s = 0; s < 4; s++) {
    c.cu.push_back(c.cu.back() + 131072);
    c.kv.push_back(131072);
  }
  c.finish(8, 8, 7);
  const long long total = steps_of<16, false>(c.p);
  if (total >> 32 == 0 || steps_fit<16, false>(c.p)) fail("steps", 0, total, 0);
  const Shares<8, unsigned long long> share(0, total, 148 * 8);
  long long covered = 0;
  for (int w = 0; w < 148 * 8; w++) {
    const long long n = (long long)share.bound(w + 1) - (long long)share.bound(w);
    if (n < total / (148 * 8) || n > total / (148 * 8) + 1) fail("a share", w, n, total);
    covered += n;
    if (share.cta_of(share.bound(w)) != w / 8) fail("a share's CTA", w, share.bound(w), w / 8);
  }
  if (covered != total) fail("shares", 0, covered, total);
  for (long long g : {0ll, (1ll << 32) - 1, 1ll << 32, (1ll << 32) + 4321, total - 1}) {
    const auto it = item_from<16, false, unsigned long long>(c.p, 0, 0, g);
    if ((long long)it.i0 > g || (long long)it.i1 <= g || it.seq != g / (total / 4))
      fail("an item past 2^32", 0, g, it.i0);
    if (it.real && it.key_of((int)(g - it.i0)) >= it.end) fail("a key past 2^32", 0, g, it.end);
  }
  Call d;  // shared pages: any number of requests over the same million keys
  for (int s = 0; s < 60000; s++) {
    d.cu.push_back(s + 1);
    d.kv.push_back(1 << 20);
  }
  d.finish(1, 8, 7);
  if (steps_of<8, true>(d.p) >> 32 == 0 || steps_fit<8, true>(d.p)) fail("requests", 0, 60000, 0);
  d.p.n_seqs = 60;
  if (!steps_fit<8, true>(d.p)) fail("requests", 0, 60, 0);
}

// Lengths up to the limit have their steps in ints, on both kernels; past it a sequence is refused.
static void check_longest() {
  Call c;
  c.cu.push_back(40);
  c.kv.push_back(kMaxKvLen);
  c.finish(1, 1, 7);
  for (int window : {0, 1, kMaxKvLen - 3, INT32_MAX}) {
    c.p.window = window;
    SeqShape<16, false> q;
    q.load(c.p, 0);
    SeqRows<256, 128> t;
    t.load(c.p, 0);
    int end, sink, low;
    t.range(c.p, 0, end, sink, low);
    if (q.bad || t.bad || q.steps(c.p, 0) <= 0 || q.pair < q.steps(c.p, 0) + q.steps(c.p, 1) ||
        end != kMaxKvLen || t.steps_to(end) <= low / 128)
      fail("the longest", window, q.pair, low);
  }
  c.kv[0]++;
  c.p.max_pages++;
  SeqRows<256, 128> t;
  t.load(c.p, 0);
  if (!t.bad) fail("past the longest", 0, c.kv[0], 0);
}

int main() {
  check_longest();
  check_long_calls();
  for (int round = 0; round < 400; round++) {
    std::mt19937 rng(round);
    auto pick = [&rng](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    Call c;
    const bool one = round % 2;
    const int group = one ? pick(1, 8) : pick(1, 12), n = pick(1, 20);
    for (int s = 0; s < n; s++) {
      const int q = one ? pick(0, 8 / group) : pick(0, round % 3 ? 40 : 400);
      c.cu.push_back(c.cu.back() + q);
      c.kv.push_back(pick(0, 3) ? pick(0, 2500) : pick(0, 40));
    }
    c.finish(group, pick(1, 4), pick(4, 7));
    c.p.window = pick(0, 2) ? 0 : pick(1, 900);
    c.p.sinks = c.p.window ? pick(0, 70) : 0;
    const int grid = pick(0, 1) ? 148 : pick(1, 40);
    if (one ? !steps_fit<8, true>(c.p) : !steps_fit<16, false>(c.p)) fail("a small call", round, n, 0);
    if (one) {
      check_items<8, true>(c.p, round);
      check_owed<8, true, 16>(c.p, grid, round);
    } else {
      check_items<16, false>(c.p, round);
      check_owed<16, false, 8>(c.p, grid, round);
    }
  }
  if (failures) std::printf("%d failures\n", failures);
  return failures ? 1 : 0;
}
