// Compares the arithmetic of yalm_b200/csrc/paged_shared_axis.cuh with counting, on the host: batches of prefixes and
// sequences as the planning kernel leaves them.  Both axes unit by unit, the walk of every block, and where the join
// looks for the records of cut units.  Prints "ok", or what differs.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define __device__
#define __forceinline__ inline
#define __align__(n) alignas(n)
static inline int __clz(unsigned x) { return x ? __builtin_clz(x) : 32; }
using std::max;
using std::min;

namespace yb {
struct PagedSeq {  // (not used here)
  int row0, n, kv;
};
struct PagedBatch {
  int n_seqs;
};
static inline PagedSeq paged_seq(const PagedBatch&, int) { return {}; }
struct SharedSeq;
struct SharedBatch;
static inline SharedSeq paged_seq(const SharedBatch& b, int v);
}  // namespace yb

#include "paged_shared_axis.cuh"

namespace yb {
static inline SharedSeq paged_seq(const SharedBatch& b, int v) { return b.seqs[v]; }
}  // namespace yb

using namespace yb;
typedef unsigned long long u64;

static std::mt19937_64 rng(4321);
static long long upto(long long n) { return (long long)(rng() % (u64)(n + 1)); }
static int spread(int hi) {
  const int bits = (int)upto(32 - __clz((unsigned)hi));
  return (int)min<long long>(hi, upto((1ll << bits)));
}

#define CHECK(c, ...)                  \
  do {                                 \
    if (!(c)) {                        \
      std::printf("%s: ", #c);         \
      std::printf(__VA_ARGS__);        \
      std::printf("\n");               \
      std::exit(1);                    \
    }                                  \
  } while (0)

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 500;
  for (int r = 0; r < rounds; ++r) {
    const int gq = 1 + (int)upto(15), U = 2 * (128 / gq), K = 1 + spread(7), S = 1 + spread(200), groups = 1 + spread(6);
    const Axis x{U, 1 << 22, K};
    std::vector<SharedSeq> seqs;
    int row = 0;
    std::vector<SharedSeq> own;
    std::vector<int> rows(groups, 0), cut(groups, 0), first_row(groups, 0);
    for (int g = 0; g < groups; ++g) cut[g] = upto(3) ? spread(2000) : 0;
    int part = 0, at_group = -1;
    for (int s = 0; s < S; ++s) {
      const int g = (int)((long long)s * groups / S), n = upto(4) ? 1 : (int)upto(3 * U);
      if (g != at_group) at_group = g, first_row[g] = row;
      SharedSeq q{};
      q.row0 = row;
      (n * gq <= kFewRows ? q.few : q.n) = n;
      q.kv = cut[g] * kKT + spread(20000) + n;
      if (!cut[g] && !upto(9)) q.kv = (int)upto(n);  // fewer slots than tokens
      q.lo = cut[g];
      q.part = cut[g] ? part + row - first_row[g] : -1;
      q.group = g;
      row += n;
      rows[g] += n;
      own.push_back(q);
    }
    for (int g = 0; g < groups; ++g) {
      SharedSeq q{};
      q.row0 = first_row[g];
      q.n = cut[g] ? rows[g] : 0;
      q.kv = cut[g] * kKT;
      q.all = 1;
      seqs.push_back(q);
    }
    seqs.insert(seqs.end(), own.begin(), own.end());
    // lengths by counting, and where everything begins
    struct Want {
      int seq, head, unit, cost;
      u64 begin;
    };
    std::vector<Want> want, few;
    u64 total = 0, few_total = 0;
    for (int v = 0; v < (int)seqs.size(); ++v) {
      SharedSeq& q = seqs[v];
      q.begin = total;
      q.few_begin = few_total;
      for (int h = 0; h < K; ++h) {
        u64 in_head = 0;
        for (int i = 0; q.n > 0 && i < (q.n + U - 1) / U; ++i) {
          const int nq = min(U, q.n - i * U);
          const long long end = q.all ? q.kv : (long long)q.kv - q.n + i * U + nq;  // slots before it are seen
          const int cost = (int)max<long long>(1, (end + 127) / 128 - q.lo);
          const Unit u = unit_of(x, q, i);
          CHECK(u.q0 == i * U && u.nq == nq && u.tile0 == q.lo && u.cost == cost && u.none == (end <= 0), "unit %d of %d: %d %d", i, v, u.cost, cost);
          CHECK(units_before(x, q, i) == in_head, "unit %d of %d: %u, counted %llu", i, v, units_before(x, q, i), in_head);
          want.push_back({v, h, i, cost, total});
          total += cost + kUnitTiles;
          in_head += cost + kUnitTiles;
        }
        CHECK(head_tiles(x, q) == in_head, "%d: %u, counted %llu", v, head_tiles(x, q), in_head);
        if (q.few > 0) {
          const int steps = max(1, (q.kv + 15) / 16 - 8 * q.lo);
          CHECK(few_steps(q) == steps && few_length(q) == (unsigned)steps + kFewUnit, "%d", v);
          few.push_back({v, h, 0, steps, few_total});
          few_total += steps + kFewUnit;
        } else {
          CHECK(few_length(q) == 0, "%d", v);
        }
      }
    }
    const SharedBatch b{seqs.data(), (int)seqs.size()};
    // ---- the blocks' walk
    const int blocks = 1 + (int)upto(147);
    u64 share;
    int more;
    size_t w = 0;
    int done = 0;
    if (total) {
      share_out(total, blocks, share, more);
      for (int c = 0; c < blocks; ++c) {
        const u64 begin = block_begin(share, more, c);
        if (begin >= total) continue;
        const size_t f = std::upper_bound(want.begin(), want.end(), begin, [](u64 v, const Want& a) { return v < a.begin; }) - want.begin() - 1;
        StartOf<SharedSeq> st{};
        st.sq = seqs[want[f].seq];
        st.seq = want[f].seq;
        st.head = want[f].head;
        st.unit = want[f].unit;
        st.off = (int)(begin - want[f].begin);
        st.left = (int)min<u64>(share + (c < more ? 1 : 0), total - begin);
        WalkOf<SharedSeq> walk(st);
        PieceOf<SharedSeq> p;
        while (walk.next(b, x, p)) {
          CHECK(w < want.size(), "a unit too many in block %d", c);
          const Want& u = want[w];
          CHECK(p.seq == u.seq && p.head == u.head && p.u.q0 == u.unit * U && p.t0 == done && p.t1 > p.t0 && p.t1 <= u.cost,
                "block %d: tiles %d to %d of unit %d of %d", c, p.t0, p.t1, u.unit, u.seq);
          done = p.t1;
          if (p.last) {
            CHECK(block_of(share, more, u.begin + done - 1) == c, "block %d", c);
            CHECK(p.from != 0 || block_of(share, more, u.begin) == c, "block %d", c);
          }
          if (done == u.cost) done = 0, ++w;
        }
      }
    }
    CHECK(w == want.size() && !done, "%zu of %zu units", w, want.size());
    // ---- the warps of few rows
    const int warps = 12 * (1 + (int)upto(147));
    few_share(few_total, warps, share, more);
    CHECK(share >= kFewLeast && (share + (more ? 1 : 0)) * warps >= few_total, "%llu", share);
    w = 0;
    done = 0;
    for (int c = 0; c < warps; ++c) {
      const u64 begin = block_begin(share, more, c);
      if (begin >= few_total) continue;
      int left = (int)min<u64>(share + (c < more ? 1 : 0), few_total - begin);
      size_t f = std::upper_bound(few.begin(), few.end(), begin, [](u64 v, const Want& a) { return v < a.begin; }) - few.begin() - 1;
      int off = (int)(begin - few[f].begin);
      for (;;) {
        const int length = few[f].cost + kFewUnit, t0 = off, t1 = min(few[f].cost, off + left);
        if (t0 < t1) {
          CHECK(w == f && t0 == done, "warp %d: steps %d to %d of %zu", c, t0, t1, f);
          CHECK(block_of(share, more, few[f].begin + t0) == c && block_of(share, more, few[f].begin + t1 - 1) == c, "warp %d", c);
          done = t1;
          if (done == few[f].cost) done = 0, ++w;
        }
        left -= min(length - off, left);
        if (left <= 0) break;
        off = 0;
        ++f;
      }
    }
    CHECK(w == few.size() && !done, "%zu of %zu units of few rows", w, few.size());
  }
  std::printf("ok\n");
}
