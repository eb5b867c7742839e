// Compares the closed forms of yalm_b200/csrc/paged_axis.cuh with counting, on the host.  For random batches up to
// the limits of the entry points: lengths on the axis unit by unit, then every block's walk: each key tile of each
// unit once, in order, and each cut unit's records where the merge looks for them.  Prints "ok", or what differs.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#define __device__
#define __forceinline__ inline
static inline int __clz(unsigned x) { return x ? __builtin_clz(x) : 32; }
using std::max;
using std::min;

namespace yb {
struct PagedSeq {
  int row0, n, kv;
};
struct PagedBatch {
  int n_seqs;
  const PagedSeq* seqs;
};
static inline PagedSeq paged_seq(const PagedBatch& b, int s) { return b.seqs[s]; }
}  // namespace yb

#include "paged_axis.cuh"

using namespace yb;
typedef unsigned long long u64;

static std::mt19937_64 rng(12345);
static long long upto(long long n) { return (long long)(rng() % (u64)(n + 1)); }
static int spread(int hi) {  // 0 .. hi, over the logarithm
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

static int pick_window() {
  const int w[] = {1 << 22, 1 << 22, 1, 2, 127, 128, 129, 1 + spread(1 << 21), 1 + spread(5000)};
  return w[upto(8)];
}

static void sequence(int n, int kv, int U, int window, bool deep) {
  const Axis x{U, window, 1};
  const PagedSeq q{0, n, kv};
  const int nu = n_units(x, q);
  CHECK(nu == (n + U - 1) / U, "n %d U %d", n, U);
  u64 sum = 0;
  for (int i = 0; i < nu; ++i) {
    if (deep || i < 3 || i + 3 > nu || i % 97 == 0)
      CHECK(units_before(x, q, i) == sum, "n %d kv %d U %d window %d unit %d: %u, counted %llu", n, kv, U, window, i,
            units_before(x, q, i), sum);
    const Unit u = unit_of(x, q, i);
    // from the definition: queries i U .., the slots that the first and the last of them see
    const long long p0 = (long long)kv - n, q0 = (long long)i * U, last = min<long long>(n, q0 + U) - 1;
    const long long lo = max<long long>(0, p0 + q0 - window + 1), hi = p0 + last;  // slots lo .. hi
    const long long cost = hi < 0 ? 1 : max<long long>(1, hi / 128 - lo / 128 + 1);
    CHECK(u.q0 == q0 && u.nq == last - q0 + 1 && u.none == (hi < 0) && u.cost == cost && u.tile0 == (int)(lo / 128),
          "n %d kv %d U %d window %d unit %d: cost %d, counted %lld", n, kv, U, window, i, u.cost, cost);
    sum += cost + kUnitTiles;
  }
  CHECK(head_tiles(x, q) == sum && sum < (1ull << 31), "n %d kv %d U %d window %d: %u, counted %llu", n, kv, U, window,
        head_tiles(x, q), sum);
}

static void batch(const std::vector<PagedSeq>& seqs, int U, int window, int K, int grid) {
  const Axis x{U, window, K};
  const PagedBatch b{(int)seqs.size(), seqs.data()};
  u64 total = 0;
  for (const PagedSeq& q : seqs) total += (u64)head_tiles(x, q) * K;
  u64 share;
  int more;
  if (!total) return;
  share_out(total, grid, share, more);
  // units in order, with the tiles that blocks have walked; a unit's records: by its first block and the later ones
  struct Want {
    int seq, head, unit, cost;
    u64 begin;
  };
  std::vector<Want> want;
  u64 at = 0;
  for (int s = 0; s < b.n_seqs; ++s)
    for (int h = 0; h < K && seqs[s].n > 0; ++h)
      for (int i = 0; i < n_units(x, seqs[s]); ++i) {
        const int c = unit_of(x, seqs[s], i).cost;
        want.push_back({s, h, i, c, at});
        at += c + kUnitTiles;
      }
  CHECK(at == total, "%llu %llu", at, total);
  size_t w = 0;
  int done = 0, first_block = -1, parts = 0;
  for (int c = 0; c < grid; ++c) {
    const u64 begin = block_begin(share, more, c);
    if (begin >= total) continue;
    Start st{};
    size_t f = std::upper_bound(want.begin(), want.end(), begin, [](u64 v, const Want& a) { return v < a.begin; }) - want.begin() - 1;
    st.sq = seqs[want[f].seq];
    st.seq = want[f].seq;
    st.head = want[f].head;
    st.unit = want[f].unit;
    st.off = (int)(begin - want[f].begin);
    st.left = (int)min<u64>(share + (c < more ? 1 : 0), total - begin);
    Walk walk(st);
    Piece p;
    int begun = 0, ended = 0;  // records that the block leaves
    int from = -1;
    while (walk.next(b, x, p)) {
      CHECK(w < want.size(), "a unit too many in block %d", c);
      const Want& u = want[w];
      CHECK(p.seq == u.seq && p.head == u.head && p.u.q0 == u.unit * U && p.t0 == done && p.t1 > p.t0 && p.t1 <= u.cost,
            "block %d: tiles %d to %d of unit %d of sequence %d", c, p.t0, p.t1, u.unit, u.seq);
      const int most = p.u.nq > U / 2 ? kSumTiles : 2 * kSumTiles;
      CHECK(p.t1 - p.t0 <= most && (p.last || p.t1 - p.t0 == most) && (from < 0 ? p.t0 : from) == p.from,
            "block %d: tiles %d to %d, from %d", c, p.t0, p.t1, p.from);
      done = p.t1;
      from = p.last ? -1 : p.from;
      if (!p.last) continue;
      if (p.from == 0) first_block = c, parts = 0;
      ++parts;
      if (p.from != 0) CHECK(++begun == 1 && c == first_block + parts - 1, "block %d: records of a unit begun before", c);
      if (p.from == 0 && p.t1 < u.cost) {
        CHECK(++ended == 1, "block %d leaves two units", c);
        CHECK(block_of(share, more, u.begin + u.cost - 1) > c, "block %d", c);
      }
      if (done == u.cost) {
        CHECK(block_of(share, more, u.begin) == first_block && block_of(share, more, u.begin + u.cost - 1) == c &&
                  c - first_block + 1 == parts,
              "unit %d of sequence %d: blocks %d to %d in %d parts", u.unit, u.seq, first_block, c, parts);
        done = 0;
        ++w;
      }
    }
    CHECK(from < 0, "block %d ends amid its pieces of a unit", c);
  }
  CHECK(w == want.size() && done == 0, "%zu of %zu units", w, want.size());
}

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 1000;
  const int N = 1 << 20, M = 1 << 21;
  for (int G = 1; G <= 16; ++G) {  // the limits themselves, for every number of query heads per kv head
    const int U = 2 * (128 / G);
    for (int window : {1 << 22, 1, 128, 1 << 20})
      for (int n : {1, U, U + 1, N})
        for (int kv : {0, 1, n - 1, n, M - 1, M}) sequence(n, max(kv, 0), U, window, false);
  }
  for (int r = 0; r < rounds; ++r) {
    const int U = 2 * (128 / (int)(1 + upto(15))), n = 1 + spread(N - 1);
    sequence(n, spread(M), U, pick_window(), n < 4000);
    std::vector<PagedSeq> seqs;
    const int S = 1 + spread(300), new_most = 1 + spread(20000 / S), kv_most = spread(M);
    int row = 0;
    for (int s = 0; s < S; ++s) {
      const int m = (int)upto(3) ? 1 : (int)upto(new_most);
      seqs.push_back({row, m, (int)upto(kv_most)});
      row += m;
    }
    batch(seqs, U, pick_window(), 1 + spread(7), upto(3) ? 148 : 1 + (int)upto(255));
  }
  std::printf("ok\n");
}
