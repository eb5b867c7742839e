// Compares where yalm_b200/csrc/paged_shared_axis.cuh has the rows' records written and joined with wide arithmetic, on
// the host: records of every size up to that of the largest batch that is accepted (2^20 tokens of 16 query heads a kv
// head).  Prints "ok", or what differs.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>

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
typedef __int128 wide;

static void fail(const char* what, int hd, int rows, int r) {
  printf("%s: head_dim %d, %d rows, row %d\n", what, hd, rows, r);
  exit(1);
}

static void check(int hd, int rows, int r) {
  const wide m = (wide)hd * rows + r, l = (wide)(hd + 1) * rows + r;
  if ((wide)record_m(hd, rows, r) != m || (wide)record_l(hd, rows, r) != l) fail("m or l", hd, rows, r);
  const wide at = record_sum(rows, r, 0);
  const RecordRow j = record_row(hd, rows, r);
  if (at + j.m != m || at + j.m + j.step != l) fail("the join's m or l", hd, rows, r);
  for (int k = 0; k < hd / 4; ++k) {
    if ((wide)record_sum(rows, r, k) != 4 * ((wide)k * rows + r)) fail("sums", hd, rows, r);
    if (at + (wide)4 * k * j.step != (wide)record_sum(rows, r, k)) fail("the join's sums", hd, rows, r);
  }
}

int main() {
  std::mt19937 rng(99);
  const int most = 16 << 20;
  for (int hd : {64, 128}) {
    for (int rows : {1, 4, 5, 256, most / 2, most - 4, most})
      for (int r : {0, 1, rows / 2, rows - 1})
        if (r < rows) check(hd, rows, r);
    for (int i = 0; i < 20000; ++i) {
      const int rows = 1 + (int)(rng() % (unsigned)(1 << (1 + rng() % 24)));
      check(hd, rows, (int)(rng() % (unsigned)rows));
    }
    std::set<size_t> seen;  // of a small record, every float once
    const int rows = 12;
    for (int r = 0; r < rows; ++r) {
      for (int k = 0; k < hd / 4; ++k)
        for (int i = 0; i < 4; ++i) seen.insert(record_sum(rows, r, k) + i);
      seen.insert(record_m(hd, rows, r));
      seen.insert(record_l(hd, rows, r));
    }
    if (seen.size() != (size_t)(hd + 2) * rows || *seen.rbegin() != seen.size() - 1) fail("places", hd, rows, 0);
  }
  puts("ok");
}
