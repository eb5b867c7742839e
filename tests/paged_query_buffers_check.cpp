// The hand-over of the paged attention's two query buffers (yalm_b200/csrc/paged_axis.cuh) between the warp that loads
// them and the two that issue products, in every order in which their steps can happen, for every sequence of up to six
// units of one or two row tiles.  No buffer may be written while products read it, products read what was loaded for them,
// and all come to their end.  Prints "ok", or the sequence that fails.
#include <algorithm>
#include <array>
#include <cstdio>
#include <cstdlib>
#include <set>
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
};
static inline PagedSeq paged_seq(const PagedBatch&, int) { return {}; }
}  // namespace yb

#include "paged_axis.cuh"

using namespace yb;

// Barriers as the hardware has them: a wait for a parity passes when the phase before the one under way has it.
struct State {
  int load = 0, half = 0;                  // the loader's unit, and its buffer of it
  int unit[2] = {0, 0}, stage[2] = {0, 0};  // of a product warp: 0 waits, 1 reads, 2 has read
  int full[2] = {0, 0};                    // phases over
  int empty[2] = {0, 0}, left[2] = {2, 2};  // phases over, arrivals still awaited
  int holds[2] = {-1, -1}, landing[2] = {-1, -1};  // the tile (2 unit + row tile) in a buffer, or on its way to it
  std::array<int, 20> key() const {
    return {load, half, unit[0], unit[1], stage[0], stage[1], full[0], full[1], empty[0], empty[1],
            left[0], left[1], holds[0], holds[1], landing[0], landing[1], 0, 0, 0, 0};
  }
};
static bool passes(int phases_over, int phase) { return ((phases_over - 1) & 1) == (phase & 1); }

static std::vector<bool> two;      // the units
static std::vector<int> turn;      // the buffer of a unit of one row tile
static const char* wrong;
static std::set<std::array<int, 20>> seen;

static int uses_before(int u, int buffer) {
  int n = 0;
  for (int i = 0; i < u; ++i) n += two[i] || turn[i] == buffer;
  return n;
}
static void go(const State& s) {
  if (wrong || !seen.insert(s.key()).second) return;
  const int N = (int)two.size();
  bool any = false;
  if (s.load < N) {  // the loader: a buffer that it has used before is waited for, then a copy is on its way
    const int b = two[s.load] ? s.half : turn[s.load], uses = uses_before(s.load, b);
    if (!uses || passes(s.empty[b], uses - 1)) {
      any = true;
      State t = s;
      for (int p = 0; p < 2; ++p)
        if (s.stage[p] == 1 && query_buffer(two[s.unit[p]], p, turn[s.unit[p]]) == b) wrong = "a buffer is written while products read it";
      if (s.landing[b] >= 0) wrong = "a buffer has two copies on their way";
      t.holds[b] = -1;
      t.landing[b] = 2 * s.load + (two[s.load] ? s.half : 0);
      if (two[s.load] && !s.half) t.half = 1;
      else t.half = 0, ++t.load;
      go(t);
    }
  }
  for (int b = 0; b < 2; ++b)
    if (s.landing[b] >= 0) {
      any = true;
      State t = s;
      t.holds[b] = s.landing[b];
      t.landing[b] = -1;
      ++t.full[b];
      go(t);
    }
  for (int p = 0; p < 2; ++p) {
    const int u = s.unit[p];
    if (u >= N) continue;
    const int b = query_buffer(two[u], p, turn[u]);
    if (s.stage[p] == 0) {
      if (!passes(s.full[b], uses_before(u, b))) continue;
      any = true;
      State t = s;
      t.stage[p] = 1;
      if (s.holds[b] != 2 * u + (two[u] ? p : 0)) wrong = "products read another tile";
      go(t);
    } else if (s.stage[p] == 1) {
      any = true;
      State t = s;
      t.stage[p] = 2;
      for (int k = 0; k < query_releases(two[u]); ++k)
        if (!--t.left[b]) ++t.empty[b], t.left[b] = 2;
      go(t);
    } else {
      // the pipelines' softmaxes take turns, a step each: pipeline 1 ends a unit after pipeline 0's last step of it, and
      // pipeline 0 after the step of pipeline 1 before that, of the same unit if it has two steps at least
      const int o = p ^ 1, need = p == 1 || two[u] ? u : u - 1;
      if (s.unit[o] < need || (s.unit[o] == need && s.stage[o] < 2)) continue;
      any = true;
      State t = s;
      t.stage[p] = 0;
      ++t.unit[p];
      go(t);
    }
  }
  if (!any && (s.load < N || s.unit[0] < N || s.unit[1] < N) && !wrong) wrong = "all wait";
}

int main() {
  for (int n = 1; n <= 6; ++n)
    for (int bits = 0; bits < 1 << n; ++bits) {
      two.assign(n, false);
      turn.assign(n, 0);
      for (int i = 0, next = 0; i < n; ++i) {
        two[i] = (bits >> i) & 1;
        turn[i] = next;
        if (!two[i]) next ^= 1;
      }
      wrong = nullptr;
      seen.clear();
      go(State{});
      if (wrong) {
        printf("%s: row tiles", wrong);
        for (int i = 0; i < n; ++i) printf(" %d", two[i] ? 2 : 1);
        puts("");
        return 1;
      }
    }
  puts("ok");
}
