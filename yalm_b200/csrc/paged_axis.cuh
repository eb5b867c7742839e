// The axis of the paged attention's work, and how blocks share it out (paged_attn.cu).  Integer arithmetic alone, on
// PagedBatch and PagedSeq, which are to be declared before; tests compile it for the host and count the units one by
// one.
#pragma once

namespace yb {

namespace {

constexpr int kKT = 128;       // slots per key tile
constexpr int kFewTiles = 4;   // shares below this are all the same
constexpr int kUnitTiles = 2;  // what a unit's start and end cost, in key tiles
// Key tiles whose products go into one sum of the tensor cores: of a unit of two row tiles, whose sums take a tile in
// eight additions of 16 slots; twice as many of a unit of one, whose two sums have half of a tile each.  The additions
// cut off what does not fit, half a last place each time on average, so a sum of values of one sign lost 3.3e-9 of itself
// a slot, however many: as much as half an fp16 rounding (2^-12) after 75000 slots, 14 roundings after 2^21.  Sums of
// 1024 additions lose a tenth of one at most; they are joined in fp32, rounded to nearest.  That costs 1 to 3 % of a call
// whose blocks have several such sums of a unit (2048 tokens over 65536 slots 2330 -> 2377 us), and nothing below.
constexpr int kSumTiles = 128;

// sum_{i < n} floor((a i + b) / 128), a, b >= 0: each round takes the whole parts out and swaps the roles of the
// axes, as Euclid's algorithm does.  Where a is a power of two (one, two, four ... query heads per kv head) two
// rounds of shifts end it.  The arguments here keep every product below 2^32.
__device__ __forceinline__ unsigned floor_sum(unsigned n, unsigned a, unsigned b) {
  unsigned s = (a >> 7) * (n * (n - 1) / 2) + (b >> 7) * n;
  a &= 127u;
  b &= 127u;
  unsigned y = a * n + b, m = a;
  n = y >> 7;
  b = y & 127u;
  if (!(m & (m - 1))) {
    if (!m) return s;
    const int sh = 31 - __clz(m);
    return s + (128u >> sh) * (n * (n - 1) / 2) + (b >> sh) * n;
  }
  a = 128u;
  while (n) {
    s += (a / m) * (n * (n - 1) / 2) + (b / m) * n;
    a %= m;
    b %= m;
    if (!a) break;
    y = a * n + b;
    n = y / m;
    b = y % m;
    const unsigned t = m;
    m = a;
    a = t;
  }
  return s;
}
// sum_{i < n} floor(max(0, a + i u) / 128)
__device__ __forceinline__ unsigned ramp(int n, int a, int u) {
  if (a < 0) {
    if (a + (n - 1) * u < 128) return 0;
    const int skip = (-a + u - 1) / u;
    n -= skip;
    a += skip * u;
  }
  return n > 0 ? floor_sum((unsigned)n, (unsigned)u, (unsigned)a) : 0u;
}

struct Unit {
  int q0, nq;      // queries [q0, q0 + nq) of the sequence
  int tile0;       // first key tile
  int cost;        // key tiles, at least 1; kUnitTiles more on the axis
  bool none;       // no slot is seen: zeros
};
struct Axis {
  int U, window, K;  // queries per unit, window, kv heads
};
__device__ __forceinline__ Unit unit_of(const Axis& x, const PagedSeq& q, int i) {
  Unit u;
  const int p0 = q.kv - q.n;
  u.q0 = i * x.U;
  u.nq = min(x.U, q.n - u.q0);
  const int end = p0 + u.q0 + u.nq;
  u.tile0 = max(0, p0 + u.q0 - x.window + 1) >> 7;
  u.none = end <= 0;
  u.cost = max(1, ((end + kKT - 1) >> 7) - u.tile0);
  return u;
}
__device__ __forceinline__ int n_units(const Axis& x, const PagedSeq& q) { return q.n <= x.U ? 1 : (q.n + x.U - 1) / x.U; }
// length on the axis of the first m units of a (sequence, kv head), m < n_units: unit i ends at slot p0 + (i + 1) U
__device__ __forceinline__ unsigned units_before(const Axis& x, const PagedSeq& q, int m) {
  if (m == 0) return 0;
  const int p0 = q.kv - q.n;
  return (unsigned)m * (1 + kUnitTiles) + ramp(m, p0 + x.U - 1, x.U) - ramp(m, p0 - x.window + 1, x.U);
}
// ... of all units of a (sequence, kv head)
__device__ __forceinline__ unsigned head_tiles(const Axis& x, const PagedSeq& q) {
  if (q.n <= 0) return 0;
  const int nu = n_units(x, q);
  return units_before(x, q, nu - 1) + (unsigned)unit_of(x, q, nu - 1).cost + kUnitTiles;
}

// Where a block starts, and its share.  Of the axis, key tiles and kUnitTiles a unit, every block takes `share`, the
// first `more` blocks one more.  A unit's start and end (the last product, the outputs, the next first scores) take
// 4000 to 5500 clocks beside 2000 (one row tile) to 3300 (two) for a key tile, so blocks of many short units would be
// the last by far: without them on the axis five prompts of head_dim 64 took 26.1 us, not 22.4, and 64 single tokens
// 110, not 105.5.  (Tiles weighted 2 : 3 by their row tiles: a mixed step 43.6 us, not 45.6, the prompts 24.2, not
// 22.5, three hundred other batches in a model of it 0.3 % less.)
// Shares of a few tiles are all the same instead, and the last blocks have none: they end no later, and cut less
// (one token over 4096 slots 16.2 -> 14.9 us; with shares of 12 tiles a mixed step took 55.5 us, not 51).
template <typename Seq>
struct StartOf {
  Seq sq;
  int seq, head, unit, off;
  int left;                  // length of this block's part of the axis
  unsigned long long begin;  // where it begins
  unsigned long long share;
  int more;
};
using Start = StartOf<PagedSeq>;
// a / b: in 32 bits where both fit, as they nearly always do
__device__ __forceinline__ unsigned long long quot(unsigned long long a, unsigned long long b) {
  if (!((a | b) >> 32)) return (unsigned)a / (unsigned)b;
  return a / b;
}
__device__ __forceinline__ unsigned long long block_begin(unsigned long long share, int more, int c) {
  return share * c + min(c, more);
}
__device__ __forceinline__ void share_out(unsigned long long total, unsigned blocks, unsigned long long& share, int& more) {
  share = quot(total, blocks);
  more = (int)(total - share * blocks);
  if (share < kFewTiles && more) ++share, more = 0;
}
// the block that holds position x
__device__ __forceinline__ int block_of(unsigned long long share, int more, unsigned long long x) {
  const unsigned long long cut = (share + 1) * more;
  return x < cut ? (int)quot(x, share + 1) : more + (int)quot(x - cut, share);
}

// The block's two query buffers.  A unit of two row tiles has one tile in each, which that pipeline alone reads; a unit of one
// has them in turn, and both pipelines read it.  A buffer is free again after two arrivals, one of each that reads it or
// two of the only one: an arrival of a pipeline that does not wait for the buffer could come for the next unit before the
// other one's for this unit, and free it under that one's products.
__device__ __forceinline__ int query_buffer(bool two, int pipeline, int turn) { return two ? pipeline : turn; }
__device__ __forceinline__ int query_releases(bool two) { return two ? 2 : 1; }  // of a pipeline that has read its buffer

// The next piece of this block's share: tiles [t0, t1) of a unit, of which the block has those from `from` on.
template <typename Seq>
struct PieceOf {
  Seq sq;
  int seq, head;
  Unit u;
  int from, t0, t1;
  bool last;  // of the block's pieces of the unit
};
using Piece = PieceOf<PagedSeq>;
template <typename Seq>
struct WalkOf {
  StartOf<Seq> st;
  Seq sq;
  int from;  // of the unit that a piece before this one began; -1: none
  __device__ __forceinline__ explicit WalkOf(const StartOf<Seq>& s) : st(s), sq(s.sq), from(-1) {}
  template <typename Batch>
  __device__ __forceinline__ bool next(const Batch& b, const Axis& x, PieceOf<Seq>& p) {
    do {
      if (st.left <= 0 || st.seq >= b.n_seqs) return false;
      p.sq = sq;
      p.seq = st.seq;
      p.head = st.head;
      p.u = unit_of(x, sq, st.unit);
      const int all = p.u.cost + kUnitTiles;
      int end = min(all, st.off + st.left);
      p.t0 = st.off;
      p.t1 = min(p.u.cost, end);
      p.from = from < 0 ? p.t0 : from;
      const int most = p.u.nq > x.U / 2 ? kSumTiles : 2 * kSumTiles;
      p.last = p.t1 - p.t0 <= most;
      if (!p.last) p.t1 = end = p.t0 + most;
      from = p.last ? -1 : p.from;
      st.left -= end - st.off;
      st.off = end;
      if (end == all && st.left > 0) {
        st.off = 0;
        if (++st.unit >= n_units(x, sq)) {
          st.unit = 0;
          if (++st.head >= x.K) {
            st.head = 0;
            do {
              if (++st.seq >= b.n_seqs) break;
              sq = paged_seq(b, st.seq);
            } while (sq.n <= 0);
          }
        }
      }
    } while (p.t0 >= p.t1);  // no tile, only the rest of a unit's length
    return true;
  }
};
using Walk = WalkOf<PagedSeq>;

}  // namespace

}  // namespace yb
