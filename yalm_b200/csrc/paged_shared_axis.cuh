// The axis of the paged attention's work (paged_axis.cuh) for a batch in which groups of sequences share a prefix: before
// the sequences come the groups' prefixes, as sequences of their own, whose tokens are those of the whole group, and
// a sequence of a group begins behind the prefix.  Sequences of few rows (single tokens) lie on an axis of their own, in
// steps of 16 slots, which warps share out (paged_few.cu).  Integer arithmetic alone; tests compile it for the host.
#pragma once

#include "paged_axis.cuh"

namespace yb {

// A group's prefix or a sequence, as the kernel that plans a call (paged_shared.cu) leaves it in the workspace.
struct __align__(16) SharedSeq {
  int row0, n;   // tokens, of a prefix those of all its sequences; n is 0 for a sequence of few rows,
  int few;       // which has its tokens here
  int kv;        // slots, the prefix's among them
  int lo;        // first key tile: 0, or the tiles of the prefix that others look after
  int table;     // row of the page table
  int part;      // where its tokens' parts lie in the workspace; -1: there is no other part of them
  int group;     // of a sequence with a part: its prefix
  int all;       // a prefix: every token sees all of its slots
  int pad[3];
  unsigned long long begin;      // where its units begin on the axis
  unsigned long long few_begin;  // and on that of few rows
};
struct SharedBatch {
  const SharedSeq* seqs;
  int n_seqs;  // with the prefixes
};

__device__ __forceinline__ Unit unit_of(const Axis& x, const SharedSeq& q, int i) {
  Unit u;
  u.q0 = i * x.U;
  u.nq = min(x.U, q.n - u.q0);
  u.tile0 = q.lo;
  const int end = q.all ? q.kv : q.kv - q.n + u.q0 + u.nq;
  u.none = end <= 0;
  u.cost = max(1, ((end + kKT - 1) >> 7) - q.lo);
  return u;
}
__device__ __forceinline__ int n_units(const Axis& x, const SharedSeq& q) { return q.n <= x.U ? 1 : (q.n + x.U - 1) / x.U; }
__device__ __forceinline__ unsigned units_before(const Axis& x, const SharedSeq& q, int m) {
  if (m == 0) return 0;
  if (q.all) return (unsigned)m * ((unsigned)(q.kv >> 7) + kUnitTiles);
  return (unsigned)m * (1 + kUnitTiles) + ramp(m, q.kv - q.n + x.U - 1, x.U) - (unsigned)m * q.lo;
}
__device__ __forceinline__ unsigned head_tiles(const Axis& x, const SharedSeq& q) {
  if (q.n <= 0) return 0;
  const int nu = n_units(x, q);
  return units_before(x, q, nu - 1) + (unsigned)unit_of(x, q, nu - 1).cost + kUnitTiles;
}

// ---- records of rows whose sums other parts join: head_dim sums as float4, then m, then l, each of all `rows` side by
// side.  Places in floats; a record of parts has up to 2^24 rows, 2^31 sums of head_dim 128.
__device__ __forceinline__ size_t record_sum(int rows, int r, int k) { return 4 * ((size_t)k * rows + r); }  // float4 k
__device__ __forceinline__ size_t record_m(int head_dim, int rows, int r) { return (size_t)head_dim * rows + r; }
__device__ __forceinline__ size_t record_l(int head_dim, int rows, int r) { return (size_t)(head_dim + 1) * rows + r; }
// The same from the row's float4 0 on, as the join goes through it: the next float4 `step` float4 further, m at `m`, l `step`
// floats behind that.
struct RecordRow {
  int step;
  long long m;
};
__device__ __forceinline__ RecordRow record_row(int head_dim, int rows, int r) { return {rows, (long long)head_dim * rows - 3ll * r}; }

// ---- few rows: a unit is (sequence, kv head), all its rows at once
constexpr int kFewRows = 8;     // tokens x query heads of a kv head
constexpr int kFewSlots = 16;   // slots of a step: of one page
constexpr int kFewUnit = 4;     // what a unit's start and end cost, in steps
constexpr int kFewLeast = 8;    // a warp's least share
__device__ __forceinline__ int few_steps(const SharedSeq& q) { return max(1, ((q.kv + kFewSlots - 1) / kFewSlots) - q.lo * (kKT / kFewSlots)); }
__device__ __forceinline__ unsigned few_length(const SharedSeq& q) { return q.few > 0 ? (unsigned)(few_steps(q) + kFewUnit) : 0u; }
__device__ __forceinline__ void few_share(unsigned long long total, unsigned warps, unsigned long long& share, int& more) {
  share_out(total, warps, share, more);
  if (share < kFewLeast) share = kFewLeast, more = 0;
}

}  // namespace yb
