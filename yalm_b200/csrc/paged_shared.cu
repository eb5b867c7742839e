// The plan of an attention call over shared prefixes: from the lengths on the device, what of each group's prefix is
// looked after once for all its sequences, and where every prefix and sequence begins on the axis of the work.
//
// A group's prefix is cut to the slots that all its sequences with new tokens have cached before them, in whole key
// tiles of 128 (the rest of it is each sequence's own work: its table has those pages too), so every token of the
// group sees all of it and no mask is needed.  It is computed once if that halves its passes over the prefix at least:
// with U tokens a unit, sum_s ceil(n_s / U) >= 2 ceil(sum_s n_s / U).  Long chunks fill their units by themselves.
//
// One block: a few loads a sequence, prefix sums, and 48 bytes written for each.
#include <math.h>

#include "launch.h"
#include "paged_shared.cuh"

namespace yb {

namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
typedef unsigned long long u64;

// Inclusive sum over the block.
__device__ __forceinline__ u64 block_sum(u64 v, u64* s_warp, u64* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  u64 w = s_warp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  const u64 before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  *total = __shfl_sync(0xffffffffu, w, kWarps - 1);
  __syncthreads();
  return v + (warp ? before : 0);
}

__global__ void __launch_bounds__(kThreads, 1) paged_shared_plan_kernel(const __grid_constant__ SharedPlanArgs a) {
  __shared__ int s_start[kMaxGroups + 1];  // first sequences
  __shared__ int s_cut[kMaxGroups];        // slots, then key tiles of the prefix that are computed once
  __shared__ int s_units[kMaxGroups];      // units of the sequences, each by itself
  __shared__ int s_part[kMaxGroups];       // where the group's tokens' parts begin
  __shared__ u64 s_warp[kWarps];
  const PagedBatch& b = a.b;
  pdl_wait();
  for (int g = threadIdx.x; g <= a.n_groups; g += kThreads) {
    s_start[g] = min(max(__ldca(a.group_start + g), 0), b.n_seqs);
    if (g < a.n_groups) {
      s_cut[g] = min(max(__ldca(a.prefix_len + g), 0), b.max_pages << b.ps_log2);
      s_units[g] = 0;
    }
  }
  __syncthreads();
  // the last group that begins at or before the sequence, if it has it: what a sequence of no group gets is -1
  auto group_of = [&](int s) {
    int lo = 0, hi = a.n_groups + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s_start[mid] <= s) lo = mid;
      else hi = mid;
    }
    return lo < a.n_groups && s_start[lo] <= s && s < s_start[lo + 1] ? lo : -1;
  };
  for (int s = threadIdx.x; s < b.n_seqs; s += kThreads) {
    const PagedSeq q = paged_seq(b, s);
    const int g = q.n > 0 ? group_of(s) : -1;
    if (g >= 0) {
      atomicMin(&s_cut[g], q.kv - q.n);
      atomicAdd(&s_units[g], (q.n + a.x.U - 1) / a.x.U);
    }
  }
  __syncthreads();
  // rows of a group's tokens
  auto row_of = [&](int s) { return min(max(__ldca(b.q_start + s), 0), b.n_tokens); };
  auto rows_of = [&](int g, int& row0) {
    row0 = row_of(s_start[g]);
    return s_start[g + 1] > s_start[g] ? max(row_of(s_start[g + 1]) - row0, 0) : 0;
  };
  {
    const int per = (a.n_groups + kThreads - 1) / kThreads, g0 = threadIdx.x * per;
    u64 mine = 0, total;
    for (int g = g0; g < min(a.n_groups, g0 + per); ++g) {
      int row0;
      const int rows = rows_of(g, row0), tiles = max(s_cut[g], 0) / kKT;
      s_cut[g] = rows && s_units[g] >= 2 * ((rows + a.x.U - 1) / a.x.U) ? tiles : 0;
      if (s_cut[g]) mine += rows;
    }
    u64 at = block_sum(mine, s_warp, &total) - mine;
    for (int g = g0; g < min(a.n_groups, g0 + per); ++g) {
      int row0;
      const int rows = s_cut[g] ? rows_of(g, row0) : 0;
      if (at + rows > (u64)a.part_tokens) s_cut[g] = 0;  // (groups that overlap, which the caller must not give)
      s_part[g] = (int)at;
      at += rows;
    }
  }
  __syncthreads();
  const int all = a.n_groups + b.n_seqs, gq = b.n_heads / b.n_kv_heads;
  auto seq_at = [&](int v) {
    SharedSeq q{};
    q.part = -1;
    if (v < a.n_groups) {
      q.n = rows_of(v, q.row0);
      if (!s_cut[v]) q.n = 0;
      q.kv = s_cut[v] * kKT;
      q.table = s_start[v];
      q.part = s_part[v];
      q.all = 1;
      return q;
    }
    const int s = v - a.n_groups, g = group_of(s);
    const PagedSeq p = paged_seq(b, s);
    q.row0 = p.row0;
    q.n = p.n;
    if (p.n * gq <= kFewRows) q.few = p.n, q.n = 0;
    q.kv = p.kv;
    q.table = s;
    if (p.n > 0 && g >= 0 && s_cut[g]) {
      int row0;
      const int rows = rows_of(g, row0), at = q.row0 - row0;
      if (at >= 0 && at + p.n <= rows) {  // (else q_start decreases)
        q.lo = s_cut[g];
        q.part = s_part[g] + at;
        q.group = g;
      }
    }
    return q;
  };
  const int per = (all + kThreads - 1) / kThreads, v0 = threadIdx.x * per;
  u64 mine = 0, few = 0, total, few_total;
  for (int v = v0; v < min(all, v0 + per); ++v) {
    const SharedSeq q = seq_at(v);
    mine += (u64)head_tiles(a.x, q) * a.x.K;
    few += (u64)few_length(q) * a.x.K;
  }
  u64 at = block_sum(mine, s_warp, &total) - mine, few_at = block_sum(few, s_warp, &few_total) - few;
  for (int v = v0; v < min(all, v0 + per); ++v) {
    SharedSeq q = seq_at(v);
    q.begin = at;
    q.few_begin = few_at;
    at += (u64)head_tiles(a.x, q) * a.x.K;
    few_at += (u64)few_length(q) * a.x.K;
    a.seqs[v] = q;
  }
  if (threadIdx.x < 32) {
    // SMs for the one kernel and the other: the least of the longer time.  A key tile of two row tiles takes an SM 1.7 us, a
    // step of few rows 0.11 us (of 8 KB, as fast as one SM reads), but all SMs together no less than 0.0013 us.
    const float tiles = (float)total * 1.7f, steps = (float)few_total * (a.head_dim == 128 ? 1.f : 0.6f);
    float best = INFINITY;
    int blocks = 0;
    for (int n = threadIdx.x; n <= a.grid; n += 32) {
      const float t = fmaxf(n ? tiles / n : total ? INFINITY : 0.f,
                            fmaxf(n < a.grid ? steps * 0.11f / (a.grid - n) : few_total ? INFINITY : 0.f, steps * 0.0013f));
      if (t < best) best = t, blocks = n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, best, o);
      const int n = __shfl_xor_sync(0xffffffffu, blocks, o);
      if (t < best || (t == best && n < blocks)) best = t, blocks = n;
    }
    if (threadIdx.x == 0) {
      SharedHead h;
      h.total = total;
      share_out(total, max(blocks, 1), h.share, h.more);
      h.few_total = few_total;
      few_share(few_total, max(a.grid - blocks, 1) * kFewWarps, h.few_share, h.few_more);
      *a.head = h;
    }
  }
}

}  // namespace

cudaError_t paged_shared_plan(const SharedPlanArgs& a, cudaStream_t s) {
  SharedPlanArgs p = a;
  return launch_kernel(reinterpret_cast<const void*>(&paged_shared_plan_kernel), dim3(1), dim3(kThreads), 0, s, true, &p);
}

}  // namespace yb
