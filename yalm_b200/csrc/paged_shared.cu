// The plan of an attention call over shared prefixes: from the lengths on the device, what of each group's prefix is
// looked after once for all its sequences, and where every prefix and sequence begins on the axis of the work.
//
// A group's prefix is cut to the slots that all its sequences with new tokens have cached before them, in whole key
// tiles of 128 (the rest of it is each sequence's own work: its table has those pages too), so every token of the
// group sees all of it and no mask is needed.  It is computed once if that halves its passes over the prefix at least:
// with U tokens a unit, sum_s ceil(n_s / U) >= 2 ceil(sum_s n_s / U).  Long chunks fill their units by themselves.
//
// One block, for small batches of few threads: a few loads a sequence, prefix sums, and 64 bytes written for each.  (4 to 5 us
// for 64 sequences; thousands are worked through by 1024 threads one after the other.)
#include <math.h>

#include "launch.h"
#include "paged_shared.cuh"

namespace yb {

namespace {

typedef unsigned long long u64;

template <int kThreads>
__global__ void __launch_bounds__(kThreads, 1) paged_shared_plan_kernel(const __grid_constant__ SharedPlanArgs a) {
  constexpr int kWarps = kThreads / 32;
  __shared__ int s_start[kMaxGroups + 1];  // first sequences
  __shared__ int s_cut[kMaxGroups];        // slots, then key tiles of the prefix that are computed once
  __shared__ int s_units[kMaxGroups];      // units of the sequences, each by itself, then where their tokens' parts begin
  __shared__ int s_row0[kMaxGroups + 1];  // first rows
  __shared__ int s_first[kMaxGroups];     // the first sequence with new tokens, whose row of the table is read
  int* const s_part = s_units;
  __shared__ u64 s_warp[2][kWarps];
  const PagedBatch& b = a.b;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = b.n_heads / b.n_kv_heads;
  pdl_trigger();  // the next kernel waits for this one's end
  pdl_wait();
  // (on its way beside the groups)
  const PagedSeq ahead = (int)threadIdx.x < b.n_seqs ? paged_seq(b, threadIdx.x) : PagedSeq{};
  for (int g = threadIdx.x; g <= a.n_groups; g += kThreads) {
    s_start[g] = min(max(__ldca(a.group_start + g), 0), b.n_seqs);
    if (g < a.n_groups) {
      s_cut[g] = min(max(__ldca(a.prefix_len + g), 0), b.max_pages << b.ps_log2);
      s_units[g] = 0;
      s_first[g] = b.n_seqs - 1;
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
  auto row_of = [&](int s) { return min(max(__ldca(b.q_start + s), 0), b.n_tokens); };
  for (int g = threadIdx.x; g <= a.n_groups; g += kThreads) s_row0[g] = row_of(s_start[g]);
  auto rows_of = [&](int g) { return s_start[g + 1] > s_start[g] ? max(s_row0[g + 1] - s_row0[g], 0) : 0; };
  for (int s = threadIdx.x; s < b.n_seqs; s += kThreads) {
    const PagedSeq q = s == (int)threadIdx.x ? ahead : paged_seq(b, s);
    const int g = q.n > 0 ? group_of(s) : -1;
    if (g >= 0) {
      atomicMin(&s_cut[g], q.kv - q.n);
      atomicAdd(&s_units[g], (q.n + a.x.U - 1) / a.x.U);
      atomicMin(&s_first[g], s);
    }
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
      const int g = g0 + lane;
      int rows = 0, tiles = 0;
      if (g < a.n_groups) {
        rows = rows_of(g);
        tiles = max(s_cut[g], 0) / kKT;
        if (!rows || s_units[g] < 2 * ((rows + a.x.U - 1) / a.x.U)) tiles = 0;
        if (!tiles) rows = 0;
      }
      int upto = rows;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      // (groups that overlap, which the caller must not give, could have more than there is room for)
      if (g < a.n_groups) {
        s_part[g] = at + upto - rows;
        s_cut[g] = at + upto <= a.part_tokens ? tiles : 0;
      }
      at = min(at + __shfl_sync(0xffffffffu, upto, 31), 1 << 21);
    }
  }
  __syncthreads();
  const int all = a.n_groups + b.n_seqs;
  auto seq_at = [&](int v) {
    SharedSeq q{};
    q.part = -1;
    if (v < a.n_groups) {
      q.row0 = s_row0[v];
      q.n = s_cut[v] ? rows_of(v) : 0;
      q.kv = s_cut[v] * kKT;
      q.table = s_first[v];
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
      const int at = q.row0 - s_row0[g];
      if (at >= 0 && at + p.n <= rows_of(g)) {  // (else q_start decreases)
        q.lo = s_cut[g];
        q.part = s_part[g] + at;
        q.group = g;
      }
    }
    return q;
  };
  const int per = (all + kThreads - 1) / kThreads, v0 = min(all, (int)threadIdx.x * per), v1 = min(all, v0 + per);
  SharedSeq one{};
  u64 mine = 0, few = 0;
  for (int v = v0; v < v1; ++v) {
    one = seq_at(v);
    mine += (u64)head_tiles(a.x, one) * a.x.K;
    few += (u64)few_length(one) * a.x.K;
  }
  u64 at = mine, few_at = few;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, at, o), y = __shfl_up_sync(0xffffffffu, few_at, o);
    if (lane >= o) at += x, few_at += y;
  }
  if (lane == 31) {
    s_warp[0][warp] = at;
    s_warp[1][warp] = few_at;
  }
  __syncthreads();
  u64 total = 0, few_total = 0;
  at -= mine;
  few_at -= few;
  for (int i = 0; i < kWarps; ++i) {
    if (i == warp) at += total, few_at += few_total;
    total += s_warp[0][i];
    few_total += s_warp[1][i];
  }
  for (int v = v0; v < v1; ++v) {
    SharedSeq q = per == 1 ? one : seq_at(v);
    q.begin = at;
    q.few_begin = few_at;
    at += (u64)head_tiles(a.x, q) * a.x.K;
    few_at += (u64)few_length(q) * a.x.K;
    a.seqs[v] = q;
  }
  if (warp == kWarps - 1) {
    // SMs for the one kernel and the other: the least of the longer time.  An SM takes 6 us and 2.2 us a key tile, or 3 us and
    // 0.136 us a step of few rows (of 8 KB, as fast as one SM reads); all SMs together no less than 0.0013 us a step.
    const float tiles = (float)total * 2.2f, steps = (float)few_total * (a.head_dim == 128 ? 1.f : 0.6f);
    float best = INFINITY;
    int blocks = 0;
    for (int n = lane; n <= a.grid; n += 32) {
      const float t = fmaxf(n ? 6.f + __fdividef(tiles, (float)n) : total ? INFINITY : 0.f,
                            fmaxf(n < a.grid ? 3.f + __fdividef(steps * 0.136f, (float)(a.grid - n)) : few_total ? INFINITY : 0.f,
                                  steps * 0.0013f));
      if (t < best) best = t, blocks = n;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float t = __shfl_xor_sync(0xffffffffu, best, o);
      const int n = __shfl_xor_sync(0xffffffffu, blocks, o);
      if (t < best || (t == best && n < blocks)) best = t, blocks = n;
    }
    if (lane == 0) {
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
  // a thread for each prefix and sequence where 1024 are enough: sums over few warps are short
  const int all = a.n_groups + a.b.n_seqs, threads = all <= 256 ? 256 : all <= 512 ? 512 : 1024;
  const void* fn = threads == 256   ? reinterpret_cast<const void*>(&paged_shared_plan_kernel<256>)
                   : threads == 512 ? reinterpret_cast<const void*>(&paged_shared_plan_kernel<512>)
                                    : reinterpret_cast<const void*>(&paged_shared_plan_kernel<1024>);
  return launch_kernel(fn, dim3(1), dim3(threads), 0, s, true, &p);
}

}  // namespace yb
