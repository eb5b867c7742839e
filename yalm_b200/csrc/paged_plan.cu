// The plan of a serving step over the paged KV cache, from the number of tokens r_s that every sequence brings:
//
//   n_s = max(r_s, 0),  q_start[s] = sum_{i < s} n_i,  kv_len[s] = kv_s + n_s (0 where r_s < 0: the sequence ends),
//   pages ceil(kv_s / P) .. ceil(kv_len[s] / P) - 1 of its table from the end of the list of free pages,
//   pos[row] = kv_s + row - q_start[s],  slots[row] = page_table[s][pos / P] P + pos % P.
//
// Ended sequences' pages go behind the free ones first.  Everything lies in the order of (sequence, page), so the
// result is the same on every run: prefix sums, no atomics that hand out places.  A step that does not fit (pages,
// rows, a sequence longer than its table) takes nothing and brings no tokens.
//
// Integers only, a few bytes a sequence and 12 a token: launches and chains of dependent loads are what it costs, so
// pages and tokens are shared out among all threads, each of which finds its sequence by a search of prefix sums in
// shared memory.  One block does all of it for up to kBlockSeqs sequences and kBlockTokens rows.  Larger batches: a
// cluster of 8 blocks does the sums and the pages, each block a stretch of the sequences, with totals exchanged over
// distributed shared memory; a second kernel over the whole GPU writes the tokens' positions and slots.
#include "cluster.cuh"
#include "launch.h"
#include "paged.cuh"

namespace yb {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
// One block or a cluster and a second kernel, by the batch's sequences and the rows it has room for (what a step brings is
// known on the device alone): 256 sequences of 30 tokens 8.4 us by one block and 9.2 by the other, of one token 4.4 and 8.8, 64 of
// one 4.1 and 7.7, 1024 of one 5.1 and 8.8.
constexpr int kBlockSeqs = 1024, kBlockTokens = 8192;
constexpr int kMostSeqs = 65536 / kCluster;  // of a block of the cluster

struct Sums {
  long long rows;  // tokens
  int more, back;  // pages taken; table entries of ended sequences (of a block at most 2^30)
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) { return {a.rows + b.rows, a.more + b.more, a.back + b.back}; }
__device__ __forceinline__ Sums operator-(const Sums& a, const Sums& b) { return {a.rows - b.rows, a.more - b.more, a.back - b.back}; }

// The last i < n with at[i] <= x, where at does not decrease and at[0] <= x: it has x, if any has.
__device__ __forceinline__ int holder(const int* at, int n, int x) {
  int lo = 0;
  while (n - lo > 1) {
    const int mid = (lo + n) / 2;
    if (at[mid] <= x) lo = mid;
    else n = mid;
  }
  return lo;
}

// Four neighbouring rows' positions and slots, r0 a multiple of 4.
constexpr int kRowsEach = 4;
__device__ __forceinline__ void write_rows(const PagedPlanArgs& a, int r0, int rows, const int (&p)[kRowsEach], const int (&page)[kRowsEach]) {
  long long slot[kRowsEach];
#pragma unroll
  for (int k = 0; k < kRowsEach; ++k) slot[k] = a.slots ? paged_slot(a, p[k], page[k]) : 0;
  const bool whole = r0 + kRowsEach <= rows;
  if (a.pos && whole && (reinterpret_cast<uintptr_t>(a.pos) & 15) == 0) {
    *reinterpret_cast<int4*>(a.pos + r0) = make_int4(p[0], p[1], p[2], p[3]);
  } else if (a.pos) {
    for (int k = 0; k < kRowsEach; ++k)
      if (r0 + k < rows) a.pos[r0 + k] = p[k];
  }
  if (a.slots && whole && (reinterpret_cast<uintptr_t>(a.slots) & 15) == 0) {
    reinterpret_cast<longlong2*>(a.slots + r0)[0] = make_longlong2(slot[0], slot[1]);
    reinterpret_cast<longlong2*>(a.slots + r0)[1] = make_longlong2(slot[2], slot[3]);
  } else if (a.slots) {
    for (int k = 0; k < kRowsEach; ++k)
      if (r0 + k < rows) a.slots[r0 + k] = slot[k];
  }
}

template <bool kOne>  // one block and everything in it
__global__ void __launch_bounds__(kThreads, 1) paged_plan_kernel(const __grid_constant__ PagedPlanArgs a) {
  __shared__ Sums s_warp[kWarps];
  __shared__ int s_long[kWarps], s_found[kWarps];
  struct Total {
    Sums sums;     // back: pages that are there
    int too_long;  // the first sequence that is, or INT_MAX
  };
  __shared__ Total s_total;
  // of each of the block's sequences: slots before; the first entry of the table that it takes a page for, or gives one
  // back of; and the sums of the sequences before it: pages, entries, rows
  extern __shared__ int s_dyn[];
  __shared__ int s_one[kOne ? 5 * (kBlockSeqs + 1) : 1];
  int* const s_kv = kOne ? s_one : s_dyn;
  constexpr int kMost = kOne ? kBlockSeqs : kMostSeqs;
  int* const s_from = s_kv + kMost + 1;
  int* const s_take = s_from + kMost + 1;
  int* const s_back = s_take + kMost + 1;
  int* const s_row = s_back + kMost + 1;  // kOne alone
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kOne ? 0 : (int)cluster_ctarank(), blocks = kOne ? 1 : kCluster;
  const int mine = (a.n_seqs + blocks - 1) / blocks;  // sequences of a block
  const int first = min(a.n_seqs, rank * mine), n = min(mine, a.n_seqs - first);
  const int per = (n + kThreads - 1) / kThreads, i0 = min(n, (int)threadIdx.x * per), i1 = min(n, i0 + per);
  const int cap = a.max_pages << a.ps_log2, up = (1 << a.ps_log2) - 1;
  auto held_of = [&](int kv) { return (kv + up) >> a.ps_log2; };
  pdl_wait();
  const int n_free0 = min(max(__ldca(a.n_free_before), 0), a.n_pages);

  // ---- sums over the sequences
  int too_long = 0x7fffffff;
  auto of_seq = [&](int i) {
    const int s = first + i, r = __ldca(a.new_len + s), kept = a.kept ? __ldca(a.kept + s) : 0;
    const int kv = min(max(__ldca(a.kv_before + s), 0), cap), held = held_of(kv);
    Sums w{0, 0, 0};
    s_kv[i] = kv;
    s_from[i] = held;
    if (r < 0) {
      s_from[i] = min(max(kept, 0), held);
      w.back = held - s_from[i];
    } else {
      w.rows = r;
      if (r > cap - kv) too_long = min(too_long, s);
      else w.more = held_of(kv + r) - held;
    }
    return w;
  };
  Sums own{0, 0, 0};
  for (int i = i0; i < i1; ++i) own = own + of_seq(i);
  Sums upto = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v{__shfl_up_sync(0xffffffffu, upto.rows, o), __shfl_up_sync(0xffffffffu, upto.more, o),
                 __shfl_up_sync(0xffffffffu, upto.back, o)};
    if (lane >= o) upto = upto + v;
  }
  too_long = __reduce_min_sync(0xffffffffu, too_long);
  if (lane == 31) {
    s_warp[warp] = upto;
    s_long[warp] = too_long;
  }
  __syncthreads();
  Sums sums = s_warp[lane];
  too_long = __reduce_min_sync(0xffffffffu, s_long[lane]);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v{__shfl_up_sync(0xffffffffu, sums.rows, o), __shfl_up_sync(0xffffffffu, sums.more, o),
                 __shfl_up_sync(0xffffffffu, sums.back, o)};
    if (lane >= o) sums = sums + v;
  }
  auto from_lane = [&](const Sums& v, int l) {
    return Sums{__shfl_sync(0xffffffffu, v.rows, l), __shfl_sync(0xffffffffu, v.more, l), __shfl_sync(0xffffffffu, v.back, l)};
  };
  const Sums block = from_lane(sums, 31);  // of the block
  Sums at = from_lane(sums, max(warp - 1, 0));
  if (warp == 0) at = Sums{0, 0, 0};
  at = at + upto - own;  // before this thread's sequences, in the block
  {
    Sums w = at;
    for (int i = i0; i < i1; ++i) {
      s_take[i] = w.more;
      s_back[i] = w.back;
      if (kOne) s_row[i] = (int)min(w.rows, 0x7fffffffll);
      if (i + 1 < i1) w = w + of_seq(i);
    }
  }
  __syncthreads();

  // A thread's part of `all` entries or pages, in order: f(sequence, the entry within its share, place among all).
  auto share = [&](const int* sums_before, int all, auto&& f) {
    const int each = (all + kThreads - 1) / kThreads, x0 = min(all, (int)threadIdx.x * each), x1 = min(all, x0 + each);
    if (x0 >= x1) return;
    int i = holder(sums_before, n, x0);
    for (int x = x0; x < x1; ++x) {
      while (i + 1 < n && sums_before[i + 1] <= x) ++i;
      f(i, x - sums_before[i], x);
    }
  };
  // ---- pages of ended sequences
  auto entry = [&](int i, int j) { return __ldca(a.page_table + (size_t)(first + i) * a.max_pages + s_from[i] + j); };
  int found = 0, gave = 0, gave_before = 0;  // pages that are there: of this thread, of the block, of the threads before
  if (block.back) {
    share(s_back, block.back, [&](int i, int j, int) {
      const int page = entry(i, j);
      found += page >= 0 && page < a.n_pages;
    });
    int v = found;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) s_found[warp] = v;
    __syncthreads();
    const int w = s_found[lane];
    gave = __reduce_add_sync(0xffffffffu, w);
    gave_before = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0) + v - found;
  }
  auto give_back = [&](int where) {  // the block's first page's place in the list
    where += gave_before;
    if (found)
      share(s_back, block.back, [&](int i, int j, int) {
        const int page = entry(i, j);
        if (page >= 0 && page < a.n_pages && where < a.n_pages) a.free_pages[where++] = page;
      });
  };
  long long rows = block.rows, back = gave, more = block.more, before_more = 0, before_rows = 0, before_back = 0;
  if (!kOne) {
    if (threadIdx.x == 0) s_total = Total{Sums{block.rows, block.more, gave}, too_long};
    cluster_sync_all();
    Total t{Sums{0, 0, 0}, 0x7fffffff};
    if (lane < kCluster) t = *dsmem_ptr(&s_total, lane);
    rows = back = more = 0;
    for (int c = 0; c < kCluster; ++c) {
      if (c == rank) before_rows = rows, before_more = more, before_back = back;
      const Sums v = from_lane(t.sums, c);
      rows += v.rows;
      more += v.more;
      back += v.back;
    }
    too_long = __reduce_min_sync(0xffffffffu, t.too_long);
    if (back) {  // (the same in all blocks)
      give_back((int)min(n_free0 + before_back, (long long)a.n_pages));
      cluster_sync_all();  // pages that one block gives back another may take
    }
  } else if (back) {
    give_back(n_free0);
    __syncthreads();
  }
  const int top = (int)min(n_free0 + back, (long long)a.n_pages);
  const bool ok = rows <= a.n_tokens && too_long == 0x7fffffff && more <= top;

  // ---- the new pages (those given back are in the list: a barrier lies between)
  if (ok)
    share(s_take, block.more, [&](int i, int j, int x) {
      a.page_table[(size_t)(first + i) * a.max_pages + s_from[i] + j] = __ldcg(a.free_pages + (top - 1 - (int)before_more - x));
    });
  {
    long long row = ok ? before_rows + at.rows : 0;
    for (int i = i0; i < i1; ++i) {
      const int s = first + i, r = __ldca(a.new_len + s), kv = s_kv[i];
      a.q_start[s] = (int)row;
      if (ok) row += max(r, 0);
      a.kv_len[s] = r < 0 ? 0 : ok ? kv + r : kv;
      if (s == a.n_seqs - 1) a.q_start[a.n_seqs] = (int)row;
    }
  }
  if (!kOne) cluster_sync_all();  // nobody leaves while others read its totals
  if (rank == 0 && threadIdx.x == 0) {
    if (a.n_seqs == 0) a.q_start[0] = 0;
    auto short_by = [](long long need, long long have) { return (int)min(max(need - have, 0ll), 0x7fffffffll); };
    a.n_free[0] = ok ? top - (int)more : top;
    a.status[1] = short_by(more, top);
    a.status[2] = short_by(rows, a.n_tokens);
    a.status[3] = too_long == 0x7fffffff ? -1 : too_long;
    a.status[0] = (more > top ? kPlanPages : 0) | (rows > a.n_tokens ? kPlanRows : 0) |
                  (too_long == 0x7fffffff ? 0 : kPlanTable);
  }
  if (kOne && ok && (a.pos || a.slots)) {
    __syncthreads();  // the table's new entries
    for (int r0 = threadIdx.x * kRowsEach; r0 < (int)rows; r0 += kThreads * kRowsEach) {
      int p[kRowsEach], page[kRowsEach], i = holder(s_row, n, r0);
#pragma unroll
      for (int k = 0; k < kRowsEach; ++k) {
        p[k] = page[k] = -1;
        if (r0 + k >= (int)rows) continue;
        while (i + 1 < n && s_row[i + 1] <= r0 + k) ++i;
        p[k] = s_kv[i] + r0 + k - s_row[i];
        if (a.slots) page[k] = __ldcg(a.page_table + (size_t)i * a.max_pages + (p[k] >> a.ps_log2));
      }
      write_rows(a, r0, (int)rows, p, page);
    }
  }
}

// Positions and slots of the rows of a large batch, which the first kernel has planned: a block has kBlockRows of them
// and looks their sequences up in a window of starts and lengths in shared memory, from one probe by all its threads on.
constexpr int kRowThreads = 256, kBlockRows = kRowThreads * kRowsEach;
constexpr int kWindow = kBlockRows + 65536 / kRowThreads + 1;
__global__ void __launch_bounds__(kRowThreads) paged_plan_rows_kernel(const __grid_constant__ PagedPlanArgs a) {
  __shared__ int s_start[kWindow + 1], s_kv[kWindow];
  pdl_wait();
  const int rows = __ldca(a.q_start + a.n_seqs), r0 = blockIdx.x * kBlockRows;
  if (r0 >= rows) return;
  const int step = (a.n_seqs + kRowThreads - 1) / kRowThreads, probe = threadIdx.x * step;
  const int le = __syncthreads_count(probe < a.n_seqs && __ldca(a.q_start + probe) <= r0);
  const int s0 = (le - 1) * step, n = min(kWindow, a.n_seqs - s0);  // (q_start[0] is 0)
  for (int i = threadIdx.x; i <= n; i += kRowThreads) {
    s_start[i] = __ldca(a.q_start + s0 + i);
    if (i < n) s_kv[i] = __ldca(a.kv_len + s0 + i);
  }
  __syncthreads();
  const int t0 = r0 + threadIdx.x * kRowsEach;
  if (t0 >= rows) return;
  int p[kRowsEach], page[kRowsEach], i = holder(s_start, n, t0);
#pragma unroll
  for (int k = 0; k < kRowsEach; ++k) {
    const int r = t0 + k;
    p[k] = page[k] = -1;
    if (r >= rows) continue;
    int s;
    if (r < s_start[n]) {
      while (s_start[i + 1] <= r) ++i;
      s = s0 + i;
      p[k] = s_kv[i] - s_start[i + 1] + r;
    } else {  // behind the window: there are sequences without a token in it
      s = s0 + n;
      for (int hi = a.n_seqs; hi - s > 1;) {
        const int mid = (s + hi) / 2;
        if (__ldca(a.q_start + mid) <= r) s = mid;
        else hi = mid;
      }
      p[k] = __ldca(a.kv_len + s) - __ldca(a.q_start + s + 1) + r;
    }
    if (a.slots) page[k] = __ldca(a.page_table + (size_t)s * a.max_pages + (p[k] >> a.ps_log2));
  }
  write_rows(a, t0, rows, p, page);
}

}  // namespace

cudaError_t paged_plan(const PagedPlanArgs& a, int device, cudaStream_t s) {
  PagedPlanArgs p = a;
  if (a.n_seqs <= kBlockSeqs && a.n_tokens <= kBlockTokens)
    return launch_kernel(reinterpret_cast<const void*>(&paged_plan_kernel<true>), dim3(1), dim3(kThreads), 0, s, true, &p);
  void* params[] = {&p};
  const void* fn = reinterpret_cast<const void*>(&paged_plan_kernel<false>);
  const size_t smem = 4 * (kMostSeqs + 1) * sizeof(int);
  static SmemCap cap;
  cudaError_t e = cap.raise(fn, device, smem);
  if (e != cudaSuccess) return e;
  e = launch_cluster_params(fn, dim3(kCluster), dim3(kThreads), smem, s, kCluster, true, params);
  if (e != cudaSuccess || (!a.pos && !a.slots) || a.n_tokens == 0) return e;
  return launch_kernel(reinterpret_cast<const void*>(&paged_plan_rows_kernel),
                       dim3((a.n_tokens + kBlockRows - 1) / kBlockRows), dim3(kRowThreads), 0, s, true, &p);
}

}  // namespace yb
