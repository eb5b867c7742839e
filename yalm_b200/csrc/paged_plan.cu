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
// Integers only, a few bytes a sequence and 12 a token: launches and chains of dependent loads are what it costs.  One
// block does all of it for up to kBlockSeqs sequences and kBlockTokens rows, the starts in shared memory, where a
// token's sequence is searched.  Larger batches: a cluster of 8 blocks does the sums and the pages, each block a
// stretch of the sequences, with totals exchanged over distributed shared memory; a second kernel over the whole GPU
// writes the tokens' positions and slots.
#include "cluster.cuh"
#include "launch.h"
#include "paged.cuh"

namespace yb {

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr int kBlockSeqs = 1024, kBlockTokens = 8192;

struct Sums {
  long long rows, more, back;  // tokens, pages taken, pages given back
};
__device__ __forceinline__ Sums operator+(const Sums& a, const Sums& b) { return {a.rows + b.rows, a.more + b.more, a.back + b.back}; }

// What a sequence brings: r < 0: it ends.  held: pages in its table before, more: pages that it takes.
struct Wish {
  int n, kv, held, more;
  bool ends, too_long;
};
__device__ __forceinline__ Wish wish(const PagedPlanArgs& a, int s, bool there) {
  Wish w{0, 0, 0, 0, false, false};
  if (!there) return w;
  const int r = __ldca(a.new_len + s), cap = a.max_pages << a.ps_log2, up = (1 << a.ps_log2) - 1;
  w.kv = min(max(__ldca(a.kv_before + s), 0), cap);
  w.held = (w.kv + up) >> a.ps_log2;
  w.ends = r < 0;
  w.n = max(r, 0);
  w.too_long = w.n > cap - w.kv;
  if (!w.too_long) w.more = ((w.kv + w.n + up) >> a.ps_log2) - w.held;
  return w;
}

// The ended sequences' pages from `kept` on, those that are there, in order, by the whole warp.  lane i's sequence is
// seq (ends: it is one); returns how many pages lane i's has, and stores them from free_pages[at] on if `at` >= 0.
__device__ __forceinline__ int give_back(const PagedPlanArgs& a, int seq, const Wish& w, long long at) {
  const int lane = threadIdx.x & 31;
  int mine = 0;
  for (unsigned todo = __ballot_sync(0xffffffffu, w.ends && w.held > 0); todo; todo &= todo - 1) {
    const int src = __ffs(todo) - 1;
    const int s = __shfl_sync(0xffffffffu, seq, src), held = __shfl_sync(0xffffffffu, w.held, src);
    long long to = __shfl_sync(0xffffffffu, at, src);
    const int* row = a.page_table + (size_t)s * a.max_pages;
    int count = 0;
    for (int j = min(max(a.kept ? __ldca(a.kept + s) : 0, 0), held) + lane; __any_sync(0xffffffffu, j < held); j += 32) {
      const int page = j < held ? __ldca(row + j) : -1;
      const bool real = page >= 0 && page < a.n_pages;
      const unsigned which = __ballot_sync(0xffffffffu, real);
      const long long mine_to = to + count + __popc(which & ((1u << lane) - 1));
      if (at >= 0 && real && mine_to < a.n_pages) a.free_pages[mine_to] = page;
      count += __popc(which);
    }
    if (lane == src) mine = count;
  }
  return mine;
}

__device__ __forceinline__ long long shfl_up(long long v, int o) { return __shfl_up_sync(0xffffffffu, v, o); }

template <bool kOne>  // one block and everything in it
__global__ void __launch_bounds__(kThreads, 1) paged_plan_kernel(const __grid_constant__ PagedPlanArgs a) {
  __shared__ Sums s_warp[kWarps];
  __shared__ int s_long[kWarps];
  struct Total {
    Sums sums;
    int too_long;  // the first sequence that is, or INT_MAX
  };
  __shared__ Total s_total;
  __shared__ int s_row[kOne ? kBlockSeqs + 1 : 1], s_kv[kOne ? kBlockSeqs : 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kOne ? 0 : (int)cluster_ctarank(), blocks = kOne ? 1 : kCluster;
  const int per = (a.n_seqs + blocks * kThreads - 1) / (blocks * kThreads);  // sequences of a thread
  const int s0 = (rank * kThreads + threadIdx.x) * per;                      // (below 2^17)
  pdl_wait();
  const int n_free0 = min(max(__ldca(a.n_free_before), 0), a.n_pages);

  Sums mine{0, 0, 0};
  int too_long = 0x7fffffff;
  for (int i = 0; i < per; ++i) {
    const int s = s0 + i;
    const Wish w = wish(a, s, s < a.n_seqs);
    if (w.too_long) too_long = min(too_long, s);
    const int back = give_back(a, s, w, -1);
    mine = mine + Sums{w.n, w.more, back};
  }
  Sums upto = mine;  // inclusive: of the warp's threads to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sums v{shfl_up(upto.rows, o), shfl_up(upto.more, o), shfl_up(upto.back, o)};
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
    const Sums v{shfl_up(sums.rows, o), shfl_up(sums.more, o), shfl_up(sums.back, o)};
    if (lane >= o) sums = sums + v;
  }
  auto from = [&](long long v, int l) { return __shfl_sync(0xffffffffu, v, l); };
  Sums all{from(sums.rows, 31), from(sums.more, 31), from(sums.back, 31)};
  const int before_warp = max(warp - 1, 0);
  Sums at{from(sums.rows, before_warp), from(sums.more, before_warp), from(sums.back, before_warp)};
  if (warp == 0) at = Sums{0, 0, 0};
  at = Sums{at.rows + upto.rows - mine.rows, at.more + upto.more - mine.more, at.back + upto.back - mine.back};
  if (!kOne) {
    if (threadIdx.x == 0) s_total = Total{all, too_long};
    cluster_sync_all();
    all = Sums{0, 0, 0};
    for (int c = 0; c < kCluster; ++c) {
      const Total* t = dsmem_ptr(&s_total, c);
      if (c < rank) at = at + t->sums;
      all = all + t->sums;
      too_long = min(too_long, t->too_long);
    }
    // (the next cluster barrier, which every block passes, comes after all of these loads)
  }
  const int top = (int)min(n_free0 + all.back, (long long)a.n_pages);
  const bool ok = all.rows <= a.n_tokens && too_long == 0x7fffffff && all.more <= top;

  if (all.back) {  // the same in every thread
    long long to = n_free0 + at.back;
    for (int i = 0; i < per; ++i) {
      const int s = s0 + i;
      to += give_back(a, s, wish(a, s, s < a.n_seqs), to);
    }
  }
  // pages that one block gives back another may take
  if (!kOne) cluster_sync_all();
  else __syncthreads();

  int row = ok ? (int)at.rows : 0;
  long long take = top - 1 - at.more;  // the next page's place in the list
  for (int i = 0; i < per; ++i) {
    const int s = s0 + i;
    const bool there = s < a.n_seqs;
    const Wish w = wish(a, s, there);
    const int more = ok ? w.more : 0;
    // a page or two by the lane itself, more by the whole warp
    if (more > 0 && more <= 2) {
      int* to = a.page_table + (size_t)s * a.max_pages + w.held;
      for (int j = 0; j < more; ++j) to[j] = __ldcg(a.free_pages + take - j);
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, more > 2); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1, count = __shfl_sync(0xffffffffu, more, src);
      const long long first = from(take, src);
      int* to = a.page_table + (size_t)__shfl_sync(0xffffffffu, s, src) * a.max_pages + __shfl_sync(0xffffffffu, w.held, src);
      for (int j = lane; j < count; j += 32) to[j] = __ldcg(a.free_pages + first - j);
    }
    take -= more;
    if (there) {
      a.q_start[s] = row;
      if (kOne) {
        s_row[s] = row;
        s_kv[s] = w.kv;
      }
      row += ok ? w.n : 0;
      a.kv_len[s] = w.ends ? 0 : ok ? w.kv + w.n : w.kv;
      if (s == a.n_seqs - 1) a.q_start[a.n_seqs] = row;
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    if (a.n_seqs == 0) a.q_start[0] = 0;
    auto short_by = [](long long need, long long have) { return (int)min(max(need - have, 0ll), 0x7fffffffll); };
    a.n_free[0] = ok ? top - (int)all.more : top;
    a.status[1] = short_by(all.more, top);
    a.status[2] = short_by(all.rows, a.n_tokens);
    a.status[3] = too_long == 0x7fffffff ? -1 : too_long;
    a.status[0] = (all.more > top ? kPlanPages : 0) | (all.rows > a.n_tokens ? kPlanRows : 0) |
                  (too_long == 0x7fffffff ? 0 : kPlanTable);
  }
  if (kOne && ok && (a.pos || a.slots)) {
    __syncthreads();  // the starts, and the table's new entries
    for (int r = threadIdx.x; r < (int)all.rows; r += kThreads) {
      int lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before the row: it has it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (s_row[mid] <= r) lo = mid;
        else hi = mid;
      }
      const int p = s_kv[lo] + r - s_row[lo];
      if (a.pos) a.pos[r] = p;
      if (a.slots) a.slots[r] = paged_slot(a, p, __ldcg(a.page_table + (size_t)lo * a.max_pages + (p >> a.ps_log2)));
    }
  }
}

// Positions and slots of the rows of a large batch, which the first kernel has planned: a thread a row.
constexpr int kRowThreads = 256;
__global__ void __launch_bounds__(kRowThreads) paged_plan_rows_kernel(const __grid_constant__ PagedPlanArgs a) {
  pdl_wait();
  const int r0 = (blockIdx.x * kRowThreads + threadIdx.x) & ~31, r = r0 + (threadIdx.x & 31);
  const int rows = __ldca(a.q_start + a.n_seqs);
  if (r0 >= rows) return;
  PagedBatch b{};
  b.q_start = a.q_start;
  b.n_seqs = a.n_seqs;
  int lo = paged_find_seq(b, r0), hi = paged_find_seq(b, min(r0 + 31, rows - 1)) + 1;
  if (r >= rows) return;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (__ldca(a.q_start + mid) <= r) lo = mid;
    else hi = mid;
  }
  const int p = __ldca(a.kv_len + lo) - __ldca(a.q_start + lo + 1) + r;
  if (a.pos) a.pos[r] = p;
  if (a.slots) a.slots[r] = paged_slot(a, p, __ldca(a.page_table + (size_t)lo * a.max_pages + (p >> a.ps_log2)));
}

}  // namespace

cudaError_t paged_plan(const PagedPlanArgs& a, cudaStream_t s) {
  PagedPlanArgs p = a;
  if (a.n_seqs <= kBlockSeqs && a.n_tokens <= kBlockTokens)
    return launch_kernel(reinterpret_cast<const void*>(&paged_plan_kernel<true>), dim3(1), dim3(kThreads), 0, s, true, &p);
  void* params[] = {&p};
  const cudaError_t e = launch_cluster_params(reinterpret_cast<const void*>(&paged_plan_kernel<false>), dim3(kCluster),
                                              dim3(kThreads), 0, s, kCluster, true, params);
  if (e != cudaSuccess || (!a.pos && !a.slots) || a.n_tokens == 0) return e;
  return launch_kernel(reinterpret_cast<const void*>(&paged_plan_rows_kernel),
                       dim3((a.n_tokens + kRowThreads - 1) / kRowThreads), dim3(kRowThreads), 0, s, true, &p);
}

}  // namespace yb
