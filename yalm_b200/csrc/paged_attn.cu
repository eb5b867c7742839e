// Attention of a batch's new tokens over the paged KV cache on the 5th-generation tensor cores:
//
//   o[token, head] = sum_t 2^(c q.k_t - m) v_t / sum_t 2^(c q.k_t - m),   c = scale * log2(e),
//
// over the slots t that the token sees, in one pass over the keys with a running maximum m and sum.
// Whole prompts, chunks and single tokens take the same path in one launch.
//
// Work.  A unit is (sequence, kv head, block of up to 2 QB queries), QB = 128 / (query heads per kv head):
// its rows are (query, head of the group) pairs, in two row tiles of 128, so every K and V tile that is
// loaded serves all query heads of its group.  A unit's cost is that of its 128-slot key tiles and of its start
// and end.  The units of the whole batch in order make one axis, which the blocks (one per SM) share out
// evenly: a long cache of few rows is cut over many blocks, and ragged lengths balance themselves.
// The cuts follow from the lengths on the device, by a closed form for a sequence's units (floor
// sums), so there is no plan to be made on the host and a captured launch follows new lengths.  A unit
// that is cut leaves (o, m, l) records in the workspace, which a second kernel merges, spread over the whole
// GPU: results do not depend on timing, and no block waits for another.
//
// Block.  Two pipelines of 128 rows share the tensor cores, one's softmax under the other's products:
//   warps 0, 3   load the K tiles and Q (a 3-D box of queries x heads), and the V tiles, into one ring, one lane a
//                page (with pages of 16 slots a tile is 16 copies, which keep one warp busier than the memory)
//   warps 1, 2   issue the products of pipeline 0 / 1, 64 slots a step: S = Q . K^T into tensor memory, then
//                O += P . V with P read from tensor memory, where it took the place of S.  S has two buffers, so
//                the scores of a step are there before the softmax of the step before is done.  (Steps of 128
//                slots leave no room for that: 512 columns hold two outputs and two such S.  A pipeline then
//                waits a third of its time for its scores.  The 64-column scores' products run at 0.67 of the rate
//                of 128-column ones, 388 clocks for eight and not 259, and still win.  2048 tokens over 16384 slots: 504 us
//                with 128 slots a step, 495 with 64; 606 with one warp for both pipelines' products.)
//   warps 4-7, 8-11   softmax of pipeline 0 / 1, a row per thread
// A unit of two row tiles runs them as the pipelines over the same slots.  A unit of one row tile (single
// tokens, short chunks) gives each pipeline half of every key tile, and merges the two at its end.
//
// P is rounded to the caches' type for the tensor cores (the weights' rounding error is that of the
// output's rounding, and averages over the slots); scores, maxima, sums and outputs are fp32.  The output is
// rescaled only when a row's maximum grew by more than 2^8: until then the old maximum serves, and every
// weight stays below 2^8.  O is summed in tensor memory over 1024 additions at most, then joined to the sums before
// (paged_axis.cuh, kSumTiles).  fp16 weights carry a factor 2^7, with which they are normal numbers from 2^-21 of
// that maximum's weight on; smaller ones are rounded by up to 2^-32 of it each.
//
// What bounds it.  Prompts and chunks: the exponentials and the passes over S and P through registers beside the
// products.  2048 tokens over 16384 slots, 32 heads of 128 on 8 kv heads, take 510 us at sustained power (1010
// TFLOP/s; 435 us, 1184 TFLOP/s, before the clock falls), with the tensor and the special-function units each busy 43 %
// of the time in a chunk of 1024.  Single tokens: the cache's bytes, 64 x 4096 slots 171 us = 6.3 TB/s, one of 2^20
// slots 605 us = 7.1 TB/s; one of 32768 slots 32 us = 4.2 TB/s, of which 8 are the launch, the first loads, the last
// tile's softmax and the merge; with heads of 64 a step has half the bytes and the same latencies, 64 x 4096 slots 117 us
// = 4.6 TB/s.
#include "paged.cuh"

#include <cuda_bf16.h>

#include <math.h>
#include <type_traits>

#include "launch.h"
#include "paged_shared.cuh"
#include "tmap.h"
#include "umma.cuh"

namespace yb {

namespace {

constexpr int kST = 64;        // slots per step
constexpr int kRows = 128;     // rows per row tile = tensor-memory lanes
constexpr int kThreads = 384;
constexpr int kMaxGrid = 256;  // blocks the workspace has room for
constexpr uint32_t kBlk = kRows * 128;  // bytes of 128 rows x 64 elements

template <int HD>
struct Cfg {
  static constexpr int kHalves = HD / 64;
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr uint32_t kTile = kHalves * kBlk;  // a row tile of Q, a K tile or a V tile
  static constexpr uint32_t kSmem = (2 + kStages) * kTile + 1024 + 1024;  // + (m, l) of pipeline 1, + alignment
};

// Called by the whole block: this block's share of the axis.
__device__ void find_start(const PagedBatch& b, const Axis& x, unsigned long long* s_warp, Start* s_start) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (b.n_seqs + kThreads - 1) / kThreads;  // sequences of a thread
  const int s0 = min(b.n_seqs, (int)threadIdx.x * per), s1 = min(b.n_seqs, s0 + per);
  unsigned long long mine = 0;
  PagedSeq q{0, 0, 0};
  unsigned per_head = 0;
  for (int s = s0; s < s1; ++s) {
    q = paged_seq(b, s);
    per_head = head_tiles(x, q);
    mine += (unsigned long long)per_head * x.K;
  }
  unsigned long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_warp[warp] = incl;
  if (threadIdx.x == 0) s_start->left = 0;
  __syncthreads();
  // the sums of the warps before this one, and of all, by the lanes of each warp
  unsigned long long sums = lane < kThreads / 32 ? s_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += v;
  }
  const unsigned long long total = __shfl_sync(0xffffffffu, sums, kThreads / 32 - 1);
  const unsigned long long before = __shfl_sync(0xffffffffu, sums, warp) - s_warp[warp] + incl - mine;
  if (!mine) return;
  unsigned long long share;
  int more;
  share_out(total, gridDim.x, share, more);
  const int c = blockIdx.x;
  const unsigned long long begin = block_begin(share, more, c);
  if (begin < before || begin >= before + mine) return;
  const int left = (int)min(share + (c < more ? 1 : 0), total - begin);
  // this thread's sequences hold the block's first position
  unsigned long long rem = begin - before;
  int s = s1 - 1;
  if (per > 1) {
    for (s = s0;; ++s) {
      q = paged_seq(b, s);
      per_head = head_tiles(x, q);
      const unsigned long long all = (unsigned long long)per_head * x.K;
      if (rem < all) break;
      rem -= all;
    }
  }
  Start st;
  st.sq = q;
  st.seq = s;
  st.head = (int)quot(rem, per_head);
  st.unit = 0;
  st.off = (int)(rem - (unsigned long long)st.head * per_head);  // within the head: find_unit
  st.left = left;
  st.begin = begin;
  st.share = share;
  st.more = more;
  *s_start = st;
}

// The same from a plan in the workspace, by one warp.
__device__ void find_start(const SharedBatch& b, const SharedHead* head, const Axis& x, StartOf<SharedSeq>* s_start) {
  const int lane = threadIdx.x & 31, c = blockIdx.x;
  // (the search's first round is on its way beside the head)
  const int step0 = (b.n_seqs + 31) / 32, at0 = (lane + 1) * step0;
  const unsigned long long probe0 = at0 < b.n_seqs ? __ldcg(&b.seqs[at0].begin) : ~0ull;
  const unsigned long long total = __ldcg(&head->total), share = __ldcg(&head->share);
  const int more = __ldcg(&head->more);
  const unsigned long long begin = block_begin(share, more, c);
  if (begin >= total) {
    if (lane == 0) s_start->left = 0;
    return;
  }
  // the last prefix or sequence that begins at or before the block: one that begins there and has no length comes earlier
  int lo = __popc(__ballot_sync(0xffffffffu, probe0 <= begin)) * step0, hi = min(b.n_seqs, lo + step0);
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const bool le = at < hi && __ldcg(&b.seqs[at].begin) <= begin;
    const int n = __popc(__ballot_sync(0xffffffffu, le));
    lo += n * step;
    hi = min(hi, lo + step);
  }
  if (lane) return;
  StartOf<SharedSeq> st;
  st.sq = paged_seq(b, lo);
  st.seq = lo;
  const unsigned long long rem = begin - st.sq.begin;
  const unsigned per_head = head_tiles(x, st.sq);
  st.head = (int)quot(rem, per_head);
  st.unit = 0;
  st.off = (int)(rem - (unsigned long long)st.head * per_head);
  st.left = (int)min(share + (c < more ? 1 : 0), total - begin);
  st.begin = begin;
  st.share = share;
  st.more = more;
  *s_start = st;
}

// Called by a whole warp: the unit in which position st.off of the head lies, and the position within it.  Unit u
// begins at units_before(u); 32 guesses at a time.
template <typename Seq>
__device__ __forceinline__ void find_unit(const Axis& x, StartOf<Seq>& st) {
  int lo = 0, hi = n_units(x, st.sq);  // units_before(lo) <= off < units_before(hi)
  if (hi == 1) return;
  const int lane = threadIdx.x & 31;
  unsigned begin = 0;  // units_before(lo)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
    const unsigned tiles = at < hi ? units_before(x, st.sq, at) : 0xffffffffu;
    const int below = __popc(__ballot_sync(0xffffffffu, tiles <= (unsigned)st.off));
    if (below) begin = __shfl_sync(0xffffffffu, tiles, below - 1);
    lo += below * step;
    hi = min(hi, lo + step);
  }
  st.off -= (int)begin;
  st.unit = lo;
}

// -------------------------------------------------------------------------------------------- numerics
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// bits [lo, hi) of a 32-bit word, lo and hi clipped to [0, 32]
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = min(max(lo, 0), 32);
  hi = min(max(hi, 0), 32);
  if (lo >= hi) return 0u;
  return (0xffffffffu >> (32 - (hi - lo))) << lo;
}

// Workspace: [0] status word; from byte 256 a Cut per block, the unit that the block begins and later blocks
// go on with; then two records per block: 0 for a unit begun by an earlier block, 1 for the one it leaves to
// later ones.  A record holds o as [HD / 4][rows] groups of 4 floats (a warp's rows side by side), then m and
// l, [rows] each.
struct __align__(16) Cut {
  int token;  // first row of the token-major buffers
  int nq;     // queries
  int head;   // kv head
  int parts;  // blocks that hold a record of it, this one first; 0: no unit
};
constexpr size_t kHeadBytes = 256 + kMaxGrid * sizeof(Cut);
template <int HD>
constexpr size_t rec_floats() { return 256 * (size_t)(HD + 2); }

// SM clocks that a wait may take.  Less than the default: without try_wait, which may suspend a warp for longer.
struct Budget {
  long long clocks;
  unsigned nap;
};
inline Budget budget_of(long long clocks) { return {clocks, clocks < kWaitBudgetCycles ? 0u : 1u}; }

}  // namespace

struct PagedAttnParams {
  PagedBatch b;
  Axis x;
  void* out;
  long long out_stride;
  Budget budget, full;  // of the waits, and of those for what is in flight at the end
  float c;              // scale * log2(e)
  int gq;               // query heads per kv head
  int oob;              // a row outside the page pool's tensor maps
  unsigned* status;
  Cut* cuts;
  float* recs;
  // with shared prefixes
  SharedBatch shared;
  const SharedHead* head;
  int n_groups;
  int part_rows;  // rows of a kv head in parts: of the tokens that have both
  float* parts;   // [prefixes, sequences][kv heads], a record of part_rows rows each
  const float* few_recs;   // of sequences of few rows
  const float* few_parts;
};

// Waits for the phase, or until the budget has run out, here or in another warp of the block, which *mark then tells.
// It returns to the same place either way: a warp votes on the mark before it leaves a loop (lanes that left by
// themselves would be waited for without end at the next vote of the others).
__device__ __forceinline__ void bounded_wait(uint64_t* bar, unsigned parity, const Budget& budget, volatile int* mark,
                                             unsigned* status) {
  if (mbar_test_wait(bar, parity)) return;
  const long long t0 = clock64();
  while (!*mark && !(budget.nap ? mbar_try_wait(bar, parity) : mbar_test_wait(bar, parity))) {
    if (clock64() - t0 > budget.clocks) {
      *mark = 1;
      atomicOr(status, kStatusMbarTimeout);
      return;
    }
  }
}

// kShared: the sequences are those of the plan in the workspace, the groups' prefixes among them.  A whole unit whose
// tokens have another part goes to `parts`, as records do: paged_join_kernel puts all parts together.
template <int HD, typename T, bool kShared>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                      const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PagedAttnParams a) {
  using C = Cfg<HD>;
  using Seq = std::conditional_t<kShared, SharedSeq, PagedSeq>;
  constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
  constexpr uint32_t kIdS = kBf16 ? umma_idesc_bf16(kRows, kST, 0, 0) : umma_idesc_f16(kRows, kST, 0, 0);
  constexpr uint32_t kIdO = kBf16 ? umma_idesc_bf16(kRows, HD, 0, 1) : umma_idesc_f16(kRows, HD, 0, 1);
  constexpr float kBias = kBf16 ? 0.f : 7.f;
  constexpr uint32_t kColO = 4 * kST;  // tensor memory: two buffers of S0, of S1, then O0, O1
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t sb = smem_u32(smem), ring = sb + 2 * C::kTile;
  float* s_ml = reinterpret_cast<float*>(smem + (2 + C::kStages) * C::kTile);  // [2][128]
  struct Bars {
    uint64_t one[C::kStages + 2 + 4 + 4 + 8 + 2];  // one arrival a phase: full, q_full, s_full, o_done, turn, idle
    uint64_t two[C::kStages + 2];              // two: empty, q_empty
    uint64_t four[4 + 1];                      // four: p_full, ml_ready
    uint64_t o_free;                           // eight
  };
  __shared__ __align__(8) Bars bars;
  uint64_t* const full = bars.one;
  uint64_t* const q_full = full + C::kStages;
  uint64_t (*const s_full)[2] = reinterpret_cast<uint64_t (*)[2]>(q_full + 2);
  uint64_t (*const o_done)[2] = s_full + 2;
  uint64_t (*const turn)[4] = reinterpret_cast<uint64_t (*)[4]>(o_done + 2);
  uint64_t* const idle = reinterpret_cast<uint64_t*>(turn + 2);
  uint64_t* const empty = bars.two;
  uint64_t* const q_empty = empty + C::kStages;
  uint64_t (*const p_full)[2] = reinterpret_cast<uint64_t (*)[2]>(bars.four);
  uint64_t& ml_ready = bars.four[4];
  uint64_t& o_free = bars.o_free;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_late;  // a wait has run out; one for what is in flight at the end
  __shared__ unsigned s_issued[2][2];  // keys, values: the slots that copies were issued into, and whose count is odd
  __shared__ unsigned long long s_scan[kThreads / 32];
  __shared__ StartOf<Seq> s_start;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedBatch& b = a.b;
  const auto& seqs = [&]() -> const auto& {
    if constexpr (kShared) return a.shared;
    else return a.b;
  }();
  auto table_of = [](const PieceOf<Seq>& c) {  // the piece's row of the page table
    if constexpr (kShared) return c.sq.table;
    else return c.seq;
  };
  auto entry = [](const int* p) { return kShared ? __ldcg(p) : __ldca(p); };
  if constexpr (kShared) {
    if (block_begin(__ldcg(&a.head->share), __ldcg(&a.head->more), blockIdx.x) >= __ldcg(&a.head->total)) {
      pdl_wait();  // nothing to do here: its SM was the other kernel's
      return;
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == 3) {
    constexpr int kOne = sizeof(bars.one) / 8, kTwo = kOne + sizeof(bars.two) / 8, kFour = kTwo + sizeof(bars.four) / 8;
    for (int i = lane; i < (int)sizeof(Bars) / 8; i += 32)
      mbar_init(reinterpret_cast<uint64_t*>(&bars) + i, i < kOne ? 1 : i < kTwo ? 2 : i < kFour ? 4 : 8);
    mbar_fence_init();
    if (lane == 0) {
      s_abort = s_late = 0;
      tma_prefetch_map(&qmap);
      tma_prefetch_map(&kmap);
      tma_prefetch_map(&vmap);
    }
  }
  // up to here nothing of what earlier kernels write was touched
  // With shared prefixes the kernel before is that of few rows, which runs beside this one on other SMs.  It has waited for
  // all that comes before it when it lets this one start; what they wrote is read from L2.  The wait for its own end
  // comes last, so that the join's is for both.
  if constexpr (!kShared) pdl_wait();
  if constexpr (kShared) {
    if (warp == 0) find_start(a.shared, a.head, a.x, &s_start);
  } else {
    find_start(b, a.x, s_scan, &s_start);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  // Once a wait has run out, here or there, no wait of the block lasts: every warp goes on to the end of its piece with
  // whatever lies in its buffers, and leaves.  (A look at the mark in every step cost 3 %.)  Barriers may be arrived at
  // early, but a copy must not be announced to one where another is landing, so the loaders look after each wait.
  // Nobody leaves the block before its copies and products have ended.
  auto wait = [&](uint64_t* bar, unsigned parity) { bounded_wait(bar, parity, a.budget, &s_abort, a.status); };
  auto aborted = [&] { return __any_sync(0xffffffffu, *static_cast<volatile int*>(&s_abort)) != 0; };
  const int QB = kRows / a.gq;
  StartOf<Seq> st0 = s_start;
  if (st0.left > 0) find_unit(a.x, st0);
  WalkOf<Seq> walk(st0);
  PieceOf<Seq> pc;
  if (warp >= 4) {
    // ------------------------------------------------------------------------------- softmax
    const int p = (warp - 4) >> 2, quad = warp & 3;  // pipeline, tensor-memory lane quadrant
    const int r = quad * 32 + lane;                  // row of the row tile
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + lanes + (uint32_t)p * 2 * kST, to = tmem + lanes + kColO;
    const int qi = r / a.gq, h = r % a.gq;
    unsigned steps = 0, singles = 0;  // a pipeline's steps in the pieces before; pieces of one row tile
    if (!kShared && threadIdx.x == 128) a.cuts[blockIdx.x].parts = 0;  // the same thread's later store tells otherwise
    // whether the 16 slots of lane i < 8 in key tile t of a piece are on a page that is there
    auto there = [&](const PieceOf<Seq>& c, int t) {
      const int slot = ((c.u.tile0 + c.t0 + t) << 7) + lane * 16;
      int id = -1;
      if (lane < 8 && slot < c.sq.kv) id = entry(b.page_table + (size_t)table_of(c) * b.max_pages + (slot >> b.ps_log2));
      return id >= 0 && id < b.n_pages;
    };
    bool more = walk.next(seqs, a.x, pc), nx = more && there(pc, 0);  // (a unit without a slot has one empty tile)
    while (more && !aborted()) {
      const bool two = pc.u.nq > QB;
      const int nk = pc.u.none ? 0 : pc.t1 - pc.t0, n = two ? 2 * nk : nk;  // key tiles, steps
      const int tile = two ? p : 0;  // row tile
      const int q = tile * QB + qi;  // query of the unit
      const bool valid = r < QB * a.gq && q < pc.u.nq;
      const bool live = quad * 32 < min(QB, pc.u.nq - tile * QB) * a.gq;  // any row of the warp
      int pos = pc.sq.kv - pc.sq.n + pc.u.q0 + q;
      if constexpr (kShared)
        if (pc.sq.all) pos = pc.sq.kv - 1;
      const int first = pc.u.tile0 + pc.t0;
      // The two warps of a quadrant share a scheduler and its special-function unit: they take their exponentials
      // in turns, one's under the other's loads, maxima and waits.  Left alone they fall into step.
      auto my_turn = [&](unsigned step) {
        if (p || step) wait(&turn[p ^ 1][quad], (p ? step : step - 1) & 1);
      };
      float m = -INFINITY, l = 0.f;
      uint32_t pages = 0;
      for (int i = 0; i < n; ++i) {
        const int t = two ? i >> 1 : i, half = two ? i & 1 : p;
        if (!two || !half) {
          pages = __ballot_sync(0xffffffffu, nx);
          if (t + 1 < nk) nx = there(pc, t + 1);
        }
        const unsigned step = steps + i, buf = step & 1;
        wait(&s_full[p][buf], (step >> 1) & 1);
        tc_fence_after();
        if (live) {
          const int k0 = (first + t) * kKT + half * kST;
          const int lo = valid ? pos - a.x.window + 1 - k0 : kST, hi = valid ? pos + 1 - k0 : 0;
          const uint32_t here = (pages >> (4 * half)) & 0xfu;
          float s[kST];
          tmem_ld64(ts + buf * kST, s);
          // rows behind the unit's last one compute with what lies in their lanes; nothing reads them
          if (!__all_sync(0xffffffffu, !valid || (lo <= 0 && hi >= kST && here == 0xfu))) {
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t pg = ((here >> (2 * w)) & 1u ? 0xffffu : 0u) | ((here >> (2 * w + 1)) & 1u ? 0xffff0000u : 0u);
              const uint32_t msk = bit_range(lo - 32 * w, hi - 32 * w) & pg;
#pragma unroll
              for (int k = 0; k < 32; ++k) s[32 * w + k] = (msk >> k) & 1u ? s[32 * w + k] : -INFINITY;
            }
          }
          float mx;
          {
            float c4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k < kST - 4; k += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) c4[e] = max3(c4[e], s[k + e], s[k + 4 + e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) c4[e] = fmaxf(c4[e], s[kST - 4 + e]);
            mx = fmaxf(max3(c4[0], c4[1], c4[2]), c4[3]) * a.c;
          }
          const bool need = valid && mx > m + 8.0f;  // the first slots seen, or a maximum grown by over 2^8
          float alpha = 1.f;
          if (__any_sync(0xffffffffu, need)) {
            const float mn = need ? mx : m;
            alpha = need ? ex2(m - mn) : 1.f;  // 0 while m is -inf
            m = mn;
            if (i > 0) {
              wait(&o_done[p][buf ^ 1], ((step - 1) >> 1) & 1);
              tc_fence_after();
#pragma unroll 1
              for (int c0 = 0; c0 < HD; c0 += 16) {
                float v[16];
                tmem_ld16(to + p * HD + c0, v);
                uint32_t u[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(v[k] * alpha);
                tmem_st16_u32(to + p * HD + c0, u);
              }
            }
          }
          my_turn(step);
          const float shift = m == -INFINITY ? 0.f : m - kBias;
          const float2 cc = make_float2(a.c, a.c), sh = make_float2(-shift, -shift);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int w = 0; w < kST / 16; ++w) {
            uint32_t pk[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int e = 16 * w + 2 * k;
              float2 t2 = fma2(make_float2(s[e], s[e + 1]), cc, sh);
              t2.x = ex2(t2.x);
              t2.y = ex2(t2.y);
              sum[k & 1] = add2(sum[k & 1], t2);
              pk[k] = pack2<T>(t2.x, t2.y);
            }
            if (w == kST / 16 - 1 && lane == 0) mbar_arrive(&turn[p][quad]);
            tmem_st8_u32(ts + buf * kST + 8 * w, pk);
          }
          l = l * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
          tmem_st_wait();
        } else {
          my_turn(step);
          if (lane == 0) mbar_arrive(&turn[p][quad]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[p][buf]);
      }
      // the piece after this one is looked up under the last product and the stores
      const int left = walk.st.left;
      PieceOf<Seq> after;
      more = walk.next(seqs, a.x, after);
      nx = more && there(after, 0);
      // ---- the piece's rows: o * w0 (+ o of pipeline 1 * w1) (+ o of the pieces before * w2)
      const bool other = !two && nk > 0;  // pipeline 0 takes pipeline 1's rows in
      float w0 = 1.f, w1 = 0.f;
      // (a barrier for each buffer: its phase before the awaited one is over, since the scores that came into the
      // buffer later followed the product of that phase)
      if (n > 0) wait(&o_done[p][(steps + n - 1) & 1], ((steps + n - 1) >> 1) & 1);
      if (other) {
        if (p == 1) {
          s_ml[r] = m;
          s_ml[kRows + r] = l;
          tc_fence_after();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&ml_ready);
            mbar_arrive(&o_free);  // pipeline 0 reads the outputs
          }
        } else {
          wait(&ml_ready, singles & 1);
          const float m1 = s_ml[r], l1 = s_ml[kRows + r], mm = fmaxf(m, m1);
          w0 = m == -INFINITY ? 0.f : ex2(m - mm);
          w1 = m1 == -INFINITY ? 0.f : ex2(m1 - mm);
          l = l * w0 + l1 * w1;
          m = mm;
        }
        ++singles;
      }
      tc_fence_after();
      const bool whole = pc.from == 0 && pc.t1 == pc.u.cost, joins = pc.t0 > pc.from;
      const int rows = pc.u.nq * a.gq, row = tile * QB * a.gq + r;
      const int token = pc.sq.row0 + pc.u.q0;
      float* rec = a.recs + ((size_t)blockIdx.x * 2 + (pc.from == 0 ? 1 : 0)) * rec_floats<HD>();
      // the outputs themselves, or a record: the block's, or with shared prefixes that of the rows in their place
      bool final = whole;
      float* to_rec = rec;
      int to_rows = rows, to_at = row;
      if constexpr (kShared)
        if (whole && pc.sq.part >= 0) {
          final = false;
          to_rows = a.part_rows;
          to_at = (pc.sq.part + pc.u.q0) * a.gq + row;
          to_rec = a.parts + (size_t)((pc.sq.all ? 0 : a.x.K) + pc.head) * (HD + 2) * a.part_rows;
        }
      T* out = static_cast<T*>(a.out) + (size_t)(token + q) * a.out_stride + (size_t)(pc.head * a.gq + h) * HD;
      if (two || p == 0) {
        float w2 = 0.f;
        if (joins && valid) {  // the thread's own record
          const float mm = fmaxf(m, rec[HD * rows + row]);
          w2 = rec[HD * rows + row] == -INFINITY ? 0.f : ex2(rec[HD * rows + row] - mm);
          const float f = m == -INFINITY ? 0.f : ex2(m - mm);
          w0 *= f;
          w1 *= f;
          l = l * f + rec[(HD + 1) * rows + row] * w2;
          m = mm;
        }
        const float inv = final ? (l != 0.f ? 1.f / l : 0.f) : 1.f;
        w0 *= inv;
        w1 *= inv;
        w2 *= inv;
        if (live && two && final && !joins && nk > 0) {
          // Whole outputs of many rows: of 32 columns a lane holds its row's four groups of 16 bytes.  Two lanes exchange
          // two of theirs, so that a store writes whole sectors of 32 bytes of every second row.
          const bool up = lane & 1;
          T* to_row[2];
          bool has[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int from = (lane & ~1) + k;
            to_row[k] = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), from)) + 8 * (lane & 1);
            has[k] = __shfl_sync(0xffffffffu, (int)valid, from);
          }
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 32) {
            float v[32];
            tmem_ld32(to + p * HD + c0, v);
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              uint32_t w[2][4];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float2 t2 = mul2(make_float2(v[8 * k + 2 * e], v[8 * k + 2 * e + 1]), make_float2(w0, w0));
                w[e / 4][e % 4] = pack2<T>(t2.x, t2.y);
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? w[0][e] : w[1][e], 1);
                if (up) w[0][e] = got; else w[1][e] = got;
              }
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if (has[x]) *reinterpret_cast<uint4*>(to_row[x] + c0 + 8 * k) = make_uint4(w[x][0], w[x][1], w[x][2], w[x][3]);
            }
          }
        } else if (live) {
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += 32) {
            float v[32];
            if (nk > 0) {
              tmem_ld32(to + p * HD + c0, v);
              if (other || final || joins) {  // a row that has seen no slot has zeros there: its weights were all 0
                const float2 w00 = make_float2(w0, w0);
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                  const float2 t2 = mul2(make_float2(v[k], v[k + 1]), w00);
                  v[k] = t2.x, v[k + 1] = t2.y;
                }
              }
              if (other) {
                const float2 w11 = make_float2(w1, w1);
                float v1[32];
                tmem_ld32(to + HD + c0, v1);
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                  const float2 t2 = fma2(make_float2(v1[k], v1[k + 1]), w11, make_float2(v[k], v[k + 1]));
                  v[k] = t2.x, v[k + 1] = t2.y;
                }
              }
            } else {
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] = 0.f;
            }
            if (!valid) continue;
            if (joins) {
              const float4* o = reinterpret_cast<const float4*>(rec) + (size_t)(c0 / 4) * rows + row;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float4 f = o[(size_t)k * rows];
                v[4 * k] = fmaf(f.x, w2, v[4 * k]);
                v[4 * k + 1] = fmaf(f.y, w2, v[4 * k + 1]);
                v[4 * k + 2] = fmaf(f.z, w2, v[4 * k + 2]);
                v[4 * k + 3] = fmaf(f.w, w2, v[4 * k + 3]);
              }
            }
            if (final) {
#pragma unroll
              for (int k = 0; k < 4; ++k)
                reinterpret_cast<uint4*>(out + c0)[k] =
                    make_uint4(pack2<T>(v[8 * k], v[8 * k + 1]), pack2<T>(v[8 * k + 2], v[8 * k + 3]),
                               pack2<T>(v[8 * k + 4], v[8 * k + 5]), pack2<T>(v[8 * k + 6], v[8 * k + 7]));
            } else {
              float4* o = reinterpret_cast<float4*>(to_rec + record_sum(to_rows, to_at, c0 / 4));
#pragma unroll
              for (int k = 0; k < 8; ++k) o[(size_t)k * to_rows] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
            }
          }
        }
        if (!final && valid) {
          to_rec[record_m(HD, to_rows, to_at)] = m;
          to_rec[record_l(HD, to_rows, to_at)] = l;
        }
        tc_fence_before();
        __syncwarp();
        if (nk > 0 && lane == 0) mbar_arrive(&o_free);
      }
      if (!kShared && !whole && pc.last && pc.from == 0 && threadIdx.x == 128) {
        const unsigned long long begin = s_start.begin + (s_start.left - left) - pc.t1;  // the unit's first tile
        const int last = block_of(s_start.share, s_start.more, begin + pc.u.cost - 1);
        a.cuts[blockIdx.x] = Cut{token, pc.u.nq, pc.head, last - (int)blockIdx.x + 1};
      }
      steps += n;
      pc = after;
    }
    tmem_st_wait();
  } else {
  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------------------------- loads
    const bool keys = warp == 0;
    const int lg = b.ps_log2, ps = 1 << lg;
    const int boxes = ps >= kKT ? 1 : kKT >> lg;  // pages per key tile
    const uint32_t box_bytes = (uint32_t)min(ps, kKT) * 128u;
    unsigned slot = 0, phase = 1, issued = 0, uses[2] = {0, 0};
    unsigned mine_into = 0, mine_odd = 0;  // the slots that this warp's copies went into, and whose count is odd
    int buf = 0;  // buffer of the next unit of one row tile
    bool ok = true;
    while (ok && walk.next(seqs, a.x, pc)) {
      if (pc.u.none) continue;
      const bool two = pc.u.nq > QB;
      const int* table = b.page_table + (size_t)table_of(pc) * b.max_pages;
      // this lane's page of a key tile, and the row of the page pool where it starts (outside the pool: zeros)
      auto page_of = [&](int tile) {
        const int at = (tile << 7) + (lane << lg);
        return lane < boxes && at < pc.sq.kv ? entry(table + (at >> lg)) : -1;
      };
      auto row_of = [&](int tile, int page) {
        if (page < 0 || page >= b.n_pages) return a.oob;
        return ((page * a.x.K + pc.head) << lg) + (((tile << 7) + (lane << lg)) & (ps - 1));
      };
      auto load = [&](const CUtensorMap* map, int row, bool mine) {
        if (mine) {
          if (issued >= C::kStages) {
            wait(&empty[slot], phase);
            if (aborted()) return false;
          }
          mine_into |= 1u << slot;
          mine_odd ^= 1u << slot;
          if (lane == 0) mbar_arrive_expect_tx(&full[slot], C::kTile);
          __syncwarp();
          if (lane < boxes)
            for (int h = 0; h < C::kHalves; ++h)
              tma_load_2d_s(ring + slot * C::kTile + h * kBlk + lane * box_bytes, map, 64 * h, row, smem_u32(&full[slot]));
        }
        ++issued;
        if (++slot == C::kStages) slot = 0, phase ^= 1;
        return true;
      };
      // a row tile of queries, once the products of the unit before have read its buffer
      auto load_q = [&](int to, int tile) {
        if (uses[to]) {
          wait(&q_empty[to], (uses[to] - 1) & 1);
          if (aborted()) return false;
        }
        ++uses[to];
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[to], (uint32_t)(QB * a.gq) * 128u * C::kHalves);
          for (int h = 0; h < C::kHalves; ++h)
            tma_load_3d_s(sb + to * C::kTile + h * kBlk, &qmap, 64 * h, pc.head * a.gq, pc.sq.row0 + pc.u.q0 + tile * QB,
                          smem_u32(&q_full[to]));
        }
        return true;
      };
      // in the order of the products, whose scores are two steps ahead of the weights: one key tile with two row
      // tiles, two with one
      const int first = pc.u.tile0 + pc.t0, n = pc.t1 - pc.t0, ahead = two ? 1 : 2;
      // the table is read a tile ahead: an entry is a trip to L2
      const int lag = keys ? 0 : ahead;
      int next = page_of(first);
      for (int j = 0; j < n + ahead && ok; ++j) {
        int row = a.oob;
        if (j >= lag && j < n + lag) {
          row = row_of(first + j - lag, next);
          if (j + 1 < n + lag) next = page_of(first + j + 1 - lag);
        }
        if (j >= ahead) ok = load(&vmap, row, !keys);
        if (ok && j < n) ok = load(&kmap, row, keys);
        if (ok && keys && j == 0) {
          if (two) {
            ok = load_q(0, 0) && load_q(1, 1);
          } else {
            ok = load_q(buf, 0);
            buf ^= 1;
          }
        }
      }
    }
    // never leave while a copy may still be landing: the last one into each slot, whichever of the two warps issued it
    // (they may have stopped at different tiles), and into each query buffer
    if (lane == 0) {
      s_issued[keys ? 0 : 1][0] = mine_into;
      s_issued[keys ? 0 : 1][1] = mine_odd;
    }
    asm volatile("bar.sync 1, 64;" ::: "memory");
    if (keys) {
      const unsigned into = s_issued[0][0] | s_issued[1][0], odd = s_issued[0][1] ^ s_issued[1][1];
      for (int i = 0; i < C::kStages; ++i)
        if ((into >> i) & 1u) bounded_wait(&full[i], ((odd >> i) & 1u) ^ 1u, a.full, &s_late, a.status);
      for (int t = 0; t < 2; ++t)
        if (uses[t]) bounded_wait(&q_full[t], (uses[t] - 1) & 1, a.full, &s_late, a.status);
    }
  } else if (warp < 3) {
    // ------------------------------------------------------------------------------- products
    const int p = warp - 1;
    const uint32_t ts = tmem + (uint32_t)p * 2 * kST, to = tmem + kColO + (uint32_t)p * HD;
    unsigned slot = 0, phase = 0, pieces = 0, steps = 0, uses[2] = {0, 0};
    int buf = 0;
    const uint32_t e = elect_lane();
    bool any = false;
    while (!aborted() && walk.next(seqs, a.x, pc)) {
      if (pc.u.none) continue;
      const bool two = pc.u.nq > QB;
      const int first = pc.u.tile0 + pc.t0, nk = pc.t1 - pc.t0, n = two ? 2 * nk : nk;
      const int qb = query_buffer(two, p, buf);
      // each pipeline's warp keeps count of both buffers, whichever it reads.  (One that it did not wait for is full by then: the
      // pipelines' softmaxes take turns, so this one has ended the unit before only after the other's products read it.)
      for (int t = two ? 0 : buf; t <= (two ? 1 : buf); ++t) {
        if (t == qb) wait(&q_full[t], uses[t] & 1);
        ++uses[t];
      }
      unsigned kslot = 0, vslot = 0;
      auto take = [&](unsigned& at) {
        at = slot;
        wait(&full[slot], phase);
        if (++slot == C::kStages) slot = 0, phase ^= 1;
      };
      // a key tile serves two steps of a unit of two row tiles, else one, on this pipeline's half
      auto begins = [&](int i) { return !two || !(i & 1); };
      auto ends = [&](int i) { return !two || (i & 1); };
      auto half_of = [&](int i) { return (uint32_t)(two ? i & 1 : p) * (kST * 128u); };  // bytes into the blocks
      auto take_k = [&](int i) {
        if (begins(i)) take(kslot);
      };
      auto take_v = [&](int i) {
        if (!begins(i)) return;
        take(vslot);
        // Slots before the first token's window, and behind the sequence's last one in its last page, may hold
        // anything: their weight is 0, and 0 * v has to be 0 (both warps write the same zeros).
        const int k0 = (first + (two ? i >> 1 : i)) * kKT;
        const uint32_t v = ring + vslot * C::kTile;
        auto zero = [&](int from, int to) {
          if (from >= to) return;
          for (int x = lane; x < (to - from) * 8 * C::kHalves; x += 32) {
            const int h = x / ((to - from) * 8), r = x % ((to - from) * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + h * kBlk + (from * 8 + r) * 16u), "r"(0u)
                         : "memory");
          }
          fence_proxy_async_smem();
          __syncwarp();
        };
        const int rem = pc.sq.kv - k0, seen = pc.sq.kv - pc.sq.n + pc.u.q0 - a.x.window + 1 - k0;
        if (rem < kKT) zero(rem, min(kKT, ((rem + (1 << b.ps_log2) - 1) >> b.ps_log2) << b.ps_log2));
        if (seen > 0) zero(0, seen);
      };
      const uint64_t dq = umma_desc_k_sw128(sb + qb * C::kTile);
      auto qk = [&](int i) {
        any = true;
        const unsigned u = (steps + i) & 1;
        const uint64_t dk = umma_desc_k_sw128(ring + kslot * C::kTile + half_of(i));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
          const uint32_t off = ((kk / 4) * kBlk + (kk % 4) * 32u) >> 4;
          umma_f16_if(e, ts + u * kST, dq + off, dk + off, kIdS, kk ? 1u : 0u);
        }
        umma_commit_if(e, &s_full[p][u]);
        if (ends(i)) umma_commit_if(e, &empty[kslot]);
        if (i == n - 1) {
          umma_commit_if(e, &q_empty[qb]);
          if (query_releases(two) == 2) umma_commit_if(e, &q_empty[qb]);
        }
      };
      // a buffer of S is free again once the product that reads P from it is issued: they execute in order
      for (int i = 0; i < min(n, 2); ++i) {
        take_k(i);
        tc_fence_after();
        qk(i);
      }
      for (int i = 0; i < n; ++i) {
        const unsigned step = steps + i, u = step & 1;
        take_v(i);
        if (i + 2 < n) take_k(i + 2);
        if (i == 0 && pieces) wait(&o_free, (pieces - 1) & 1);
        const uint64_t dv = umma_desc_sw128(ring + vslot * C::kTile + half_of(i), kBlk, 1024);
        wait(&p_full[p][u], (step >> 1) & 1);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kST / 16; ++kk)
          umma_f16_ta_if(e, to, ts + u * kST + kk * 8, dv + ((kk * 2048u) >> 4), kIdO, (i || kk) ? 1u : 0u);
        umma_commit_if(e, &o_done[p][u]);
        if (ends(i)) umma_commit_if(e, &empty[vslot]);
        if (i + 2 < n) qk(i + 2);
      }
      steps += n;
      ++pieces;
      if (!two) buf ^= 1;
    }
    if (any) {  // nor while a product may still be reading
      umma_commit_if(e, &idle[p]);
      bounded_wait(&idle[p], 0, a.full, &s_late, a.status);
    }
  }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if constexpr (kShared) pdl_wait();
}

// The units that were cut: out = sum_parts 2^(m - M) o / sum_parts 2^(m - M) l.  Blocks x look after the unit that
// attention block x began; 8 elements of a row are a thread's for up to 4 parts (a prompt's unit over two or
// three blocks, 4096 such groups), else the work of 8 lanes that share out the parts and join them by
// shuffles (a single token's unit over 18 blocks, 64 groups), so that every load is under way at once.  The
// order of the sum depends on the number of parts alone.  24 slices of a unit's groups: chunk 512 42.0 us, 42.5 with 16,
// 42.6 with 32.
constexpr int kMergeThreads = 128, kMergeSlices = 24, kMergeParts = 4;
template <int HD, typename T>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const __grid_constant__ PagedAttnParams a) {
  pdl_wait();
  const int4 d = __ldcg(reinterpret_cast<const int4*>(a.cuts + blockIdx.x));  // token, nq, head, parts
  const int rows = d.y * a.gq, lanes = d.w > kMergeParts ? 8 : 1;
  const int lane = threadIdx.x & 31, items = d.w ? rows * (HD / 8) * lanes : 0;
  for (int w0 = blockIdx.y * kMergeThreads + (threadIdx.x & ~31); w0 < items; w0 += kMergeSlices * kMergeThreads) {
    const int item = min(w0 + lane, items - 1), e = item / lanes, sub = item % lanes;
    const int row = e % rows, c8 = e / rows;
    float mm = -INFINITY, ll = 0.f, acc[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k] = 0.f;
    auto join = [&](float m, float l, const float (&v)[8]) {
      const float mn = fmaxf(mm, m);
      const float old = mm == -INFINITY ? 0.f : ex2(mm - mn), w = m == -INFINITY ? 0.f : ex2(m - mn);
      mm = mn;
      ll = ll * old + l * w;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] = acc[j] * old + v[j] * w;
    };
    for (int k0 = sub; k0 < d.w; k0 += kMergeParts * lanes) {
      float m[kMergeParts], l[kMergeParts];
      float4 o[kMergeParts][2];
#pragma unroll
      for (int k = 0; k < kMergeParts; ++k) {
        m[k] = -INFINITY;
        l[k] = 0.f;
        o[k][0] = o[k][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        const int part = k0 + k * lanes;
        if (part < d.w) {
          const float* rec = a.recs + ((size_t)(blockIdx.x + part) * 2 + (part == 0 ? 1 : 0)) * rec_floats<HD>();
          const float4* ro = reinterpret_cast<const float4*>(rec) + (size_t)(2 * c8) * rows + row;
          o[k][0] = __ldcg(ro);
          o[k][1] = __ldcg(ro + rows);
          m[k] = __ldcg(rec + HD * rows + row);
          l[k] = __ldcg(rec + (HD + 1) * rows + row);
        }
      }
#pragma unroll
      for (int k = 0; k < kMergeParts; ++k) {
        const float v[8] = {o[k][0].x, o[k][0].y, o[k][0].z, o[k][0].w, o[k][1].x, o[k][1].y, o[k][1].z, o[k][1].w};
        join(m[k], l[k], v);
      }
    }
    for (int x = 1; x < lanes; x <<= 1) {
      float v[8];
      const float m = __shfl_xor_sync(0xffffffffu, mm, x), l = __shfl_xor_sync(0xffffffffu, ll, x);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = __shfl_xor_sync(0xffffffffu, acc[k], x);
      join(m, l, v);
    }
    if (sub || w0 + lane >= items) continue;
    const float inv = ll != 0.f ? 1.f / ll : 0.f;
    T* out = static_cast<T*>(a.out) + (size_t)(d.x + row / a.gq) * a.out_stride + (size_t)(d.z * a.gq + row % a.gq) * HD + 8 * c8;
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv),
                                                pack2<T>(acc[4] * inv, acc[5] * inv), pack2<T>(acc[6] * inv, acc[7] * inv));
  }
}

// Shared prefixes: out = sum_parts 2^(m - M) o / sum_parts 2^(m - M) l over all parts of a row, those of its own slots and
// those of its group's prefix, each a record in `parts` or, of a unit that was cut, several of the blocks' or warps'.
// Blocks (x, y) look after sequence x, a warp after up to 8 rows of a kv head: where their parts lie is found once for
// them.  A row has 32 / rows lanes, which take turns at its float4, so that records of either kind are read by pieces of
// 64 bytes and more, up to 8 parts at once.  (A warp a row, with the parts shared out among its lanes, took 945
// instructions a row, mostly for that search: 64 single tokens 8.6 us.)
constexpr int kJoinThreads = 128, kJoinRows = 8, kJoinParts = 8;
template <int HD, typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttnParams a) {
  constexpr int kF = HD / 4;  // float4 of a row
  constexpr int kN = 4;       // of a lane at once
  pdl_wait();
  const PagedBatch& b = a.b;
  const SharedSeq own = paged_seq(a.shared, a.n_groups + blockIdx.x);
  const unsigned long long share = __ldcg(&a.head->share), few_share = __ldcg(&a.head->few_share);
  const int more = __ldcg(&a.head->more), few_more = __ldcg(&a.head->few_more);
  SharedSeq prefix{};
  if (own.part >= 0) prefix = paged_seq(a.shared, own.group);
  const int lane = threadIdx.x & 31;
  const int tokens = max(own.n, own.few), rows = tokens * a.gq;  // of a kv head
  const unsigned few_head = few_length(own), own_head = head_tiles(a.x, own), prefix_head = head_tiles(a.x, prefix);
  if (!tokens) return;
  const int groups = (rows + kJoinRows - 1) / kJoinRows, items = groups * a.x.K;
  // lanes of a row: a power of two
  const int log_rows = rows > 4 ? 3 : rows > 2 ? 2 : rows - 1, lanes = 32 >> log_rows;
  const int c = lane & (lanes - 1);
  // Where a unit's parts lie: n records, the first one apart; a row's float4 k is at k * step float4.
  struct Parts {
    int n;
    const float *first, *rest;  // rest: the second one's
    size_t next;                // floats from that to the one after it
    RecordRow row;
  };
  // of the tensor-core kernel
  auto of_unit = [&](const SharedSeq& q, unsigned per_head, int head, int token, int h) {
    const int at = own.row0 + token - q.row0, unit = at / a.x.U;
    const Unit u = unit_of(a.x, q, unit);
    const unsigned long long begin = q.begin + (unsigned long long)per_head * head + units_before(a.x, q, unit);
    const int block = block_of(share, more, begin);
    Parts p;
    p.n = block_of(share, more, begin + u.cost - 1) - block + 1;
    const bool whole = p.n == 1;
    const int rs = whole ? a.part_rows : u.nq * a.gq, r = whole ? (q.part + at) * a.gq + h : (at - u.q0) * a.gq + h;
    p.first = (whole ? a.parts + (size_t)((q.all ? 0 : a.x.K) + head) * (HD + 2) * rs
                     : a.recs + ((size_t)block * 2 + 1) * rec_floats<HD>()) + record_sum(rs, r, 0);
    p.rest = a.recs + (size_t)(block + 1) * 2 * rec_floats<HD>() + record_sum(rs, r, 0);
    p.next = 2 * rec_floats<HD>();
    p.row = record_row(HD, rs, r);
    return p;
  };
  // of the kernel of few rows
  auto of_few = [&](int head, int token, int h) {
    const unsigned long long begin = own.few_begin + (unsigned long long)few_head * head;
    const int warp = block_of(few_share, few_more, begin);
    Parts p;
    p.n = block_of(few_share, few_more, begin + few_steps(own) - 1) - warp + 1;
    const size_t row = (size_t)(token * a.gq + h) * few_row_floats(HD), rec = kFewRows * few_row_floats(HD);
    p.first = p.n == 1 ? a.few_parts + ((size_t)(own.part + token) * b.n_heads + head * a.gq + h) * few_row_floats(HD)
                       : a.few_recs + ((size_t)warp * 2 + 1) * rec + row;
    p.rest = a.few_recs + (size_t)(warp + 1) * 2 * rec + row;
    p.next = 2 * rec;
    p.row = RecordRow{1, HD};
    return p;
  };
  const int warps = gridDim.y * (kJoinThreads / 32);
  for (int item = blockIdx.y * (kJoinThreads / 32) + (threadIdx.x >> 5); item < items; item += warps) {
    const int head = item / groups, row = (item - head * groups) * kJoinRows + lane / lanes;
    if (row >= rows) continue;
    const int token = row / a.gq, h = row - token * a.gq;
    const Parts one = own.few ? of_few(head, token, h) : of_unit(own, own_head, head, token, h);
    if (one.n == 1 && own.part < 0) continue;  // the outputs are in their place
    Parts two = one;
    two.n = 0;
    if (own.part >= 0) two = of_unit(prefix, prefix_head, head, token, h);
    const int n = one.n + two.n;
    T* out = static_cast<T*>(a.out) + (size_t)(own.row0 + token) * a.out_stride + (size_t)(head * a.gq + h) * HD;
    for (int f0 = c; f0 < kF; f0 += kN * lanes) {
      float mm = -INFINITY, ll = 0.f;
      float4 acc[kN];
#pragma unroll
      for (int k = 0; k < kN; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int p0 = 0; p0 < n; p0 += kJoinParts) {
        float4 o[kJoinParts][kN];
        float m[kJoinParts], l[kJoinParts];
#pragma unroll
        for (int e = 0; e < kJoinParts; ++e) {
          m[e] = -INFINITY;
          l[e] = 0.f;
#pragma unroll
          for (int k = 0; k < kN; ++k) o[e][k] = make_float4(0.f, 0.f, 0.f, 0.f);
          const int i = p0 + e;
          if (i >= n) continue;
          const bool second = i >= one.n;
          const int part = second ? i - one.n : i, step = second ? two.row.step : one.row.step;
          const long long m_at = second ? two.row.m : one.row.m;
          const float* rec = part ? (second ? two.rest : one.rest) + (part - 1) * (second ? two.next : one.next)
                                  : second ? two.first : one.first;
#pragma unroll
          for (int k = 0; k < kN; ++k)
            if (f0 + k * lanes < kF) o[e][k] = __ldcg(reinterpret_cast<const float4*>(rec) + (size_t)(f0 + k * lanes) * step);
          m[e] = __ldcg(rec + m_at);
          l[e] = __ldcg(rec + m_at + step);
        }
        float mn = mm;
#pragma unroll
        for (int e = 0; e < kJoinParts; ++e) mn = fmaxf(mn, m[e]);
        const float old = mm == -INFINITY ? 0.f : ex2(mm - mn);
        mm = mn;
        ll *= old;
#pragma unroll
        for (int k = 0; k < kN; ++k) acc[k] = make_float4(acc[k].x * old, acc[k].y * old, acc[k].z * old, acc[k].w * old);
#pragma unroll
        for (int e = 0; e < kJoinParts; ++e) {
          const float w = m[e] == -INFINITY ? 0.f : ex2(m[e] - mn);
          ll = fmaf(l[e], w, ll);
#pragma unroll
          for (int k = 0; k < kN; ++k) {
            acc[k].x = fmaf(o[e][k].x, w, acc[k].x);
            acc[k].y = fmaf(o[e][k].y, w, acc[k].y);
            acc[k].z = fmaf(o[e][k].z, w, acc[k].z);
            acc[k].w = fmaf(o[e][k].w, w, acc[k].w);
          }
        }
      }
      const float inv = ll != 0.f ? 1.f / ll : 0.f;
#pragma unroll
      for (int k = 0; k < kN; ++k)
        if (f0 + k * lanes < kF)
          *reinterpret_cast<uint2*>(out + 4 * (f0 + k * lanes)) =
              make_uint2(pack2<T>(acc[k].x * inv, acc[k].y * inv), pack2<T>(acc[k].z * inv, acc[k].w * inv));
    }
  }
}

int paged_attention_grid(int n_sms) { return n_sms < kMaxGrid ? n_sms : kMaxGrid; }

size_t paged_attention_scratch(int head_dim, int n_sms) {
  const int grid = paged_attention_grid(n_sms);
  return kHeadBytes + (size_t)grid * 2 * (head_dim == 128 ? rec_floats<128>() : rec_floats<64>()) * 4;
}

// Rows (queries x query heads of a kv head) of the tokens that have a part in `parts`: of all, or of the most that groups
// computed once may have, which is a unit's for every sequence (paged_shared.cu).
static int part_tokens(const PagedBatch& b) {
  const long long most = (long long)b.n_seqs * 2 * (kRows / (b.n_heads / b.n_kv_heads));
  return (int)(b.n_tokens < most ? b.n_tokens : most);
}
static long long part_rows(const PagedBatch& b) { return ((long long)part_tokens(b) * (b.n_heads / b.n_kv_heads) + 3) / 4 * 4; }
// Its workspace: that of a call without prefixes, the plan, the parts.
static size_t shared_plan_at(int head_dim, int n_sms) { return (paged_attention_scratch(head_dim, n_sms) + 255) / 256 * 256; }
static size_t shared_parts_at(const PagedBatch& b, int n_groups, int head_dim, int n_sms) {
  return shared_plan_at(head_dim, n_sms) + 256 + ((size_t)n_groups + b.n_seqs) * sizeof(SharedSeq);
}
static size_t few_parts_at(const PagedBatch& b, int n_groups, int head_dim, int n_sms) {
  return shared_parts_at(b, n_groups, head_dim, n_sms) + (size_t)2 * b.n_kv_heads * (head_dim + 2) * part_rows(b) * 4;
}
static size_t few_recs_at(const PagedBatch& b, int n_groups, int head_dim, int n_sms) {
  return few_parts_at(b, n_groups, head_dim, n_sms) + (size_t)part_tokens(b) * b.n_heads * few_row_floats(head_dim) * 4;
}
size_t paged_shared_scratch(const PagedBatch& b, int n_groups, int head_dim, int n_sms) {
  return few_recs_at(b, n_groups, head_dim, n_sms) +
         (size_t)paged_attention_grid(n_sms) * kFewWarps * 2 * kFewRows * few_row_floats(head_dim) * 4;
}

namespace {
template <int HD, typename T, bool kShared>
cudaError_t launch(const PagedAttnArgs& a, int device, int grid, bool bf16, cudaStream_t s) {
  const int K = a.b.n_kv_heads, ps = 1 << a.b.ps_log2, gq = a.b.n_heads / K, qb = kRows / gq;
  const long long rows = (long long)a.b.n_pages * K * ps;
  CUtensorMap qm, km, vm;
  const int box = ps < kKT ? ps : kKT;
  if (!tmap_16_3d_sw128(&qm, a.q, bf16, {HD, a.b.n_heads, a.b.n_tokens}, {HD, a.q_stride}, {64, gq, qb}) ||
      !tmap_f16_2d_sw128(&km, static_cast<const __half*>(a.k_pages), rows, HD, 64, box) ||
      !tmap_f16_2d_sw128(&vm, static_cast<const __half*>(a.v_pages), rows, HD, 64, box))
    return cudaErrorInvalidValue;
  PagedAttnParams p{};
  p.b = a.b;
  p.x = Axis{2 * qb, a.window < (1 << 22) ? a.window : 1 << 22, K};
  p.out = a.out;
  p.out_stride = a.out_stride;
  p.budget = budget_of(a.wait_budget);
  p.full = budget_of(kWaitBudgetCycles);
  p.c = a.scale * 1.4426950408889634f;
  p.gq = gq;
  p.oob = (int)rows;
  p.status = static_cast<unsigned*>(a.scratch);
  p.cuts = reinterpret_cast<Cut*>(static_cast<char*>(a.scratch) + 256);
  p.recs = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kHeadBytes);
  const void* fn = reinterpret_cast<const void*>(&paged_attn_kernel<HD, T, kShared>);
  static SmemCap cap;
  cudaError_t e = cap.raise(fn, device, Cfg<HD>::kSmem);
  if (e != cudaSuccess) return e;
  if constexpr (kShared) {
    char* const base = static_cast<char*>(a.scratch);
    const size_t plan = shared_plan_at(HD, a.n_sms);
    SharedPlanArgs sp{a.b, a.group_start, a.prefix_len, a.n_groups, HD, p.x, grid, part_tokens(a.b), reinterpret_cast<SharedHead*>(base + plan),
                      reinterpret_cast<SharedSeq*>(base + plan + 256)};
    p.shared = SharedBatch{sp.seqs, a.n_groups + a.b.n_seqs};
    p.head = sp.head;
    p.n_groups = a.n_groups;
    p.part_rows = (int)part_rows(a.b);
    p.parts = reinterpret_cast<float*>(base + shared_parts_at(a.b, a.n_groups, HD, a.n_sms));
    p.few_parts = reinterpret_cast<float*>(base + few_parts_at(a.b, a.n_groups, HD, a.n_sms));
    p.few_recs = reinterpret_cast<float*>(base + few_recs_at(a.b, a.n_groups, HD, a.n_sms));
    if ((e = paged_shared_plan(sp, s)) != cudaSuccess) return e;
    const PagedFewArgs f{a.b, p.shared, p.head, a.q, a.out, a.k_pages, a.v_pages, a.q_stride, a.out_stride, K, gq, p.c,
                         const_cast<float*>(p.few_recs), const_cast<float*>(p.few_parts), p.status, a.wait_budget};
    if ((e = paged_few(f, HD, bf16 ? 2 : 1, device, grid, s)) != cudaSuccess) return e;
  }
  void* args[] = {&qm, &km, &vm, &p};
  // both kernels set up under the end of the one before (programmatic launch): 37.0 -> 33.1 us for one token over
  // 32767 slots, 47.8 -> 43.9 us for the chunk of 512
  if ((e = launch_kernel_params(fn, dim3(grid), dim3(kThreads), Cfg<HD>::kSmem, s, true, args)) != cudaSuccess) return e;
  if constexpr (kShared) {
    // enough warps for all rows if they are spread evenly over the sequences
    const long long items = (((long long)a.b.n_tokens * gq / a.b.n_seqs + kJoinRows - 1) / kJoinRows + 1) * K;
    const long long slices = (items + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
    return launch_kernel(reinterpret_cast<const void*>(&paged_join_kernel<HD, T>), dim3(a.b.n_seqs, (unsigned)(slices < 1024 ? slices : 1024)),
                         dim3(kJoinThreads), 0, s, true, &p);
  }
  if (a.b.max_pages * ps <= kKT) return cudaSuccess;  // every unit is one key tile: nothing is cut
  return launch_kernel(reinterpret_cast<const void*>(&paged_merge_kernel<HD, T>), dim3(grid, kMergeSlices),
                       dim3(kMergeThreads), 0, s, true, &p);
}
}  // namespace

template <bool kShared>
static cudaError_t launch_any(const PagedAttnArgs& a, int head_dim, int type, int device, int grid, cudaStream_t s) {
  if (head_dim == 128)
    return type == 1 ? launch<128, __half, kShared>(a, device, grid, false, s)
                     : launch<128, __nv_bfloat16, kShared>(a, device, grid, true, s);
  return type == 1 ? launch<64, __half, kShared>(a, device, grid, false, s)
                   : launch<64, __nv_bfloat16, kShared>(a, device, grid, true, s);
}
cudaError_t paged_attention(const PagedAttnArgs& a, int head_dim, int type, int device, int n_sms, cudaStream_t s) {
  return launch_any<false>(a, head_dim, type, device, paged_attention_grid(n_sms), s);
}
cudaError_t paged_attention_shared(const PagedAttnArgs& a, int head_dim, int type, int device, cudaStream_t s) {
  return launch_any<true>(a, head_dim, type, device, paged_attention_grid(a.n_sms), s);
}

}  // namespace yb
