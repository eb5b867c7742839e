// A token for every row of logits l, from a given random number each:
//
//   w_i = exp((l_i - max l) / T);  the k first tokens by (l descending, i ascending);  of those the fewest, in that
//   order, whose weights sum to at least p times theirs;  of those the ones with w_i >= min_p;  of those, in the
//   order of i, the first whose running sum reaches coin times the sum.
//
// Weights are computed in 64 bits and held as whole multiples of 2^-43 (the largest is 2^43; up to 2^20 of them fit
// 64 bits), so sums are exact and the same in any order: atomics and any split of a row give the same token.  What
// rounds to none of them (under 2^-44) is out of the draw.
//
// A cluster of blocks has a row, each block a stretch of it, which is read once into shared memory (rows too long for
// that are read again, from L2); every later pass reads that.  The limits are found on a histogram of the weights'
// logarithms, 16 bins an octave, whose bins are stretches of the sorted order (counts and sums, merged over the
// cluster by its first block).  Where the limit's bin and all before it hold at most kList tokens, as a usual
// top-k or top-p has, they are gathered in the first block, sorted, and the rest happens there.  Else the limit's
// place is narrowed down by histograms of the range (value, then place in the row, as one 64-bit number) until
// at most kList tokens are in it, and the draw is one more pass over the row in its order.
#include "sample_rows.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "cluster.cuh"
#include "launch.h"
#include "paged.cuh"

namespace yb {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kOctaves = 44, kPerOctave = 16, kBins = kOctaves * kPerOctave;
constexpr int kList = 2048;
constexpr double kOne = 8796093022208.0;      // 2^43
constexpr size_t kMaxStage = 160 * 1024;      // bytes of a row's stretch that shared memory takes
constexpr int kMaxCluster = 8;

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Numbers in the order of the values (no NaN comes here; -0 counts as 0), and back.
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned u = __float_as_uint(l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// In the order of the limits: the larger value first, then the smaller index.
__device__ __forceinline__ u64 place_of(float l, int i) { return ((u64)key_of(l) << 32) | (unsigned)~i; }

// The row's weights.
struct Weights {
  double max, c;  // log2(e) / T
  float maxf;
  bool flat;  // all that equal the maximum weigh the same, all else nothing (T is 0, or the maximum infinite)
  // the weight's logarithm; NaN or far below -kOctaves for what has none
  __device__ __forceinline__ double log2_of(float l) const {
    if (flat) return l == maxf ? 0.0 : -1e30;
    return ((double)l - max) * c;
  }
  __device__ __forceinline__ double of(double t) const { return t >= -kOctaves ? exp2(t) : 0.0; }
};
__device__ __forceinline__ u64 whole(double w) { return __double2ull_rn(w * kOne); }
__device__ __forceinline__ int bin_of(double t) { return min((int)((float)t * -(float)kPerOctave), kBins - 1); }
// the least whole sum that is at least x * sum, 1 .. sum
__device__ __forceinline__ u64 share_of(float x, u64 sum) {
  if (!(x > 0.f)) return 1;
  if (x >= 1.f) return sum;
  const u64 v = __double2ull_ru((double)x * __ull2double_rn(sum));
  return v < 1 ? 1 : v < sum ? v : sum;
}

struct Pair {
  unsigned n;
  u64 sum;
};
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) { return {a.n + b.n, a.sum + b.sum}; }
__device__ __forceinline__ Pair warp_scan(Pair v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Pair u{__shfl_up_sync(0xffffffffu, v.n, o), __shfl_up_sync(0xffffffffu, v.sum, o)};
    if (lane >= o) v = v + u;
  }
  return v;
}

// What the cluster's first block tells the others: where a limit lies.
struct Order {
  enum { kNone, kGather, kSelect } what;
  bool by_rank;    // top-k is the limit, else top-p
  int bin;         // the histogram's bin that it is in
  u64 lo, hi;      // or the range of places
  Pair before;     // what comes before the bin or range
  unsigned in;     // tokens in it
  u64 of, goal;    // the sum that top-p is a share of, and that share
};

struct Shared {
  unsigned count[kBins], low[kBins], high[kBins];  // of sums, the low and the high 32 bits
  u64 list[kList], mass[kList];
  Pair warps[kWarps];
  u64 lo[kWarps], hi[kWarps];
  u64 block_lo, block_hi, block_sum;
  float max[kWarps], block_max;
  unsigned listed, found;
  Order order;
};

// Inclusive scan over the block of a value a thread; every thread is to call it.
__device__ __forceinline__ Pair block_scan(Shared& s, Pair v, Pair* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  v = warp_scan(v);
  if (lane == 31) s.warps[warp] = v;
  __syncthreads();
  Pair w = warp_scan(lane < kWarps ? s.warps[lane] : Pair{0, 0});
  const int before = max(warp - 1, 0);
  Pair at{__shfl_sync(0xffffffffu, w.n, before), __shfl_sync(0xffffffffu, w.sum, before)};
  if (warp == 0) at = Pair{0, 0};
  if (total) *total = Pair{__shfl_sync(0xffffffffu, w.n, kWarps - 1), __shfl_sync(0xffffffffu, w.sum, kWarps - 1)};
  __syncthreads();
  return at + v;
}

__device__ __forceinline__ void clear_bins(Shared& s) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = s.low[i] = s.high[i] = 0;
}
__device__ __forceinline__ void add_to_bin(Shared& s, int b, u64 w) {
  const unsigned lo = (unsigned)w;
  atomicAdd(&s.count[b], 1u);
  const unsigned was = atomicAdd(&s.low[b], lo), hi = (unsigned)(w >> 32) + (was + lo < was ? 1u : 0u);
  if (hi) atomicAdd(&s.high[b], hi);
}
// The first block: takes the other blocks' bins in.
__device__ __forceinline__ void merge_bins(Shared& s, int blocks) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    unsigned n = 0;
    u64 sum = 0;
    for (int c = 0; c < blocks; ++c) {
      const Shared* o = dsmem_ptr(&s, c);
      n += o->count[i];
      sum += o->low[i] + ((u64)o->high[i] << 32);
    }
    s.count[i] = n;
    s.low[i] = (unsigned)sum;
    s.high[i] = (unsigned)(sum >> 32);
  }
  __syncthreads();
}
constexpr int kBinsPer = (kBins + kThreads - 1) / kThreads;

// Descending, n a power of two.
__device__ __forceinline__ void sort_list(u64* v, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int t = threadIdx.x; t < n / 2; t += kThreads) {
        const int i = 2 * t - (t & (step - 1)), j = i + step;
        const u64 a = v[i], b = v[j];
        if ((a < b) == ((i & size) == 0)) {
          v[i] = b;
          v[j] = a;
        }
      }
      __syncthreads();
    }
}
// Fills the list up with zeros to a power of two, sorts it, and leaves running sums of the weights in s.mass.
// by_index: the list holds (~index, value) instead of (value, ~index).
__device__ __forceinline__ void order_list(Shared& s, int n, const Weights& w, bool by_index) {
  int all = 1;
  while (all < n) all <<= 1;
  for (int i = n + threadIdx.x; i < all; i += kThreads) s.list[i] = 0;
  __syncthreads();
  sort_list(s.list, all);
  const int per = (n + kThreads - 1) / kThreads, i0 = threadIdx.x * per;
  Pair mine{0, 0};
  for (int i = i0; i < min(n, i0 + per); ++i) {
    const unsigned key = by_index ? (unsigned)s.list[i] : (unsigned)(s.list[i] >> 32);
    mine.sum += whole(w.of(w.log2_of(value_of(key))));
    s.mass[i] = mine.sum;
  }
  const u64 before = block_scan(s, mine, nullptr).sum - mine.sum;
  for (int i = i0; i < min(n, i0 + per); ++i) s.mass[i] += before;
  __syncthreads();
}
// The first place in the list whose running sum reaches `sum`; the last if none does.
__device__ __forceinline__ int reaches(Shared& s, int n, u64 sum) {
  if (threadIdx.x == 0) s.found = n - 1;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (s.mass[i] >= sum && (i == 0 || s.mass[i - 1] < sum)) s.found = i;
  __syncthreads();
  const int at = s.found;
  __syncthreads();
  return at;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a, int stretch, int staged) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Shared s;
  const int blocks = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int r = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = min(a.vocab, rank * stretch), n = min(a.vocab, i0 + stretch) - i0;  // this block's stretch
  constexpr int kVec = 16 / sizeof(T);
  pdl_wait();
  const T* g = static_cast<const T*>(a.logits) + (size_t)r * a.stride + i0;
  // a stretch lies in shared memory as far from a 16-byte boundary as in memory
  const int shift = (int)(reinterpret_cast<uintptr_t>(g) / sizeof(T) % kVec);
  T* x = staged ? reinterpret_cast<T*>(smem_raw) + shift : const_cast<T*>(g);
  Weights w;
  {
    float m = -INFINITY;
    const int head = min(n, (kVec - shift) % kVec), body = (n - head) / kVec * kVec;
    auto one = [&](int i) {
      const T v = g[i];
      if (staged) x[i] = v;
      m = fmaxf(m, to_float(v));
    };
    if (threadIdx.x < head) one(threadIdx.x);
    if (threadIdx.x < n - head - body) one(head + body + threadIdx.x);
    constexpr int kAhead = 4;
    for (int i = threadIdx.x; i < body / kVec; i += kThreads * kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i + k * kThreads < body / kVec) v[k] = __ldcs(reinterpret_cast<const uint4*>(g + head) + i + k * kThreads);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i + k * kThreads < body / kVec) {
          if (staged) reinterpret_cast<uint4*>(x + head)[i + k * kThreads] = v[k];
          const T* e = reinterpret_cast<const T*>(&v[k]);
#pragma unroll
          for (int j = 0; j < kVec; ++j) m = fmaxf(m, to_float(e[j]));
        }
    }
    m = fmaxf(m, -INFINITY);  // (NaN alone)
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s.max[warp] = m;
    __syncthreads();
    m = s.max[lane % kWarps];
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (threadIdx.x == 0) s.block_max = m;
    cluster_sync_all();
    for (int c = 0; c < blocks; ++c) m = fmaxf(m, *dsmem_ptr(&s.block_max, c));
    w.maxf = m;
  }
  const float temp = a.temperature ? __ldca(a.temperature + r) : 1.f;
  const bool greedy = !(temp > 0.f);
  w.max = w.maxf;
  w.flat = greedy || w.maxf == INFINITY;
  w.c = 1.4426950408889634 / (double)temp;
  const float coin = greedy ? 0.f : __ldca(a.coin + r);
  const float given_min = greedy || !a.min_p ? 0.f : __ldca(a.min_p + r);
  const float min_p = given_min > 0.f ? fminf(given_min, 1.f) : 0.f;
  const float top_p = greedy || !a.top_p ? 1.f : __ldca(a.top_p + r);
  const int top_k = greedy || !a.top_k ? 0 : __ldca(a.top_k + r);
  const bool by_p = top_p < 1.f, by_k = top_k > 0 && top_k < a.vocab;
  const double least = min_p;

  auto answer = [&](int token, float prob) {
    a.tokens[r] = token;
    if (a.prob) a.prob[r] = prob;
  };
  if (w.maxf == -INFINITY) {  // nothing to draw
    if (rank == 0 && threadIdx.x == 0) answer(0, 0.f);
    cluster_sync_all();  // the others may still read this block's maximum
    return;
  }
  // A warp's part of the stretch: whole steps of 32 tokens, in the order of the row.
  const int part = (n + kThreads - 1) / kThreads * 32, p0 = min(n, warp * part), p1 = min(n, p0 + part);
  auto each = [&](auto&& f) {
    for (int i = p0 + lane; i < p1; i += 32) f(i, to_float(x[i]));
  };
  const Order* const told = dsmem_ptr(&s.order, 0);
  Shared* const first = const_cast<Shared*>(dsmem_ptr(&s, 0));
  // The first block merges the bins of all, and tells where `rank` (if any) or else the sum `goal` is reached; bin j is
  // places hi - (j + 1) width + 1 .. hi - j width of the range, or of the logarithms (width 0).
  auto find = [&](bool by_rank, Pair before, u64 goal, u64 of, u64 lo, u64 hi, u64 width) {
    merge_bins(s, blocks);
    Pair mine{0, 0}, bin[kBinsPer], total;
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const int b = threadIdx.x * kBinsPer + k;
      bin[k] = b < kBins ? Pair{s.count[b], s.low[b] + ((u64)s.high[b] << 32)} : Pair{0, 0};
      mine = mine + bin[k];
    }
    const Pair upto = block_scan(s, mine, &total);
    before = before + Pair{upto.n - mine.n, upto.sum - mine.sum};
    if (!width) {  // the first histogram: it holds all weights
      if (!of) of = total.sum;
      if (by_rank && (unsigned)top_k >= total.n) by_rank = false;
      goal = share_of(top_p, of);
    }
    if (threadIdx.x == 0) {
      s.order.what = Order::kNone;
      s.listed = 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const Pair after = before + bin[k];
      const int b = threadIdx.x * kBinsPer + k;
      if (by_rank ? before.n < (unsigned)top_k && (unsigned)top_k <= after.n : by_p && before.sum < goal && goal <= after.sum) {
        Order o;
        o.what = !width && after.n <= kList ? Order::kGather : Order::kSelect;
        o.by_rank = by_rank;
        o.bin = b;
        o.hi = hi - b * width;
        o.lo = o.hi - lo < width ? lo : o.hi - width + 1;
        o.before = before;
        o.in = bin[k].n;
        o.of = of;
        o.goal = goal;
        s.order = o;
      }
      before = after;
    }
  };
  auto put = [&](u64 at) {  // (the counts leave room for all that come)
    const unsigned to = atomicAdd(&first->listed, 1u);
    if (to < kList) first->list[to] = at;
  };
  u64 limit = 0;  // places from here on are kept
  if (by_k || by_p) {
    bool want_k = by_k;
    u64 of = 0;
    for (;;) {  // once, or once for each limit
      clear_bins(s);
      __syncthreads();
      each([&](int, float l) {
        const double t = w.log2_of(l);
        const u64 v = whole(w.of(t));
        if (v) add_to_bin(s, bin_of(t), v);
      });
      cluster_sync_all();
      if (rank == 0) find(want_k, Pair{0, 0}, 0, of, 0, 0, 0);
      cluster_sync_all();
      Order o = *told;
      if (o.what == Order::kNone) break;  // as many are kept as there are
      if (o.what == Order::kGather) {
        each([&](int i, float l) {
          const double t = w.log2_of(l);
          if (bin_of(t) <= o.bin && whole(w.of(t))) put(place_of(l, i0 + i));
        });
        cluster_sync_all();
        if (rank) return;
        const int m = min((int)s.listed, kList);
        order_list(s, m, w, false);
        int keep = o.by_rank ? min(top_k, m) : m;
        const u64 share = share_of(top_p, o.by_rank ? s.mass[keep - 1] : o.of);
        if (by_p) keep = min(keep, reaches(s, m, share) + 1);
        if (least > 0.0) {
          if (threadIdx.x == 0) s.found = 1;
          __syncthreads();
          for (int i = threadIdx.x; i < keep; i += kThreads)
            if (w.of(w.log2_of(value_of((unsigned)(s.list[i] >> 32)))) >= least) atomicMax(&s.found, i + 1u);
          __syncthreads();
          keep = (int)s.found;
        }
        const u64 sum = s.mass[keep - 1];
        __syncthreads();
        for (int i = threadIdx.x; i < keep; i += kThreads) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;
        order_list(s, keep, w, true);
        const int at = reaches(s, keep, share_of(coin, sum));
        if (threadIdx.x == 0)
          answer((int)~(unsigned)(s.list[at] >> 32), (float)((double)(s.mass[at] - (at ? s.mass[at - 1] : 0)) / (double)sum));
        return;
      }
      // ---- the limit's own place, among too many: the ends of the bin's places first
      u64 lo = ~0ull, hi = 0;
      each([&](int i, float l) {
        const double t = w.log2_of(l);
        if (t >= -kOctaves && bin_of(t) == o.bin && whole(w.of(t))) {
          const u64 at = place_of(l, i0 + i);
          lo = at < lo ? at : lo;
          hi = at > hi ? at : hi;
        }
      });
      for (int d = 16; d; d >>= 1) {
        const u64 l = __shfl_xor_sync(0xffffffffu, lo, d), h = __shfl_xor_sync(0xffffffffu, hi, d);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
      }
      if (lane == 0) {
        s.lo[warp] = lo;
        s.hi[warp] = hi;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int k = 1; k < kWarps; ++k) {
          lo = s.lo[k] < lo ? s.lo[k] : lo;
          hi = s.hi[k] > hi ? s.hi[k] : hi;
        }
        s.block_lo = lo;
        s.block_hi = hi;
      }
      cluster_sync_all();
      lo = ~0ull, hi = 0;
      for (int c = 0; c < blocks; ++c) {
        const u64 l = *dsmem_ptr(&s.block_lo, c), h = *dsmem_ptr(&s.block_hi, c);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
      }
      o.lo = lo;
      o.hi = hi;
      while (o.in > kList) {  // each round leaves one of kBins parts of a range that has at most 2^64 places
        const u64 width = (o.hi - o.lo) / kBins + 1;
        clear_bins(s);
        __syncthreads();
        each([&](int i, float l) {
          const u64 at = l == l ? place_of(l, i0 + i) : 0;
          if (at >= o.lo && at <= o.hi) add_to_bin(s, (int)((o.hi - at) / width), whole(w.of(w.log2_of(l))));
        });
        cluster_sync_all();
        if (rank == 0) find(o.by_rank, o.before, o.goal, o.of, o.lo, o.hi, width);
        cluster_sync_all();
        o = *told;
      }
      each([&](int i, float l) {
        const u64 at = l == l ? place_of(l, i0 + i) : 0;
        if (at >= o.lo && at <= o.hi) put(at);
      });
      cluster_sync_all();
      if (rank == 0) {
        const int m = min((int)s.listed, kList);
        order_list(s, m, w, false);
        const int at = o.by_rank ? top_k - (int)o.before.n - 1 : reaches(s, m, o.goal - o.before.sum);
        if (threadIdx.x == 0) {
          s.order.lo = s.list[at];
          s.order.of = o.before.sum + s.mass[at];
        }
      }
      cluster_sync_all();
      limit = told->lo;
      of = told->of;
      want_k = false;
      if (!o.by_rank || !by_p) break;
    }
  }
  // ---- the draw, in the order of the row
  auto kept = [&](int i, float l) -> u64 {
    if (limit && !(l == l && place_of(l, i) >= limit)) return 0;
    const double v = w.of(w.log2_of(l));
    return v >= least ? whole(v) : 0;
  };
  u64 mine = 0;
  each([&](int i, float l) { mine += kept(i0 + i, l); });
  for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if (lane == 0) s.lo[warp] = mine;
  __syncthreads();
  u64 before = 0, sum = 0;
  for (int k = 0; k < kWarps; ++k) {
    if (k == warp) before = sum;
    sum += s.lo[k];
  }
  if (threadIdx.x == 0) s.block_sum = sum;
  cluster_sync_all();
  sum = 0;
  for (int c = 0; c < blocks; ++c) {
    if (c == rank) before += sum;
    sum += *dsmem_ptr(&s.block_sum, c);
  }
  const u64 goal = share_of(coin, sum);
  if (before < goal && goal <= before + mine) {
    for (int i = p0; i < p1; i += 32) {
      const float l = i + lane < p1 ? to_float(x[i + lane]) : -INFINITY;
      const u64 v = kept(i0 + i + lane, l);
      const u64 upto = before + warp_scan(Pair{0, v}).sum;
      const unsigned there = __ballot_sync(0xffffffffu, upto >= goal);
      if (there) {
        if (lane == __ffs(there) - 1) answer(i0 + i + lane, greedy ? 1.f : (float)((double)v / (double)sum));
        break;
      }
      before = __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  cluster_sync_all();  // nobody leaves while others read its shared memory
}

template <typename T>
cudaError_t launch(const SampleRowsArgs& a, int device, cudaStream_t s) {
  // blocks a row: enough that a stretch fits shared memory, and that a short row's passes are short
  int blocks = 1;
  while (blocks < kMaxCluster && a.vocab > 4096 * blocks) blocks *= 2;
  const int stretch = ((a.vocab + blocks - 1) / blocks + 31) / 32 * 32;
  const size_t bytes = (size_t)stretch * sizeof(T) + 16;
  const int staged = bytes <= kMaxStage;
  const void* fn = reinterpret_cast<const void*>(&sample_rows_kernel<T>);
  static SmemCap cap;
  const cudaError_t e = cap.raise(fn, device, kMaxStage);
  if (e != cudaSuccess) return e;
  SampleRowsArgs p = a;
  int st = stretch, sg = staged;
  void* params[] = {&p, &st, &sg};
  return launch_cluster_params(fn, dim3((unsigned)(a.rows * blocks)), dim3(kThreads), staged ? bytes : 0, s, blocks, true, params);
}

}  // namespace

cudaError_t sample_rows(const SampleRowsArgs& a, int type, int device, cudaStream_t s) {
  if (type == 0) return launch<float>(a, device, s);
  if (type == 1) return launch<__half>(a, device, s);
  return launch<__nv_bfloat16>(a, device, s);
}

}  // namespace yb
