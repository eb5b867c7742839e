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
// that are read again, from L2); every later pass reads that.  The limits are found on a histogram of the distance
// to the maximum, 16 bins an octave of the weight, whose bins are stretches of the sorted order:
//   top-k: of counts of maxima of parts of the row, which need no weights; what lies above the limit's bin is listed;
//   top-p alone: of about the weights, in 32 bits, one atomic a logit; then one pass of exact sums (all, those before the
//     limit's bin, those that are kept by warp) that lists the bin, or all up to it where they are few.  The sums tell
//     whether the bin was the right one.  (Exact weights in the histogram took four atomics a logit, 17 us of 63 for 64
//     rows of 131072, and a further pass over them.)
//   what does not fit the list, kList tokens in the first block: by exact histograms, of the limit's own range of (value,
//     place in the row, as one 64-bit number) until it does.
// A list is worked on in the first block: by comparing each with each where they are few, else by histograms of
// the list's own range, which a round or three narrow down to one token.  (Sorting the list took 2.5 us for 64 tokens and
// 8 to 13 us for 2048, twice.)  Without such a list the draw is a pass over the row in its order.
//
// What it costs: one read for the largest logit (temperature 0: 64 rows of 131072 in 16 bits 7.7 us, 256 of fp32 41, half of
// the memory's rate: a block has no load under way while it works), else about 39 instructions a logit for a weight in 64
// bits and its sum (27 us), 105 in all for top-p (56), and 5 to 10 phases of a cluster, about 1 us each (one row of 32000:
// 3.8 us at temperature 0, 7.8 without limits, 9.5 with top-k).
#include "sample_rows.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include "cluster.cuh"
#include "launch.h"
#include "paged.cuh"

namespace yb {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kOctaves = 44, kPerOctave = 16, kBins = kOctaves * kPerOctave;
constexpr int kEach = 4, kList = kThreads * kEach;  // tokens of a list: 4 a thread
constexpr int kBinsPer = (kBins + kThreads - 1) / kThreads;
constexpr int kShortList = 128;
constexpr int kMaxima = 4;  // of a thread, of each fourth chunk that it reads
constexpr int kPart = 14;  // kMostLogits of 2^kPart, and 2 % more, fit 32 bits
constexpr int kRounds = 8;  // kBins^7 is more than 2^64, the places that a range may have
constexpr u64 kOne = 1ull << 43;                    // the largest weight
constexpr float kLeastTemperature = 0x1p-60f, kMostTemperature = 0x1p90f;
constexpr size_t kMaxStage = 160 * 1024;            // bytes of a row's stretch that shared memory takes
constexpr int kMaxCluster = 8;
constexpr int kMostLogits = kSampleMaxVocab / kMaxCluster;  // of a block: sums by parts of weights are sized for them

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// 16 bytes of logits
template <typename T>
struct Chunk {
  static constexpr int kN = 16 / sizeof(T);
  union {
    uint4 raw;
    T v[kN];
  };
  __device__ __forceinline__ Chunk() {}
  __device__ __forceinline__ explicit Chunk(uint4 r) : raw(r) {}
  __device__ __forceinline__ float operator[](int j) const { return to_float(v[j]); }
};
template <typename T>
__device__ __forceinline__ T minus_infinity();
template <>
__device__ __forceinline__ float minus_infinity() { return -INFINITY; }
template <>
__device__ __forceinline__ __half minus_infinity() { return __ushort_as_half(0xfc00); }
template <>
__device__ __forceinline__ __nv_bfloat16 minus_infinity() { return __ushort_as_bfloat16(0xff80); }

// Numbers in the order of the values (no NaN comes here; -0 counts as 0), and back.
__device__ __forceinline__ unsigned key_of(float l) {
  const unsigned u = __float_as_uint(l + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// In the order of the limits: the larger value first, then the smaller index.
__device__ __forceinline__ u64 place_of(float l, int i) { return ((u64)key_of(l) << 32) | (unsigned)~i; }

// A finite fp32 number in 64 bits, by its bits: the conversion unit takes 16 a clock at most, and was what the weights
// waited for.  Zeros and numbers below 2^-126 come out wrong by up to 2^-126, which no temperature here sees.
__device__ __forceinline__ double widen(float l) {
  const unsigned u = __float_as_uint(l);
  return __hiloint2double((int)((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(u << 29));
}
constexpr double kUnits = 4503599627370496.0;  // 2^52: added, it leaves a whole number of units in the low bits

// The row's weights, by all lanes of a warp at once: 2^t = 2^(k / 32) 2^r with k the nearest whole number to 32 t; lane
// j holds 2^(j / 32), and 2^r, |r| <= 1/64, is its Taylor series up to r^5 (2^-48.7 relative).  The last product adds
// 2^52, which rounds to whole units.  11 operations in 64 bits, where exp2 takes about 25.
struct Weights {
  double max, c, root;  // the maximum, log2(e) / T, 2^(lane / 32 + 43)
  float maxf, cut;      // what lies below cut has no weight
  float none;           // nor has this, which stands for all that lies below it, and for NaN
  float per_bin;        // bins a unit of l
  // a number at or below all logits of the bins up to b that have a weight, and one above those of bin b > 0
  __device__ __forceinline__ float ceiling_of_bin(int b) const {
    return fminf(maxf, __double2float_ru(max - (b - 1) * (double)(1.f - 0x1p-20f) / per_bin));
  }
  __device__ __forceinline__ float floor_of_bins(int b) const {
    return b == kBins - 1 ? cut : fmaxf(cut, __double2float_rd(max - (b + 1) * (double)(1.f + 0x1p-20f) / per_bin));
  }
  double of_t;  // log2(e) / T before the maximum is known
  __device__ __forceinline__ void prepare(float temp) {
    root = exp2((threadIdx.x & 31) * (1.0 / 32) + 43.0);
    of_t = 1.4426950408889634 / (double)fminf(fmaxf(temp, kLeastTemperature), kMostTemperature);
  }
  __device__ __forceinline__ void init(float m) {
    maxf = m;
    max = widen(m);  // (2^128 for infinity)
    if (m == INFINITY) {  // the infinite ones weigh the same, the largest finite number 2^-50 of it
      c = 50.0 * 0x1p-104;
      cut = m;
      none = FLT_MAX;
      per_bin = 0.f;
      return;
    }
    // Where the number below the maximum weighs nothing already, nothing changes down to 2^-50 of it: logarithms stay
    // small enough for the exponents below.  (At |m| >= 2^127 that is so at every temperature; -infinity counts as -2^128.)
    const unsigned u = __float_as_uint(m);
    const double gap = max - widen(__uint_as_float(m > 0.f ? u - 1 : m < 0.f ? u + 1 : 0x80000001u));
    c = fmin(of_t, (double)__fdividef(50.f, (float)gap));
    const double octave = (double)__frcp_rn((float)c);
    cut = fmaxf((float)(max - kOctaves * octave), -FLT_MAX);
    none = __double2float_rd(max - (kOctaves + 2) * octave);
    per_bin = (float)(c * kPerOctave);
  }
  __device__ __forceinline__ bool some(float l) const { return l >= cut; }
  // 2^23 + the bin (or more than the last one's) of what has a weight; the sum rounds to a whole number
  __device__ __forceinline__ float bin_above(float l) const { return fmaf(fminf(maxf - l, FLT_MAX), per_bin, 8388608.f); }
  __device__ __forceinline__ int bin(float l) const { return min(__float_as_int(bin_above(l)) - 0x4b000000, kBins - 1); }
  // The same, and about 2^kPart times the weight's ratio to that of the bin's middle: 2^-x by its series up to x^2, |x| <= 1/32.
  __device__ __forceinline__ int bin_and_part(float l, unsigned* part) const {
    const float d = fminf(maxf - l, FLT_MAX), b = fmaf(d, per_bin, 8388608.f), x = fmaf(d, per_bin, 8388608.f - b);
    constexpr float kSlope = 0.69314718f / kPerOctave, kScale = 1 << kPart;
    const float y = fmaf(x, fmaf(x, 0.5f * kSlope * kSlope * kScale, -kSlope * kScale), kScale + 8388608.f);
    *part = (unsigned)(__float_as_int(y) - 0x4b000000);
    return min(__float_as_int(b) - 0x4b000000, kBins - 1);
  }
  // 2^52 + the weight in units
  __device__ __forceinline__ double above(float l) const {
    const double t = (widen(fmaxf(l, none)) - max) * c;
    constexpr double kRound = 6755399441055744.0;  // 1.5 2^52
    double k = fma(t, 32.0, kRound);
    const int n = __double2loint(k);
    k -= kRound;
    const double r = fma(k, -1.0 / 32, t);
    double p = fma(r, 0.00133335581464284434, 0.00961812910762847716);
    p = fma(r, p, 0.0555041086648215800);
    p = fma(r, p, 0.240226506959100712);
    p = fma(r, p, 0.693147180559945309);
    p = fma(r, p, 1.0);
    const int hi = __shfl_sync(0xffffffffu, __double2hiint(root), n), lo = __shfl_sync(0xffffffffu, __double2loint(root), n);
    return fma(__hiloint2double(hi + (n & ~31) * (1 << 15), lo), p, kUnits);
  }
  __device__ __forceinline__ u64 of(float l) const {
    return (u64)__double_as_longlong(above(l)) - 0x4330000000000000ull;
  }
};
// The least whole sum that is at least x * sum, 1 .. sum: in whole numbers, x = m 2^-d with 24 bits m, since a sum of up to 2^63
// does not fit the 53 bits of a 64-bit floating-point number.
__device__ __forceinline__ u64 share_of(float x, u64 sum) {
  if (!(x > 0.f)) return 1;
  if (x >= 1.f) return sum;
  const unsigned u = __float_as_uint(x), e = u >> 23;
  const u64 m = e ? (u & 0x7fffffu) | 0x800000u : u;
  const unsigned d = 150 - (e ? e : 1);  // 24 .. 149
  const u64 lo = m * sum, hi = __umul64hi(m, sum);  // hi < 2^24
  if (d >= 88) return 1;  // the whole product is below 2^87
  if (d >= 64) return (hi >> (d - 64)) + (lo || (hi & ((1ull << (d - 64)) - 1)));
  return (hi << (64 - d) | lo >> d) + ((lo & ((1ull << d) - 1)) != 0);
}

struct Pair {
  unsigned n;
  u64 sum;
};
__device__ __forceinline__ Pair operator+(const Pair& a, const Pair& b) { return {a.n + b.n, a.sum + b.sum}; }
__device__ __forceinline__ u64 warp_scan(u64 v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ Pair warp_scan(Pair v) {
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
  bool by_rank;  // top-k is the limit, else top-p
  int bin;       // the histogram's bin that it is in
  u64 lo, hi;    // or the range of places
  Pair before;   // what comes before the bin or range
  unsigned in;   // tokens in it
  u64 of, goal;  // the sum that top-p is a share of, and that share
};

struct Shared {
  // of sums of weights 15 bits, the next 15, and the rest, each summed by itself: kMostLogits (2^17) of them fit 32 bits
  unsigned count[kBins], low[kBins], mid[kBins], high[kBins];
  u64 list[kList];
  Pair warps[kWarps];
  u64 sums[kWarps], lo[kWarps], hi[kWarps];
  u64 block_sum, told;
  // What the first block found, for the others.  Nothing that it does by itself after cluster_arrive (finish, and select,
  // which has `told` for its own threads) writes this or `listed`: the others may read them as late as they leave.
  u64 verdict;
  Pair found_before;
  unsigned mine;  // tokens that the block has listed for the first one
  u64 weights, before;  // of the block's logits: all, those of the bins before the limit's
  float coin, top_p;  // the row's settings
  int top_k;
  u64 least;  // weight
  float max[kWarps], block_max;
  int block_first;  // index of the block's first maximum
  unsigned listed;
  int found;
  Order order;
  __device__ __forceinline__ u64* of_list() { return reinterpret_cast<u64*>(low); }  // weights of a short list
};

// Inclusive scans over the block of a value a thread; every thread is to call them.
__device__ __forceinline__ Pair block_scan(Shared& s, Pair v, Pair* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  v = warp_scan(v);
  if (lane == 31) s.warps[warp] = v;
  __syncthreads();
  const Pair w = warp_scan(lane < kWarps ? s.warps[lane] : Pair{0, 0});
  const int before = max(warp - 1, 0);
  const Pair at{__shfl_sync(0xffffffffu, w.n, before), __shfl_sync(0xffffffffu, w.sum, before)};
  *total = Pair{__shfl_sync(0xffffffffu, w.n, kWarps - 1), __shfl_sync(0xffffffffu, w.sum, kWarps - 1)};
  __syncthreads();
  return warp ? at + v : v;
}
__device__ __forceinline__ void clear_bins(Shared& s, bool sums) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
    if (sums) s.low[i] = s.mid[i] = s.high[i] = 0;
  }
}
__device__ __forceinline__ void add_to_bin(Shared& s, int b, double above) {  // 2^52 + the weight
  const unsigned lo = (unsigned)__double2loint(above), hi = (lo >> 30) | (unsigned)(__double2hiint(above) - 0x43300000) << 2;
  atomicAdd(&s.count[b], 1u);
  atomicAdd(&s.low[b], lo & 0x7fffu);
  atomicAdd(&s.mid[b], (lo >> 15) & 0x7fffu);
  if (hi) atomicAdd(&s.high[b], hi);
}

__device__ __forceinline__ void add_to_bin(Shared& s, int b, u64 w) {
  atomicAdd(&s.low[b], (unsigned)w & 0x7fffu);
  atomicAdd(&s.mid[b], (unsigned)(w >> 15) & 0x7fffu);
  if (w >> 30) atomicAdd(&s.high[b], (unsigned)(w >> 30));
}
__device__ __forceinline__ u64 block_sum(Shared& s, u64 v) {
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) s.sums[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.sums[threadIdx.x & (kWarps - 1)];
  for (int d = kWarps / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  __syncthreads();
  return v;
}
// Of a list of different numbers, 4 a thread (0: none), the one at which, from the largest down, `rank` (by_rank) or the
// sum `goal` of their weights is reached.  Each round leaves one of kBins parts of the range that is still in question,
// until few are left (they take the place of what is in s.list), which are compared each with each.
__device__ __forceinline__ u64 select(Shared& s, u64 (&v)[kEach], const u64 (&weight)[kEach], bool by_rank, unsigned rank, u64 goal) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b0 = threadIdx.x * kBinsPer;
  for (int round = 0;; ++round) {
    u64 lo = ~0ull, hi = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (v[e]) {
        lo = v[e] < lo ? v[e] : lo;
        hi = v[e] > hi ? v[e] : hi;
      }
    auto ends = [&](int d) {
      for (; d; d >>= 1) {
        const u64 l = __shfl_xor_sync(0xffffffffu, lo, d), h = __shfl_xor_sync(0xffffffffu, hi, d);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
      }
    };
    ends(16);
    if (lane == 0) {
      s.lo[warp] = lo;
      s.hi[warp] = hi;
    }
    clear_bins(s, !by_rank);
    if (threadIdx.x == 0) {
      s.found = -1;  // (a goal beyond the sum would end with none)
      s.mine = 0;
      s.told = 0;
    }
    __syncthreads();
    lo = s.lo[lane % kWarps];
    hi = s.hi[lane % kWarps];
    ends(kWarps / 2);
    if (lo >= hi || round == kRounds) {
      __syncthreads();
      return hi;
    }
    const float per = (float)kBins / ((float)(hi - lo) + 1.f);  // (roundings keep the order)
    int bin[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      bin[e] = min((int)((float)(hi - v[e]) * per), kBins - 1);
      if (!v[e]) continue;
      if (by_rank) atomicAdd(&s.count[bin[e]], 1u);
      else add_to_bin(s, bin[e], weight[e]);
    }
    __syncthreads();
    Pair part[kBinsPer], mine{0, 0}, total;
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const int b = b0 + k;
      part[k] = Pair{0, 0};
      if (b < kBins) {
        if (by_rank) part[k].n = s.count[b];
        else part[k].sum = s.low[b] + ((u64)s.mid[b] << 15) + ((u64)s.high[b] << 30);
      }
      mine = mine + part[k];
    }
    Pair before = block_scan(s, mine, &total);
    before = Pair{before.n - mine.n, before.sum - mine.sum};
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const Pair after = before + part[k];
      if (by_rank ? before.n < rank && rank <= after.n : before.sum < goal && goal <= after.sum) {
        s.found = b0 + k;
        s.found_before = before;
      }
      before = after;
    }
    __syncthreads();
    const int found = s.found;
    rank -= s.found_before.n;
    goal -= s.found_before.sum;
    u64* const weights = s.of_list();
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (bin[e] != found) v[e] = 0;
      if (!v[e]) continue;
      const unsigned to = atomicAdd(&s.mine, 1u);
      if (to < kShortList) {
        s.list[to] = v[e];
        weights[to] = weight[e];
      }
    }
    __syncthreads();
    const int left = (int)s.mine;
    if (left <= kShortList) {
      if (threadIdx.x < left) {
        const u64 own = s.list[threadIdx.x];
        unsigned larger = 0;
        u64 before = 0;
        for (int j = 0; j < left; ++j) {
          const bool more = s.list[j] > own;
          larger += more;
          before += more ? weights[j] : 0;
        }
        if (by_rank ? larger + 1 == rank : before < goal && goal <= before + weights[threadIdx.x]) s.told = own;
      }
      __syncthreads();
      const u64 at = s.told;
      __syncthreads();
      return at;
    }
  }
}

template <typename T, bool kStaged>
__global__ void __launch_bounds__(kThreads, 2) sample_rows_kernel(const __grid_constant__ SampleRowsArgs a, int stretch) {
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ Shared s;
  constexpr int kVec = Chunk<T>::kN;
  const int blocks = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
  const int r = blockIdx.x / blocks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i0 = min(a.vocab, rank * stretch), n = min(a.vocab, i0 + stretch) - i0;  // this block's stretch
  pdl_wait();
  const float temp = a.temperature ? __ldca(a.temperature + r) : 1.f;
  const bool greedy = !(temp > 0.f);

  // The stretch in chunks of 16 bytes, as they lie in memory: element 0 is the chunk 0's element `shift`, and what lies
  // before and behind counts as -infinity.
  const T* g = static_cast<const T*>(a.logits) + (size_t)r * a.stride + i0;
  const int shift = (int)(reinterpret_cast<uintptr_t>(g) / sizeof(T) % kVec);
  const int chunks = n > 0 ? (shift + n + kVec - 1) / kVec : 0;
  const uint4* const from = reinterpret_cast<const uint4*>(g - shift);
  uint4* const stage = reinterpret_cast<uint4*>(smem_raw);
  auto fetch = [&](int c, bool again) -> Chunk<T> {
    if (c * kVec >= shift && (c + 1) * kVec <= shift + n) return Chunk<T>(again ? __ldca(from + c) : __ldcs(from + c));
    Chunk<T> v;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int i = c * kVec + j - shift;
      v.v[j] = i >= 0 && i < n ? g[i] : minus_infinity<T>();
    }
    return v;
  };
  Weights w;
  w.prepare(temp);
  float own;  // the largest logit that this thread has read
  {
    constexpr int kAhead = kMaxima;
    float part[kMaxima];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) part[k] = -INFINITY;
    for (int c = threadIdx.x; c < chunks; c += kThreads * kAhead) {
      Chunk<T> v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (c + k * kThreads < chunks) v[k] = fetch(c + k * kThreads, !kStaged);
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (c + k * kThreads < chunks) {
          if (kStaged) stage[c + k * kThreads] = v[k].raw;
#pragma unroll
          for (int j = 0; j < kVec; ++j) part[k] = fmaxf(part[k], v[k][j]);
        }
    }
    reinterpret_cast<float4*>(s.list)[threadIdx.x] = make_float4(part[0], part[1], part[2], part[3]);
    float m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    own = m;
    if (threadIdx.x == 0) {  // (registers are short)
      const float min_p = a.min_p ? __ldca(a.min_p + r) : 0.f;
      s.coin = __ldca(a.coin + r);
      s.top_p = a.top_p ? __ldca(a.top_p + r) : 1.f;
      s.top_k = a.top_k ? __ldca(a.top_k + r) : 0;
      s.least = !(min_p > 0.f) ? 0 : min_p >= 1.f ? kOne : __double2ull_ru(min_p * (double)kOne);
    }
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) s.max[warp] = m;
    if (threadIdx.x == 0) s.block_first = a.vocab;
    __syncthreads();
    m = s.max[lane % kWarps];
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (greedy && own == m && m > -INFINITY) {  // the few threads that have met it look where
      int first = a.vocab;
      for (int c = threadIdx.x; c < chunks && first == a.vocab; c += kThreads) {
        const Chunk<T> v = kStaged ? Chunk<T>(stage[c]) : fetch(c, true);
#pragma unroll
        for (int j = kVec - 1; j >= 0; --j)
          if (v[j] == m) first = i0 + c * kVec + j - shift;
      }
      atomicMin(&s.block_first, first);
    }
    if (threadIdx.x == 0) s.block_max = m;
    cluster_sync_all();
    // (lanes read the blocks of the cluster side by side: a trip to another block's memory each)
    if (lane < blocks) m = fmaxf(m, *dsmem_ptr(&s.block_max, lane));
    for (int o = kMaxCluster / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = __shfl_sync(0xffffffffu, m, 0);
    w.init(m);
  }
  auto answer = [&](int token, float prob) {
    a.tokens[r] = token;
    if (a.prob) a.prob[r] = prob;
  };
  if (greedy || w.maxf == -INFINITY) {
    if (rank == 0 && warp == 0) {
      int first = a.vocab;
      if (lane < blocks && w.maxf > -INFINITY && *dsmem_ptr(&s.block_max, lane) == w.maxf) first = *dsmem_ptr(&s.block_first, lane);
      first = __reduce_min_sync(0xffffffffu, first);
      if (lane == 0) answer(first < a.vocab ? first : 0, first < a.vocab ? 1.f : 0.f);  // (or there is nothing to draw)
    }
    cluster_sync_all();  // nobody leaves while others read its shared memory
    return;
  }
  const bool by_p = s.top_p < 1.f, by_k = s.top_k > 0 && s.top_k < a.vocab;
  // A warp's part of the stretch; f is called by whole warps, with -infinity behind the end.
  const int part = (chunks + kWarps - 1) / kWarps, c0 = min(chunks, warp * part), c1 = min(chunks, c0 + part);
  auto chunk_at = [&](int c, int end) -> Chunk<T> {
    if (c < end) return kStaged ? Chunk<T>(stage[c]) : fetch(c, true);
    Chunk<T> v;
#pragma unroll
    for (int j = 0; j < kVec; ++j) v.v[j] = minus_infinity<T>();
    return v;
  };
  auto index_of = [&](int c, int j) { return i0 + c * kVec + j - shift; };
  // Four logits at a time, f(index of the first, logits).
  auto each4 = [&](auto&& f) {
    Chunk<T> next;
    if (!kStaged) next = chunk_at(c0 + lane, c1);
    for (int b = c0; b < c1; b += 32) {
      const Chunk<T> v = kStaged ? chunk_at(b + lane, c1) : next;
      if (!kStaged) next = chunk_at(b + 32 + lane, c1);
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        const float l[4] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
        f(index_of(b + lane, j), l);
      }
    }
  };
  auto each = [&](auto&& f) {
    each4([&](int i, const float (&l)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f(i + j, l[j]);
    });
  };
  const Order* const told = dsmem_ptr(&s.order, 0);
  Shared* const first = const_cast<Shared*>(dsmem_ptr(&s, 0));
  // Merges the bins of all blocks, and tells where `rank` (if any) or else the sum `goal` is reached; bin j is places
  // hi - (j + 1) width + 1 .. hi - j width of the range, or of the first histogram's (width 0).  Counts the first block
  // reads from all; of counts and sums, four words a bin, each block sums up a part and leaves it in the first one's list.
  auto tell = [&](bool by_rank, Pair before, u64 goal, u64 of, u64 lo, u64 hi, u64 width) {
    Pair mine{0, 0}, bin[kBinsPer], total;
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const int b = threadIdx.x * kBinsPer + k;
      bin[k] = Pair{0, 0};
      if (!by_rank) {
        if (b < kBins) bin[k] = Pair{(unsigned)s.list[kBins + b], s.list[b]};
      } else {
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c)  // all on their way at once
          if (c < blocks && b < kBins) bin[k].n += dsmem_ptr(&s, c)->count[b];
      }
      mine = mine + bin[k];
    }
    const Pair upto = block_scan(s, mine, &total);
    before = before + Pair{upto.n - mine.n, upto.sum - mine.sum};
    if (!width) {  // the first histogram: it holds all weights
      of = total.sum;
      goal = share_of(s.top_p, of);
    }
    if (threadIdx.x == 0) {
      s.order.what = Order::kNone;
      s.order.in = 0;
      s.listed = 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kBinsPer; ++k) {
      const Pair after = before + bin[k];
      const int b = threadIdx.x * kBinsPer + k;
      if (by_rank ? before.n < (unsigned)s.top_k && (unsigned)s.top_k <= after.n : before.sum < goal && goal <= after.sum) {
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
  auto find = [&](bool by_rank, Pair before, u64 goal, u64 of, u64 lo, u64 hi, u64 width) {
    cluster_sync_all();
    if (!by_rank) {
      const int per = (kBins + blocks - 1) / blocks, end = min(kBins, (rank + 1) * per);
      for (int b = rank * per + threadIdx.x; b < end; b += kThreads) {
        unsigned n = 0;
        u64 sum = 0;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
          if (c >= blocks) continue;
          const Shared* o = dsmem_ptr(&s, c);
          n += o->count[b];
          sum += o->low[b] + ((u64)o->mid[b] << 15) + ((u64)o->high[b] << 30);
        }
        first->list[b] = sum;
        first->list[kBins + b] = n;
      }
      cluster_sync_all();
    }
    if (rank == 0) tell(by_rank, before, goal, of, lo, hi, width);
    cluster_sync_all();
  };
  // Lists in the first block what f(list) lists of the block's logits (the counts leave room for all, or s.listed tells):
  // every block in its own list, which is then copied to a place behind those of others.
  auto collect = [&](auto&& f) {
    unsigned* const listed = rank ? &s.mine : &s.listed;
    if (rank && threadIdx.x == 0) s.mine = 0;
    __syncthreads();
    f([&](int i, float l) {
      const unsigned to = atomicAdd(listed, 1u);
      if (to < kList) s.list[to] = place_of(l, i);
    });
    if (rank) {
      __syncthreads();
      if (threadIdx.x == 0) s.found = (int)atomicAdd(&first->listed, s.mine);
      __syncthreads();
      for (unsigned i = threadIdx.x; i < min(s.mine, (unsigned)kList); i += kThreads)
        if (s.found + i < kList) first->list[s.found + i] = s.list[i];
    }
    cluster_sync_all();
  };
  // What is from least_l to most_l and passes a test.
  auto pick = [&](float least_l, float most_l, auto&& test) {
    collect([&](auto&& list) {
      each4([&](int i, const float (&l)[4]) {
        if (fmaxf(fmaxf(l[0], l[1]), fmaxf(l[2], l[3])) >= least_l) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (l[j] >= least_l && l[j] <= most_l && test(i + j, l[j])) list(i + j, l[j]);
        }
      });
    });
  };
  // The first block's list, 4 tokens a thread, and their weights.
  u64 v[kEach], weight[kEach];
  int listed = 0;
  auto take_list = [&] {
    listed = min((int)s.listed, kList);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int i = e * kThreads + threadIdx.x;
      v[e] = i < listed ? s.list[i] : 0;
      weight[e] = 0;
      if (e * kThreads < listed) weight[e] = w.of(value_of((unsigned)(v[e] >> 32)));
      if (!v[e]) weight[e] = 0;
    }
    __syncthreads();
  };
  // The list holds the first tokens, at least those that are kept: by rank, or else by the share of the sum `of`.
  auto finish = [&](bool by_rank, u64 of) {
    take_list();
    if (listed <= kShortList) {  // each with each: the larger ones' number and sum, then the sum of those of a lower index
      u64* const weights = s.of_list();
      const int i = threadIdx.x;
      if (i < listed) weights[i] = weight[0];
      __syncthreads();
      int larger = 0;
      u64 before = 0, lower = 0, sum = 0;
      if (i < listed)
        for (int j = 0; j < listed; ++j) {
          const bool more = s.list[j] > v[0];
          larger += more;
          before += more ? weights[j] : 0;
        }
      bool keep = i < listed && (!by_rank || larger < s.top_k);
      if (by_p) {
        const u64 all = by_rank ? block_sum(s, keep ? weight[0] : 0) : of;
        keep = keep && before < share_of(s.top_p, all);
      }
      keep = keep && weight[0] >= s.least && weight[0];
      __syncthreads();
      if (i < listed) weights[i] = keep ? weight[0] : 0;
      __syncthreads();
      if (keep) {
        for (int j = 0; j < listed; ++j) {
          sum += weights[j];
          lower += (unsigned)s.list[j] > (unsigned)v[0] ? weights[j] : 0;  // (indices are held inverted)
        }
        const u64 share = share_of(s.coin, sum);
        if (lower < share && share <= lower + weight[0])
          answer((int)~(unsigned)v[0], (float)((double)weight[0] / (double)sum));
      }
      return;
    }
    u64 from = 0, x[kEach];
    auto all_from = [&] {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        x[e] = v[e] >= from ? v[e] : 0;
        sum += x[e] ? weight[e] : 0;
      }
      return sum;
    };
    if (by_rank && s.top_k < listed) {
      all_from();
      from = select(s, x, weight, true, (unsigned)s.top_k, 0);
    }
    if (by_p) {
      u64 sum = all_from();
      if (by_rank) of = block_sum(s, sum);
      from = select(s, x, weight, false, 0, share_of(s.top_p, of));
    }
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {  // in the order of the row
      x[e] = v[e] && v[e] >= from && weight[e] >= s.least && weight[e] ? v[e] << 32 | v[e] >> 32 : 0;
      mine += x[e] ? weight[e] : 0;
    }
    const u64 sum = block_sum(s, mine), at = select(s, x, weight, false, 0, share_of(s.coin, sum));
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (v[e] && (v[e] << 32 | v[e] >> 32) == at) answer((int)~(unsigned)v[e], (float)((double)weight[e] / (double)sum));
  };
  if (by_k) {
    // The k-th largest of the threads' maxima, of every fourth chunk each, is no larger than the k-th largest logit, and few
    // tokens lie between the two: a histogram of 2048 maxima a block instead of all its logits.  (With one maximum a
    // thread, 1000 tokens of 61 rows of 49999 in 2 blocks a row took 34 us.)
    clear_bins(s, false);
    __syncthreads();
    const float4 part = reinterpret_cast<const float4*>(s.list)[threadIdx.x];
    for (const float l : {part.x, part.y, part.z, part.w})
      if (w.some(l)) atomicAdd(&s.count[w.bin(l)], 1u);
    find(true, Pair{0, 0}, 0, 0, 0, 0, 0);
    const Order o = *told;
    if (o.what == Order::kGather) {
      pick(w.floor_of_bins(o.bin), INFINITY, [](int, float) { return true; });  // (perhaps more than there is room for)
      const unsigned got = *dsmem_ptr(&s.listed, 0);
      if (got <= kList) {
        cluster_arrive();
        if (rank == 0) finish(true, 0);
        cluster_wait();
        return;
      }
    }
  }
  u64 limit = 0;  // places from here on are kept: larger values, and of this one the indices up to limit_i
  float limit_l = 0.f;
  int limit_i = 0;
  auto in_limit = [&](int i, float l) { return l > limit_l || (l == limit_l && i <= limit_i); };
  auto set_limit = [&](u64 at) {
    limit = at;
    limit_l = value_of((unsigned)(limit >> 32));
    limit_i = (int)~(unsigned)limit;
  };
  const double least_above = kUnits + (double)s.least;
  bool summed = false;  // s.lo holds the sums of what the warps' parts of the row keep
  if (by_p && !by_k) {
    // One histogram of about the weights, an atomic a logit, says in which bin the limit should lie; then a pass sums
    // exactly the weights before that bin, and all, and lists the bin.  The sums tell if the limit is in it: else, and
    // where the bin has too many, what is below does it by exact histograms.
    clear_bins(s, false);
    __syncthreads();
    each4([&](int, const float (&l)[4]) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w.some(l[j])) {
          unsigned some;
          const int b = w.bin_and_part(l[j], &some);
          atomicAdd(&s.count[b], some);
        }
    });
    cluster_sync_all();
    const int per = (kBins + blocks - 1) / blocks, end = min(kBins, (rank + 1) * per);
    for (int b = rank * per + threadIdx.x; b < end; b += kThreads) {
      u64 some = 0;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c)
        if (c < blocks) some += dsmem_ptr(&s, c)->count[b];
      first->list[b] = __float2ull_rn((float)some * exp2f(20.f - b * (1.f / kPerOctave)));
      first->list[kBins + b] = (some + (1u << (kPart - 1))) >> kPart;  // to 2 %
    }
    cluster_sync_all();
    if (rank == 0) tell(false, Pair{0, 0}, 0, 0, 0, 0, 0);
    cluster_sync_all();
    const Order o = *told;
    if (o.in <= kList) {
      const bool whole = o.before.n + o.in <= kList * 7 / 8;  // what comes before the bin is listed, too
      const float upper = o.bin == kBins - 1 ? INFINITY : 8388608.f + (float)o.bin, edge = whole ? 0.f : 8388608.f + (float)o.bin;
      double all = 0.0, before = 0.0, keep = 0.0;
      collect([&](auto&& list) {
        each4([&](int i, const float (&l)[4]) {
          double v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = w.above(l[j]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float b = w.bin_above(l[j]);
            const double u = v[j] - kUnits;
            all += u;
            if (b < edge) {
              before += u;
              if (v[j] >= least_above) keep += u;
            } else if (b <= upper && w.some(l[j])) {
              list(i + j, l[j]);
            }
          }
        });
        const u64 all_sum = block_sum(s, __double2ull_rn(all)), before_sum = block_sum(s, __double2ull_rn(before));
        if (threadIdx.x == 0) {
          s.weights = all_sum;
          s.before = before_sum;
        }
      });
      u64 kept_sum = __double2ull_rn(keep);
      for (int d = 16; d; d >>= 1) kept_sum += __shfl_xor_sync(0xffffffffu, kept_sum, d);
      if (rank == 0) {
        u64 sum = 0, prior = 0;
        for (int c = 0; c < blocks; ++c) {
          sum += *dsmem_ptr(&s.weights, c);
          prior += *dsmem_ptr(&s.before, c);
        }
        const bool fits = s.listed <= kList;
        take_list();
        const u64 goal = share_of(s.top_p, sum), here = block_sum(s, (weight[0] + weight[1]) + (weight[2] + weight[3]));
        u64 at = 0;
        if (whole) {
          at = fits && goal <= here ? sum : 0;
        } else if (fits && prior < goal && goal <= prior + here) {
          u64 x[kEach];
#pragma unroll
          for (int e = 0; e < kEach; ++e) x[e] = v[e];
          at = select(s, x, weight, false, 0, goal - prior);
        }
        if (threadIdx.x == 0) s.verdict = at;
      }
      if (threadIdx.x < kWarps && rank) s.low[threadIdx.x] = s.mid[threadIdx.x] = s.high[threadIdx.x] = 0;
      cluster_sync_all();
      const u64 at = *dsmem_ptr(&s.verdict, 0);
      if (at && whole) {
        cluster_arrive();
        if (rank == 0) finish(false, at);
        cluster_wait();
        return;
      }
      if (at) {
        set_limit(at);
        if (rank == 0) {
          if (threadIdx.x < kWarps) s.low[threadIdx.x] = s.mid[threadIdx.x] = s.high[threadIdx.x] = 0;
          __syncthreads();
        }
        // the listed ones that are kept, to the sum of the warp whose part they are in
        auto add = [&](u64 place, u64 of) {
          const int i = (int)~(unsigned)place - i0;
          if (place >= limit && of >= s.least && i < n) add_to_bin(s, (i + shift) / kVec / part, of);
        };
        if (rank == 0) {
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (v[e]) add(v[e], weight[e]);
        } else {
          const int listed = (int)s.mine;
          for (int b = warp * 32; b < listed; b += kThreads) {
            const u64 place = b + lane < listed ? s.list[b + lane] : 0, of = w.of(value_of((unsigned)(place >> 32)));
            if (place) add(place, of);
          }
        }
        __syncthreads();
        if (lane == 0) s.lo[warp] = kept_sum + s.low[warp] + ((u64)s.mid[warp] << 15) + ((u64)s.high[warp] << 30);
        summed = true;
      }
    }
  }
  for (int kind = by_k ? 0 : 1; kind < (by_p && !summed ? 2 : 1); ++kind) {  // top-k, then (if that did not see to it) top-p
    const bool by_rank = kind == 0;
    clear_bins(s, !by_rank);
    __syncthreads();
    if (by_rank) {
      each([&](int, float l) {
        if (w.some(l)) atomicAdd(&s.count[w.bin(l)], 1u);
      });
    } else {
      each4([&](int i, const float (&l)[4]) {
        bool in[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) in[j] = limit ? in_limit(i + j, l[j]) : w.some(l[j]);
        if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) return;
        double v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = w.above(l[j]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (in[j]) add_to_bin(s, w.bin(l[j]), v[j]);
      });
    }
    find(by_rank, Pair{0, 0}, 0, 0, 0, 0, 0);
    Order o = *told;
    if (o.what == Order::kNone) continue;  // no more than k tokens have a weight
    if (o.what == Order::kGather) {
      pick(w.floor_of_bins(o.bin), INFINITY, [&](int i, float l) { return w.bin(l) <= o.bin && (!limit || in_limit(i, l)); });
      if (rank) return;
      finish(by_rank, o.of);
      return;
    }
    // ---- the limit's own place, among too many: a range of values that holds the bin's, whatever index they have
    const int only = o.bin;  // of the first histogram, whose bins these tokens are in
    const float floor_l = w.floor_of_bins(only), ceiling_l = only ? w.ceiling_of_bin(only) : w.maxf;
    o.lo = (u64)key_of(floor_l) << 32;
    o.hi = (u64)key_of(ceiling_l) << 32 | 0xffffffffu;
    auto in_range = [&](float l, u64 at) { return w.bin(l) == only && at >= o.lo && at <= o.hi; };
    for (int round = 0; o.in > kList && round < kRounds; ++round) {  // each leaves one of kBins parts of the range
      const u64 width = (o.hi - o.lo) / kBins + 1;
      clear_bins(s, !by_rank);
      __syncthreads();
      each([&](int i, float l) {
        if (!__any_sync(0xffffffffu, l >= floor_l && l <= ceiling_l)) return;
        const u64 at = l >= floor_l ? place_of(l, i) : 0;
        const bool in = l >= floor_l && (!limit || in_limit(i, l)) && in_range(l, at);
        const double v = by_rank ? 0.0 : w.above(l);
        if (!in) return;
        const int b = (int)((o.hi - at) / width);
        if (by_rank) atomicAdd(&s.count[b], 1u);
        else add_to_bin(s, b, v);
      });
      find(by_rank, o.before, o.goal, o.of, o.lo, o.hi, width);
      o = *told;
    }
    pick(floor_l, ceiling_l, [&](int i, float l) { return (!limit || in_limit(i, l)) && in_range(l, place_of(l, i)); });
    if (rank == 0) {
      take_list();
      const u64 at = select(s, v, weight, by_rank, (unsigned)s.top_k - o.before.n, o.goal - o.before.sum);
      if (threadIdx.x == 0) s.verdict = at;
    }
    cluster_sync_all();
    set_limit(*dsmem_ptr(&s.verdict, 0));
  }
  // ---- the draw, in the order of the row
  // Sums of a thread's weights, up to kMostLogits / 512 of them, are whole numbers of 64-bit floating point.
  auto kept = [&](int i, const float (&l)[4], double (&v)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = 0.0;
    bool in[4] = {true, true, true, true};
    if (limit) {
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = in_limit(i + j, l[j]);
      if (!__any_sync(0xffffffffu, in[0] || in[1] || in[2] || in[3])) return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = w.above(l[j]);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = in[j] && v[j] >= least_above ? v[j] - kUnits : 0.0;
  };
  u64 mine;
  if (!summed) {
    double some = 0.0;
    if (limit) {
      each4([&](int i, const float (&l)[4]) {
        double v[4];
        kept(i, l, v);
        some += (v[0] + v[1]) + (v[2] + v[3]);
      });
    } else {
      each4([&](int, const float (&l)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double v = w.above(l[j]);
          if (v >= least_above) some += v - kUnits;
        }
      });
    }
    mine = __double2ull_rn(some);
    for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0) s.lo[warp] = mine;
  }
  __syncthreads();
  u64 sum = 0;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) sum += s.lo[k];
  if (threadIdx.x == 0) s.block_sum = sum;
  cluster_sync_all();
  u64 before, all;  // of the blocks before this one, of the row
  {
    const u64 here = lane < blocks ? *dsmem_ptr(&s.block_sum, lane) : 0, upto = warp_scan(here);
    before = __shfl_sync(0xffffffffu, upto - here, rank);
    all = __shfl_sync(0xffffffffu, upto, 31);
  }
  const u64 share = share_of(s.coin, all);
  if (before < share && share <= before + sum) {  // the token is in this block
    int owner = 0;
    while (share > before + s.lo[owner]) before += s.lo[owner++];
    // all warps look after a sixteenth each of that warp's part
    const int o0 = min(chunks, owner * part), o1 = min(chunks, o0 + part), sub = (o1 - o0 + kWarps - 1) / kWarps;
    const int s0 = min(o1, o0 + warp * sub), s1 = min(o1, s0 + sub);
    u64 v[kVec], here = 0;
    auto weights_at = [&](int b) {
      const Chunk<T> x = chunk_at(b + lane, s1);
      here = 0;
#pragma unroll
      for (int j = 0; j < kVec; j += 4) {
        const float l[4] = {x[j], x[j + 1], x[j + 2], x[j + 3]};
        double f[4];
        kept(index_of(b + lane, j), l, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) here += v[j + k] = __double2ull_rn(f[k]);
      }
    };
    mine = 0;
    for (int b = s0; b < s1; b += 32) {
      weights_at(b);
      mine += here;
    }
    for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0) s.hi[warp] = mine;
    __syncthreads();
    for (int k = 0; k < warp; ++k) before += s.hi[k];
    if (before < share && share <= before + mine)
      for (int b = s0; b < s1; b += 32) {
        weights_at(b);
        u64 upto = before + warp_scan(here);
        const unsigned there = __ballot_sync(0xffffffffu, upto >= share);
        if (there) {
          if (lane == __ffs(there) - 1) {
            upto -= here;
            bool done = false;
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
              upto += v[j];
              if (!done && upto >= share) {
                done = true;
                answer(index_of(b + lane, j), (float)((double)v[j] / (double)all));
              }
            }
          }
          break;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
      }
  }
  cluster_sync_all();
}

template <typename T>
cudaError_t launch(const SampleRowsArgs& a, int device, int n_sms, cudaStream_t s) {
  // Blocks a row, the cheapest of 1 to 8 by what was measured without limits (in us): a wave of blocks takes 6.5 to 6.8 (8 in
  // clusters of 8 that fill more than half of the SMs) and 0.29 for each 1000 logits of a block, 0.32 if other waves
  // follow, 0.57 if an SM has two blocks, 1.15 times as much for rows in 32 bits that shared memory does not take.  The last
  // wave counts by its part.  Clusters of 4 that have their SMs for themselves, and those of 8, leave an eighth of
  // the places empty.  Measured with 1, 2, 4, 8 blocks a row: 61 rows of 49999: 24, 14.8, 16, 23; 64 of 131072 in 16 bits: 44,
  // 26, 26, 37; 256 of those: 81, 101, 94, 128; 64 of 131072 in 32 bits: 51, 30, 34, 34; one row of 32000: 15.4, 11.6, 8.8,
  // 7.7.  For the 61 rows it says 14.1 with 2 and 13.9 with 4, so they take 4: 1 us lost without limits, 2 gained by rows of
  // mixed settings (33 with 2, 31 with 4).
  int blocks = 1, stretch = 0;
  bool staged = false;
  float best = FLT_MAX;
  for (int c = 1; c <= kMaxCluster; c *= 2) {
    if (c > 1 && a.vocab < 2048 * c) break;
    const int st = ((a.vocab + c - 1) / c + 31) / 32 * 32;
    if (st > kMostLogits) continue;
    const size_t bytes = (size_t)st * sizeof(T) + 32;
    const bool in = bytes <= kMaxStage, one = in && bytes > kMaxStage / 2;  // one: block on an SM
    const float all = (float)a.rows * c, places = (one ? 1.f : 2.f) * n_sms * (c == 8 || (c == 4 && one) ? 0.875f : 1.f);
    const float waves = all <= places ? 1.f : 0.45f * ceilf(all / places) + 0.55f * all / places;
    const bool alone = all <= (c == 8 ? 0.5f : 1.f) * n_sms;
    const float start = c == 1 ? 6.5f : c < 8 || alone ? 6.8f : 8.f;
    const float each = (alone ? 0.29e-3f : one ? 0.32e-3f : 0.57e-3f) * (in || sizeof(T) == 2 ? 1.f : 1.15f);
    const float t = waves * (start + (float)st * each);
    if (t < best) best = t, blocks = c, stretch = st, staged = in;
  }
  const size_t bytes = (size_t)stretch * sizeof(T) + 32;
  const void* fn = staged ? reinterpret_cast<const void*>(&sample_rows_kernel<T, true>)
                          : reinterpret_cast<const void*>(&sample_rows_kernel<T, false>);
  static SmemCap cap;
  const cudaError_t e = cap.raise(reinterpret_cast<const void*>(&sample_rows_kernel<T, true>), device, kMaxStage);
  if (e != cudaSuccess) return e;
  SampleRowsArgs p = a;
  void* params[] = {&p, &stretch};
  return launch_cluster_params(fn, dim3((unsigned)(a.rows * blocks)), dim3(kThreads), staged ? bytes : 0, s, blocks, true, params);
}

}  // namespace

cudaError_t sample_rows(const SampleRowsArgs& a, int type, int device, int n_sms, cudaStream_t s) {
  if (type == 0) return launch<float>(a, device, n_sms, s);
  if (type == 1) return launch<__half>(a, device, n_sms, s);
  return launch<__nv_bfloat16>(a, device, n_sms, s);
}

}  // namespace yb
