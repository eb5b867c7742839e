// Append to the paged KV cache: one pass over the projections of the batch's new tokens that clips
// them, RMS-normalises every query and key head over its head_dim elements, rotates queries and keys by
// their positions, writes the queries token-major and stores keys and values in their pages:
//
//   x <- clip(x);  q, k: x <- x / sqrt(mean(x^2) + eps) * w;  (a, b) <- (a cos - b sin, a sin + b cos).
//
// Memory-bound: every element is read once and written once, if the instructions stay few (a kernel that issued
// 183 of a warp for every KB moved was bound by them, at a third of the bandwidth; this one issues 107).  8192
// tokens of 32 + 2 x 8 heads of 128 take 35.7 us = 5.6 TB/s (50 us = 6.0 TB/s from fp32), 512 tokens 5.3 us, 64 tokens
// 2.7 us.  A warp has a
// row (token), or a share of its heads where there are few rows, and waits for no other.  A lane holds 16 elements
// of a head, 8 neighbours in either half, so a head is 8 (head_dim 128) or 4 lanes and a warp has 4 or 8 heads at
// a time; loads and stores are 16 bytes a lane and whole lines a head, the sum of squares is 3 or 2 shuffles, and
// the other element of a rotation's pair lies in the same lane (where half-split pairs take a part of the head, it
// comes by shared memory, for 170 instructions a KB and 8 to 12 spilled bytes a thread, which the seven blocks an SM are
// worth: 1803 tokens of 64 + 2 x 8 heads 20.9 us, 16.7 with neighbouring pairs, 15.6 where whole heads are rotated).  Norm weight and angle are one factor for each element of a pair, r (v_e w_e cos + v_f
// w_f (-+sin)), formed once a row and kept in shared memory: in registers they would halve the warps that an SM
// holds.  The loads of the first heads are under way before the row's sequence, its page and the angles are looked
// up, and each later one starts when its registers are free.
#include "paged.cuh"

#include <cuda_bf16.h>

#include <math.h>

#include "launch.h"

namespace yb {

namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
constexpr int kWarpsPerSm = 32;  // rows are shared out among warps up to this many an SM

// how a rotation's pairs lie: (2j, 2j + 1) or (j, j + R / 2), over the whole head or a part of it
enum Pairs { kNeighbours, kHalves, kPartNeighbours, kPartHalves };

// 8 elements as they lie in memory
template <typename S>
struct Raw {
  uint4 v[sizeof(S) / 2];
};
template <typename S>
__device__ __forceinline__ void load8(Raw<S>& r, const S* p) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(S) / 2; ++i) r.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
}
__device__ __forceinline__ float2 unpack(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ float2 unpack(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <typename S>
__device__ __forceinline__ void widen(const Raw<S>& r, float (&x)[8]) {
  const uint32_t u[4] = {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack(u[i], S());
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
__device__ __forceinline__ void widen<float>(const Raw<float>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[4 * i] = __uint_as_float(r.v[i].x);
    x[4 * i + 1] = __uint_as_float(r.v[i].y);
    x[4 * i + 2] = __uint_as_float(r.v[i].z);
    x[4 * i + 3] = __uint_as_float(r.v[i].w);
  }
}
__device__ __forceinline__ uint32_t pack(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where element e of a head lies in a row of shared memory: groups of four by the lanes that hold them, so that
// neighbouring lanes read neighbouring groups (in the head's own order they would meet in the same banks).
template <int HD>
__device__ __forceinline__ int at(int e) {
  return (((e / (HD / 2)) * 2 + ((e >> 2) & 1)) * (HD / 16) + (e % (HD / 2)) / 8) * 4 + (e & 3);
}

template <int HD, typename S, typename T, int P>
__global__ void __launch_bounds__(kThreads, 7) paged_append_kernel(const __grid_constant__ PagedAppendArgs a, int shares,
                                                                int share_groups) {
  constexpr int kLanes = HD / 16;                   // lanes of a head
  constexpr int kHeads = 32 / kLanes;               // heads of a group, which a warp takes at a time
  constexpr int kAhead = sizeof(S) == 4 ? 1 : 2;    // groups loaded ahead
  constexpr bool kNear = P == kNeighbours || P == kPartNeighbours, kPart = P == kPartNeighbours || P == kPartHalves;
  __shared__ __align__(16) float s_fac[kWarps][2][2][HD];  // queries, keys: the factors of v_e and v_f
  __shared__ __align__(16) float s_head[P == kPartHalves ? kWarps : 1][P == kPartHalves ? 512 + 4 : 4];  // heads, four zeros
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = blockIdx.x * kWarps + warp, row = id / shares, share = id % shares;
  if (row >= a.b.n_tokens) return;
  pdl_wait();
  const int l = lane % kLanes, sub = lane / kLanes;  // elements 8 l + j and HD / 2 + 8 l + j of a head, j < 8
  const int H = a.b.n_heads, K = a.b.n_kv_heads, R = a.rotary_dim;
  // groups: those of the query heads, then the key heads', then the value heads'
  const int gq = (H + kHeads - 1) / kHeads, gk = (K + kHeads - 1) / kHeads;
  const int g_begin = share * share_groups, g_end = min(g_begin + share_groups, gq + 2 * gk);
  const S* x = static_cast<const S*>(a.qkv) + (size_t)row * a.qkv_stride + 8 * l;

  Raw<S> raw[kAhead][2];
  auto kind_of = [&](int g) { return g < gq ? 0 : g < gq + gk ? 1 : 2; };
  auto head_of = [&](int g, int kind) { return (g - (kind == 0 ? 0 : kind == 1 ? gq : gq + gk)) * kHeads + sub; };
  auto load = [&](Raw<S> (&to)[2], int g) {
    const int kind = kind_of(g), h = head_of(g, kind);
    if (h >= (kind == 0 ? H : K)) return;
    const S* from = x + (size_t)((kind == 0 ? 0 : kind == 1 ? H : H + K) + h) * HD;
    load8(to[0], from);
    load8(to[1], from + HD / 2);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (g_begin + i < g_end) load(raw[i], g_begin + i);

  // the row's sequence, slot and page
  const int seq = paged_find_seq(a.b, row);
  if (seq < 0) return;
  const PagedSeq sq = paged_seq(a.b, seq);
  if (row - sq.row0 >= sq.n) return;
  const int slot = sq.kv - sq.n + row - sq.row0, pos = a.pos ? __ldca(a.pos + row) : slot;
  int page = -1;
  if (slot >= 0) page = __ldca(a.b.page_table + (size_t)seq * a.b.max_pages + (slot >> a.b.ps_log2));
  const bool there = page >= 0 && page < a.b.n_pages;
  const int d = kNear ? 1 : P == kHalves ? HD / 2 : R / 2;  // distance of a pair's elements
  float (&fac)[2][2][HD] = s_fac[warp];
#pragma unroll
  for (int j = lane; j < HD / 2; j += 32) {
    int e = 2 * j, f = 2 * j + 1;  // a pair, or two elements that are not rotated
    float c = 1.f, s = 0.f;
    if (!kPart || j < R / 2) {
      if (!kNear) e = j, f = j + d;
      // the angle in 64 bits, less whole turns: at a position of 10^5 its product in 32 bits would be off by 0.004
      const double halves = (double)pos * (double)__ldca(a.inv_freq + j) * 0.3183098861837907;  // half turns
      sincospif((float)(halves - 2.0 * rint(0.5 * halves)), &s, &c);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float* w = k ? a.k_norm : a.q_norm;
      const float we = w ? __ldca(w + e) : 1.f, wf = w ? __ldca(w + f) : 1.f;
      fac[k][0][at<HD>(e)] = we * c;
      fac[k][0][at<HD>(f)] = wf * c;
      fac[k][1][at<HD>(e)] = -s * wf;
      fac[k][1][at<HD>(f)] = s * we;
    }
  }
  if (P == kPartHalves && lane < 4) s_head[warp][512 + lane] = 0.f;
  __syncwarp();

  const bool clipped = a.clip < 3.4028234e38f;
  const size_t in_page = ((((size_t)max(page, 0) * K) << a.b.ps_log2) + (slot & ((1 << a.b.ps_log2) - 1))) * HD + 8 * l;
  T* const q_out = static_cast<T*>(a.q_out) + (size_t)row * a.q_stride + 8 * l;
#pragma unroll 1
  for (int g0 = g_begin; g0 < g_end; g0 += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int g = g0 + i;
      if (g >= g_end) break;
      const int kind = kind_of(g);
      float v[16];
      {
        float lo[8], hi[8];
        widen(raw[i][0], lo);
        widen(raw[i][1], hi);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = lo[j], v[8 + j] = hi[j];
      }
      if (g + kAhead < g_end) load(raw[i], g + kAhead);
      if (clipped) {
#pragma unroll
        for (int m = 0; m < 16; ++m) v[m] = v[m] < -a.clip ? -a.clip : (v[m] > a.clip ? a.clip : v[m]);
      }
      float r = 1.f;
      const bool norm = kind == 0 ? a.q_norm != nullptr : kind == 1 && a.k_norm;
      if (norm) {
        float2 ss = mul2(make_float2(v[0], v[1]), make_float2(v[0], v[1]));
#pragma unroll
        for (int m = 2; m < 16; m += 2) ss = fma2(make_float2(v[m], v[m + 1]), make_float2(v[m], v[m + 1]), ss);
        float t = ss.x + ss.y;
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        r = rsqrtf(fmaf(t, 1.f / HD, a.eps));
      }
      float* mine = &s_head[P == kPartHalves ? warp : 0][P == kPartHalves ? sub * HD : 0];
      if (P == kPartHalves && kind < 2) {
        __syncwarp();  // the lanes have read what they need of the group before
#pragma unroll
        for (int m = 0; m < 16; m += 4)
          *reinterpret_cast<float4*>(mine + at<HD>((m >> 3) * (HD / 2) + 8 * l + (m & 7))) = make_float4(v[m], v[m + 1], v[m + 2], v[m + 3]);
        __syncwarp();
      }
      const int h = head_of(g, kind);
      const bool store = h < (kind == 0 ? H : K) && (kind == 0 || there);
      T* out = kind == 0 ? q_out + h * HD
                         : static_cast<T*>(kind == 1 ? a.k_pages : a.v_pages) + in_page + ((size_t)h << a.b.ps_log2) * HD;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float y[8];
        if (kind < 2) {
          float other[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) other[j] = kNear ? v[8 * c + (j ^ 1)] : v[8 * (c ^ 1) + j];
          const int e0 = c * (HD / 2) + 8 * l;
          if (P == kPartHalves) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {  // d is a multiple of 4: four neighbours' partners are neighbours
              const int e = e0 + j, f = e < d ? e + d : e - d;
              const float4 o = *reinterpret_cast<const float4*>(e < R ? mine + at<HD>(f) : &s_head[warp][512]);
              other[j] = o.x, other[j + 1] = o.y, other[j + 2] = o.z, other[j + 3] = o.w;
            }
          }
          if (P == kPartNeighbours) {  // an element that is not rotated takes nothing from another, not even 0 * inf
#pragma unroll
            for (int j = 0; j < 8; ++j) other[j] = e0 + j < R ? other[j] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 o = *reinterpret_cast<const float4*>(&fac[kind][0][at<HD>(e0 + j)]),
                         q = *reinterpret_cast<const float4*>(&fac[kind][1][at<HD>(e0 + j)]);
            y[j] = fmaf(other[j], q.x, v[8 * c + j] * o.x);
            y[j + 1] = fmaf(other[j + 1], q.y, v[8 * c + j + 1] * o.y);
            y[j + 2] = fmaf(other[j + 2], q.z, v[8 * c + j + 2] * o.z);
            y[j + 3] = fmaf(other[j + 3], q.w, v[8 * c + j + 3] * o.w);
          }
          if (norm) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
              const float2 t = mul2(make_float2(y[j], y[j + 1]), make_float2(r, r));
              y[j] = t.x, y[j + 1] = t.y;
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = v[8 * c + j];
        }
        if (store)
          *reinterpret_cast<uint4*>(out + c * (HD / 2)) =
              make_uint4(pack(y[0], y[1], T()), pack(y[2], y[3], T()), pack(y[4], y[5], T()), pack(y[6], y[7], T()));
      }
    }
  }
}

template <int HD, typename S, typename T>
const void* pick_pairs(int pairs) {
  switch (pairs) {
    case kNeighbours: return reinterpret_cast<const void*>(&paged_append_kernel<HD, S, T, kNeighbours>);
    case kHalves: return reinterpret_cast<const void*>(&paged_append_kernel<HD, S, T, kHalves>);
    case kPartNeighbours: return reinterpret_cast<const void*>(&paged_append_kernel<HD, S, T, kPartNeighbours>);
  }
  return reinterpret_cast<const void*>(&paged_append_kernel<HD, S, T, kPartHalves>);
}
template <int HD, typename S>
const void* pick_type(int type, int pairs) {
  return type == 1 ? pick_pairs<HD, S, __half>(pairs) : pick_pairs<HD, S, __nv_bfloat16>(pairs);
}
template <int HD>
const void* pick(int src, int type, int pairs) {
  return src == 0 ? pick_type<HD, float>(type, pairs) : src == 1 ? pick_type<HD, __half>(type, pairs) : pick_type<HD, __nv_bfloat16>(type, pairs);
}

}  // namespace

cudaError_t paged_append(const PagedAppendArgs& a, int head_dim, int src_type, int type, int n_sms, cudaStream_t s) {
  const bool whole = a.rotary_dim == head_dim;
  const int pairs = a.half ? (whole ? kHalves : kPartHalves) : (whole ? kNeighbours : kPartNeighbours);
  const void* fn = head_dim == 128 ? pick<128>(src_type, type, pairs) : pick<64>(src_type, type, pairs);
  // few rows: a warp has a part of a row's groups of heads
  const int in_group = 512 / head_dim;
  const int groups = (a.b.n_heads + in_group - 1) / in_group + 2 * ((a.b.n_kv_heads + in_group - 1) / in_group);
  int shares = kWarpsPerSm * n_sms / a.b.n_tokens;
  shares = shares < 1 ? 1 : shares > groups ? groups : shares;
  int share_groups = (groups + shares - 1) / shares;
  shares = (groups + share_groups - 1) / share_groups;
  const long long warps = (long long)a.b.n_tokens * shares;
  void* args[] = {const_cast<PagedAppendArgs*>(&a), &shares, &share_groups};
  return launch_kernel_params(fn, dim3((unsigned)((warps + kWarps - 1) / kWarps)), dim3(kThreads), 0, s, true, args);
}

}  // namespace yb
