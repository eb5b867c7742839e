// Append to the paged KV cache: one pass over the projections of the batch's new tokens that clips
// them, RMS-normalises every query and key head over its head_dim elements, rotates queries and keys by
// their positions, writes the queries token-major and stores keys and values in their pages.
#include "paged.cuh"

#include <cuda_bf16.h>

#include <math.h>

namespace yb {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// One CTA per row; a warp takes a head at a time.
template <int HD, typename S, typename T>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const PagedAppendArgs a) {
  __shared__ float s_cos[HD / 2], s_sin[HD / 2];
  __shared__ int s_seq;
  __shared__ float s_head[kThreads / 32][HD];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    const int s = paged_find_seq(a.b, row);
    if (lane == 0) s_seq = s;
  }
  __syncthreads();
  const int seq = s_seq;
  if (seq < 0) return;
  const PagedSeq q = paged_seq(a.b, seq);
  if (row - q.row0 >= q.n) return;
  const int slot = q.kv - q.n + row - q.row0;
  const int pos = a.pos ? __ldg(a.pos + row) : slot;
  // the angle in 64 bits: at a position of 10^5 its product in 32 bits would be off by 0.004
  for (int j = threadIdx.x; j < a.rotary_dim / 2; j += kThreads) {
    const double t = (double)pos * (double)a.inv_freq[j];
    const double turns = rint(t * 0.15915494309189535);
    sincosf((float)fma(-turns, 6.283185307179586, t), &s_sin[j], &s_cos[j]);
  }
  __syncthreads();
  int page = -1;
  if (slot >= 0) page = __ldg(a.b.page_table + (size_t)seq * a.b.max_pages + (slot >> a.b.ps_log2));
  const bool store = page >= 0 && page < a.b.n_pages;
  const int H = a.b.n_heads, K = a.b.n_kv_heads, R = a.rotary_dim;
  for (int h = warp; h < H + 2 * K; h += kThreads / 32) {
    const S* x = static_cast<const S*>(a.qkv) + (size_t)row * a.qkv_stride + (size_t)h * HD;
    float v[HD / 32], ss = 0.f;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const float t = to_f(x[lane + 32 * i]);
      v[i] = t < -a.clip ? -a.clip : (t > a.clip ? a.clip : t);
      ss += v[i] * v[i];
    }
    const float* w = h < H ? a.q_norm : h < H + K ? a.k_norm : nullptr;
    if (w) {
      const float r = 1.0f / sqrtf(warp_sum(ss) / HD + a.eps);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) v[i] *= r * w[lane + 32 * i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) s_head[warp][lane + 32 * i] = v[i];
    __syncwarp();
    T* out;
    if (h < H) {
      out = static_cast<T*>(a.q_out) + (size_t)row * a.q_stride + (size_t)h * HD;
    } else {
      if (!store) continue;
      const int g = h < H + K ? h - H : h - H - K;
      out = static_cast<T*>(h < H + K ? a.k_pages : a.v_pages) +
            ((((size_t)page * K + g) << a.b.ps_log2) + (slot & ((1 << a.b.ps_log2) - 1))) * HD;
    }
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) {
      const int e = lane + 32 * i;
      float y = v[i];
      if (h < H + K && e < R) {
        const bool first = a.half ? e < R / 2 : !(e & 1);
        const int j = a.half ? (first ? e : e - R / 2) : e >> 1;
        const float o = s_head[warp][a.half ? (first ? e + R / 2 : e - R / 2) : (e ^ 1)];
        y = first ? v[i] * s_cos[j] - o * s_sin[j] : o * s_sin[j] + v[i] * s_cos[j];
      }
      put(out + e, y);
    }
  }
}

template <int HD, typename S>
const void* pick_type(int type) {
  return type == 1 ? reinterpret_cast<const void*>(&paged_append_kernel<HD, S, __half>)
                   : reinterpret_cast<const void*>(&paged_append_kernel<HD, S, __nv_bfloat16>);
}
template <int HD>
const void* pick(int src, int type) {
  return src == 0 ? pick_type<HD, float>(type) : src == 1 ? pick_type<HD, __half>(type) : pick_type<HD, __nv_bfloat16>(type);
}

}  // namespace

cudaError_t paged_append(const PagedAppendArgs& a, int head_dim, int src_type, int type, cudaStream_t s) {
  const void* fn = head_dim == 128 ? pick<128>(src_type, type) : pick<64>(src_type, type);
  void* args[] = {const_cast<PagedAppendArgs*>(&a)};
  return cudaLaunchKernel(fn, dim3(a.b.n_tokens), dim3(kThreads), args, 0, s);
}

}  // namespace yb
