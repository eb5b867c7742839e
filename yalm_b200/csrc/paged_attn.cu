// Attention of a batch's new tokens over the paged KV cache, the simplest form: a warp per (row, head),
// one key at a time, online softmax.
#include "paged.cuh"

#include <cuda_bf16.h>

#include <math.h>

namespace yb {

namespace {

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <int HD, typename T>
__global__ void __launch_bounds__(128) paged_attn_kernel(const PagedAttnArgs a) {
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.b.n_heads) return;
  const int seq = paged_find_seq(a.b, row);
  if (seq < 0) return;
  const PagedSeq sq = paged_seq(a.b, seq);
  if (row - sq.row0 >= sq.n) return;
  const int p = sq.kv - sq.n + row - sq.row0;
  const int g = h / (a.b.n_heads / a.b.n_kv_heads);
  constexpr int V = HD / 32;
  const T* qp = static_cast<const T*>(a.q) + (size_t)row * a.q_stride + (size_t)h * HD;
  float q[V], o[V], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) q[i] = to_f(qp[lane + 32 * i]) * a.scale, o[i] = 0.f;
  const int t0 = p >= a.window ? p - a.window + 1 : 0;
  const int mask = (1 << a.b.ps_log2) - 1;
  for (int t = t0; t <= p; ++t) {
    const int page = __ldg(a.b.page_table + (size_t)seq * a.b.max_pages + (t >> a.b.ps_log2));
    if (page < 0 || page >= a.b.n_pages) continue;
    const size_t at = ((((size_t)page * a.b.n_kv_heads + g) << a.b.ps_log2) + (t & mask)) * HD;
    const T* k = static_cast<const T*>(a.k_pages) + at;
    const T* v = static_cast<const T*>(a.v_pages) + at;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) s += q[i] * to_f(k[lane + 32 * i]);
    s = warp_sum(s);
    const float mn = fmaxf(m, s), c = expf(m - mn), w = expf(s - mn);
    l = l * c + w;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = o[i] * c + w * to_f(v[lane + 32 * i]);
    m = mn;
  }
  T* out = static_cast<T*>(a.out) + (size_t)row * a.out_stride + (size_t)h * HD;
#pragma unroll
  for (int i = 0; i < V; ++i) put(out + lane + 32 * i, l > 0.f ? o[i] / l : 0.f);
}

}  // namespace

size_t paged_attention_scratch(int head_dim, int n_sms) { return 256; }

cudaError_t paged_attention(const PagedAttnArgs& a, int head_dim, int type, cudaStream_t s) {
  const void* fn = head_dim == 128 ? (type == 1 ? reinterpret_cast<const void*>(&paged_attn_kernel<128, __half>)
                                                : reinterpret_cast<const void*>(&paged_attn_kernel<128, __nv_bfloat16>))
                                   : (type == 1 ? reinterpret_cast<const void*>(&paged_attn_kernel<64, __half>)
                                                : reinterpret_cast<const void*>(&paged_attn_kernel<64, __nv_bfloat16>));
  void* args[] = {const_cast<PagedAttnArgs*>(&a)};
  return cudaLaunchKernel(fn, dim3(a.b.n_tokens, (a.b.n_heads + 3) / 4), dim3(128), args, 0, s);
}

}  // namespace yb
