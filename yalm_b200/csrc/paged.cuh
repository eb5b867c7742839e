// The paged KV cache of a batch of sequences: append (norm, rotation, store) and attention
// (paged_append.cu, paged_attn.cu; entry points in paged_capi.cu).
#pragma once

#include <cuda_runtime.h>
#include <atomic>
#include <cstddef>
#include <cstdint>

#include "common.cuh"

namespace yb {

// Raises a kernel's dynamic shared-memory cap, once per device.
struct SmemCap {
  std::atomic<unsigned long long> done{0};  // devices, by bit
  cudaError_t raise(const void* fn, int device, size_t bytes) {
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

// The batch as the kernels see it (include/yalm_b200.h, yb_paged_batch).  The lengths and the table are
// read on the device, so a captured launch follows them; every index made from them is clamped to
// the buffers' bounds here, whatever they hold.  What the caller may have written just before is read by ordinary
// loads (__ldca), after griddepcontrol.wait: the kernels may be resident while the one before them still writes, and
// non-coherent loads (__ldg) are for what stays as it is as long as a kernel lives.
struct PagedBatch {
  const int* q_start;     // [n_seqs + 1] first row of each sequence's new tokens
  const int* kv_len;      // [n_seqs] slots in the sequence's cache, the new tokens among them
  const int* page_table;  // [n_seqs][max_pages]
  int n_seqs, n_tokens;
  int n_heads, n_kv_heads;
  int n_pages, max_pages;
  int ps_log2;  // log2 of the page size
};

// A sequence's rows and slots: its new tokens are rows [row0, row0 + n), its cache holds slots
// [0, kv); new token i has slot kv - n + i (negative where kv_len is below the token count).
struct PagedSeq {
  int row0, n, kv;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedBatch& b, int s) {
  PagedSeq r;
  r.row0 = min(max(__ldca(b.q_start + s), 0), b.n_tokens);
  r.n = min(max(__ldca(b.q_start + s + 1), r.row0), b.n_tokens) - r.row0;
  r.kv = min(max(__ldca(b.kv_len + s), 0), b.max_pages << b.ps_log2);
  return r;
}

// The sequence whose rows hold `row` (the last s with q_start[s] <= row), or -1 when the row lies
// before the first or behind the last sequence.  Called by a whole warp.
__device__ __forceinline__ int paged_find_seq(const PagedBatch& b, int row) {
  // invariant: q_start[lo] <= row (lo = -1: nothing known), q_start[hi] > row (hi = n_seqs + 1: past the end)
  int lo = -1, hi = b.n_seqs + 1;
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;  // 32 probes, ascending
    const bool le = at < hi && __ldca(b.q_start + at) <= row;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    const int nlo = lo + c * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  return lo >= 0 && lo < b.n_seqs ? lo : -1;
}

struct PagedAppendArgs {
  PagedBatch b;
  const void* qkv;     // [n_tokens][(n_heads + 2 n_kv_heads) head_dim], rows qkv_stride elements apart
  void* q_out;         // [n_tokens][n_heads * head_dim], rows q_stride elements apart
  void* k_pages;       // [n_pages][n_kv_heads][page size][head_dim]
  void* v_pages;
  long long qkv_stride, q_stride;
  const float* q_norm;  // [head_dim] or null
  const float* k_norm;
  const float* inv_freq;  // [rotary_dim / 2]
  const int* pos;         // [n_tokens] rotary positions, or null: the slots
  float eps, clip;
  int rotary_dim;
  int half;  // pairs (j, j + rotary_dim / 2) instead of (2j, 2j + 1)
};
// src_type: element type of qkv, type: of q_out and the caches (0 fp32, 1 fp16, 2 bf16)
cudaError_t paged_append(const PagedAppendArgs& a, int head_dim, int src_type, int type, int n_sms, cudaStream_t s);

struct PagedAttnArgs {
  PagedBatch b;
  const void* q;  // [n_tokens][n_heads * head_dim], rows q_stride elements apart
  void* out;      // the same shape, rows out_stride elements apart
  const void* k_pages;
  const void* v_pages;
  long long q_stride, out_stride;
  float scale;
  int window;  // slots a token sees, itself counted; INT_MAX: all of them
  long long wait_budget;  // clocks after which a wait in the kernel gives up
  void* scratch;
};
int paged_attention_grid(int n_sms);  // blocks
size_t paged_attention_scratch(int head_dim, int n_sms);
cudaError_t paged_attention(const PagedAttnArgs& a, int head_dim, int type, int device, int n_sms, cudaStream_t s);

}  // namespace yb
