// Attention of a batch in which groups of sequences share a prefix: what the planning kernel (paged_shared.cu) leaves
// for the attention's kernels (paged_attn.cu).
#pragma once

#include "paged.cuh"
#include "paged_shared_axis.cuh"

namespace yb {

constexpr int kMaxGroups = 2048;

// How the axes are shared out (paged_axis.cuh): the first one among the first `blocks` blocks of its kernel, that of few
// rows among the warps of the first grid - blocks blocks of its own, so that both run at the same time.
struct SharedHead {
  unsigned long long total, share;
  unsigned long long few_total, few_share;
  int more, few_more;
};
struct SharedPlanArgs {
  PagedBatch b;
  const int* group_start;  // [n_groups + 1] sequences
  const int* prefix_len;   // [n_groups] slots
  int n_groups, head_dim;
  Axis x;
  int grid;         // SMs, and blocks of either kernel
  int part_tokens;  // tokens that the workspace has room for two parts of
  SharedHead* head;
  SharedSeq* seqs;  // [n_groups + n_seqs]
};
cudaError_t paged_shared_plan(const SharedPlanArgs& a, cudaStream_t s);

// ---- sequences of few rows (paged_few.cu)
constexpr int kFewThreads = 384, kFewWarps = kFewThreads / 32;  // one block an SM
constexpr __host__ __device__ int few_stages(int head_dim) { return head_dim == 128 ? 2 : 4; }
// A warp's records: 0 for a unit begun by an earlier warp, 1 for the one it leaves to later ones.  A row is o [head_dim],
// m, l and two floats for alignment.
inline __host__ __device__ size_t few_row_floats(int head_dim) { return (size_t)head_dim + 4; }
struct PagedFewArgs {
  PagedBatch b;
  SharedBatch shared;
  const SharedHead* head;
  const void* q;
  void* out;
  const void* k_pages;
  const void* v_pages;
  long long q_stride, out_stride;
  int K, gq;
  float c;       // scale * log2(e)
  float* recs;   // [warps][2][kFewRows] rows
  float* parts;  // [tokens with a part][n_heads] rows
  unsigned* status;
  long long wait_budget;
};
cudaError_t paged_few(const PagedFewArgs& a, int head_dim, int type, int device, int grid, cudaStream_t s);

// (from L2: the attention kernel starts while the one before it, which waits for the plan, still runs)
__device__ __forceinline__ SharedSeq paged_seq(const SharedBatch& b, int v) {
  union {
    int4 w[sizeof(SharedSeq) / 16];
    SharedSeq q;
  } u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(SharedSeq) / 16; ++i) u.w[i] = __ldcg(reinterpret_cast<const int4*>(b.seqs + v) + i);
  return u.q;
}

}  // namespace yb
