// Attention of a batch in which groups of sequences share a prefix: what the planning kernel (paged_shared.cu) leaves
// for the attention's kernels (paged_attn.cu).
#pragma once

#include "paged.cuh"
#include "paged_shared_axis.cuh"

namespace yb {

constexpr int kMaxGroups = 2048;

// How the axis is shared out (paged_axis.cuh).
struct SharedHead {
  unsigned long long total, share;
  int more;
};
struct SharedPlanArgs {
  PagedBatch b;
  const int* group_start;  // [n_groups + 1] sequences
  const int* prefix_len;   // [n_groups] slots
  int n_groups;
  Axis x;
  int grid;         // blocks of the attention
  int part_tokens;  // tokens that the workspace has room for two parts of
  SharedHead* head;
  SharedSeq* seqs;  // [n_groups + n_seqs]
};
cudaError_t paged_shared_plan(const SharedPlanArgs& a, cudaStream_t s);

__device__ __forceinline__ SharedSeq paged_seq(const SharedBatch& b, int v) {
  union {
    int4 w[sizeof(SharedSeq) / 16];
    SharedSeq q;
  } u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(SharedSeq) / 16; ++i) u.w[i] = __ldca(reinterpret_cast<const int4*>(b.seqs + v) + i);
  return u.q;
}

}  // namespace yb
