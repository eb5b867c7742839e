// A token for every row of logits (sample_rows.cu).
#pragma once

#include <cuda_runtime.h>

namespace yb {

constexpr int kSampleMaxVocab = 1 << 20;

struct SampleRowsArgs {
  int* tokens;         // [rows]
  float* prob;         // [rows] or null
  const void* logits;  // [rows][vocab], rows stride elements apart
  long long stride;
  int rows, vocab;
  const float* coin;         // [rows]
  const float* temperature;  // [rows] or null: 1
  const int* top_k;          // [rows] or null: no limit; and so on
  const float* top_p;
  const float* min_p;
};
// type: of the logits, 0 fp32, 1 fp16, 2 bf16
cudaError_t sample_rows(const SampleRowsArgs& a, int type, int device, int n_sms, cudaStream_t s);

}  // namespace yb
