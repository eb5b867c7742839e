// C entry point of the sampler for rows of logits: argument checks and launch.
#include "checks.h"
#include "engine.h"
#include "sample_rows.cuh"

using namespace yb;

extern "C" int yb_sample_rows_dev(int* tokens_dev, float* prob_dev, const void* logits, long long logits_stride,
                                  int dtype, int rows, int vocab, const float* coin_dev, const float* temperature_dev,
                                  const int* top_k_dev, const float* top_p_dev, const float* min_p_dev, void* stream) {
  if (dtype < 0 || dtype > 2) return set_error(YB_E_UNSUPPORTED, "logits must be fp32, fp16 or bf16 (dtype 0, 1, 2)");
  if (rows < 0 || vocab <= 0) return set_error(YB_E_INVALID, "negative rows or empty vocabulary");
  if (rows > 65536 || vocab > kSampleMaxVocab) return set_error(YB_E_UNSUPPORTED, "at most 65536 rows of 2^20 logits");
  if (rows > 1 && (logits_stride < vocab || logits_stride > (1ll << 31)))
    return set_error(YB_E_INVALID, "logits_stride must be from vocab to 2^31");
  if (rows == 0) return 0;
  if (!tokens_dev || !logits || !coin_dev) return set_error(YB_E_INVALID, "null tokens_dev, logits or coin_dev");
  if (reinterpret_cast<uintptr_t>(logits) & (dtype ? 1 : 3)) return set_error(YB_E_INVALID, "logits must be aligned to their type");
  for (const void* v : {(const void*)tokens_dev, (const void*)prob_dev, (const void*)coin_dev,
                        (const void*)temperature_dev, (const void*)top_k_dev, (const void*)top_p_dev, (const void*)min_p_dev})
    if (!aligned4(v)) return set_error(YB_E_INVALID, "the rows' buffers must be 4-byte aligned");
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  const int rc = check_device(dev, {{"tokens_dev", tokens_dev}, {"prob_dev", prob_dev}, {"logits", logits},
                                    {"coin_dev", coin_dev}, {"temperature_dev", temperature_dev},
                                    {"top_k_dev", top_k_dev}, {"top_p_dev", top_p_dev}, {"min_p_dev", min_p_dev}});
  if (rc) return rc;
  SampleRowsArgs a{};
  a.tokens = tokens_dev;
  a.prob = prob_dev;
  a.logits = logits;
  a.stride = rows > 1 ? logits_stride : 0;
  a.rows = rows;
  a.vocab = vocab;
  a.coin = coin_dev;
  a.temperature = temperature_dev;
  a.top_k = top_k_dev;
  a.top_p = top_p_dev;
  a.min_p = min_p_dev;
  YB_CK(sample_rows(a, dtype, dev, device_sms(dev), static_cast<cudaStream_t>(stream)));
  return 0;
}
