// C entry points of the paged KV cache: argument checks and launches.
#include "engine.h"
#include "paged.cuh"

#include <atomic>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <utility>

using namespace yb;

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// Shapes and NULLs, before any CUDA call.  *empty: nothing to do.
int check_batch(const yb_paged_batch* b, PagedBatch* out, bool* empty) {
  if (!b) return set_error(YB_E_INVALID, "null batch");
  if (b->dtype != YB_DTYPE_F16 && b->dtype != YB_DTYPE_BF16)
    return set_error(YB_E_UNSUPPORTED, "the paged cache holds fp16 or bf16 (dtype 1 or 2)");
  if (b->head_dim != 64 && b->head_dim != 128) return set_error(YB_E_UNSUPPORTED, "head_dim must be 64 or 128");
  if (b->n_heads <= 0 || b->n_kv_heads <= 0 || b->n_heads % b->n_kv_heads)
    return set_error(YB_E_INVALID, "n_heads must be a positive multiple of n_kv_heads");
  if (b->n_heads / b->n_kv_heads > 16 || b->n_heads > 1024)
    return set_error(YB_E_UNSUPPORTED, "at most 16 query heads per kv head and 1024 heads");
  int lg = 4;
  while (lg < 8 && (1 << lg) != b->page_size) ++lg;
  if ((1 << lg) != b->page_size) return set_error(YB_E_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
  if (b->n_seqs < 0 || b->n_tokens < 0 || b->n_pages <= 0 || b->max_pages <= 0)
    return set_error(YB_E_INVALID, "negative batch size or empty page pool");
  if (b->n_seqs > 65536 || b->n_tokens > (1 << 20) || ((long long)b->max_pages << lg) > (1 << 21))
    return set_error(YB_E_UNSUPPORTED, "at most 65536 sequences, 2^20 new tokens and 2^21 slots per sequence");
  if (((long long)b->n_pages * b->n_kv_heads << lg) > INT_MAX - 256)
    return set_error(YB_E_UNSUPPORTED, "the page pool has too many rows (n_pages * n_kv_heads * page_size)");
  *empty = b->n_seqs == 0 || b->n_tokens == 0;  // its buffers of no elements may be null
  if (!b->k_pages || !b->v_pages || (!*empty && (!b->q_start_dev || !b->kv_len_dev || !b->page_table_dev)))
    return set_error(YB_E_INVALID, "null buffer in the batch");
  if (!aligned16(b->k_pages) || !aligned16(b->v_pages))
    return set_error(YB_E_INVALID, "k_pages and v_pages must be 16-byte aligned");
  if (!aligned4(b->q_start_dev) || !aligned4(b->kv_len_dev) || !aligned4(b->page_table_dev))
    return set_error(YB_E_INVALID, "q_start_dev, kv_len_dev and page_table_dev must be 4-byte aligned");
  out->q_start = b->q_start_dev;
  out->kv_len = b->kv_len_dev;
  out->page_table = b->page_table_dev;
  out->n_seqs = b->n_seqs;
  out->n_tokens = b->n_tokens;
  out->n_heads = b->n_heads;
  out->n_kv_heads = b->n_kv_heads;
  out->n_pages = b->n_pages;
  out->max_pages = b->max_pages;
  out->ps_log2 = lg;
  return 0;
}

// Rows of `width` elements of `size` bytes, `stride` elements apart: 16-byte aligned, not overlapping.
int check_rows(const char* name, const void* p, long long stride, long long width, int size, bool empty) {
  if (!p && !empty) return set_error(YB_E_INVALID, std::string("null ") + name);
  if (!aligned16(p) || stride < width || stride > (1ll << 31) || stride * size % 16)
    return set_error(YB_E_INVALID, std::string(name) + ": rows must be 16-byte aligned and at least " +
                                       std::to_string(width) + " elements apart");
  return 0;
}

// Every buffer must be memory that the current device `dev` can read: a host pointer or another device's
// memory is refused here instead of faulting in the kernel.
int check_device(int dev, std::initializer_list<std::pair<const char*, const void*>> bufs) {
  for (const auto& b : bufs) {
    if (!b.second) continue;
    cudaPointerAttributes at;
    YB_CK(cudaPointerGetAttributes(&at, b.second));
    if (at.type != cudaMemoryTypeManaged && (at.type != cudaMemoryTypeDevice || at.device != dev))
      return set_error(YB_E_INVALID, std::string(b.first) + " is not memory of the current device");
  }
  return 0;
}

// SMs of a device, asked for once (148 without one, so that sizes can be computed anywhere)
int device_sms(int dev) {
  static std::atomic<int> known[64];
  if (dev >= 0 && dev < 64) {
    const int n = known[dev].load(std::memory_order_relaxed);
    if (n) return n;
  }
  int n = 0;
  if (dev < 0 || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
    cudaGetLastError();
    return 148;
  }
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// What one of the attention's blocks may have to walk is counted in 31 bits: the units (blocks of up to 2 * (128 /
// query heads per kv head) queries) of every sequence and kv head, with the key tiles of 128 slots of the longest cache
// and 3 more each, shared out over the blocks.
int check_share(const yb_paged_batch* b, const PagedBatch& p, int dev) {
  const long long queries = 2 * (128 / (b->n_heads / b->n_kv_heads));
  const long long units = b->n_tokens / queries + (b->n_seqs < b->n_tokens ? b->n_seqs : b->n_tokens);
  const long long tiles = (((long long)b->max_pages << p.ps_log2) >> 7) + 3;
  if (units * b->n_kv_heads * tiles / paged_attention_grid(device_sms(dev)) >= INT_MAX)
    return set_error(YB_E_UNSUPPORTED, "the batch may have too many slots to attend to on this device "
                                       "((n_tokens / queries of a unit + n_seqs) * n_kv_heads * max_pages * page_size)");
  return 0;
}

// The current device, or -1 where there is none (sizes can be asked for without one).
int current_device() {
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return -1;
  }
  return dev;
}

std::atomic<long long> wait_budget{kWaitBudgetCycles};

}  // namespace

extern "C" int yb_paged_append_dev(const yb_paged_batch* b, void* q_out, long long q_out_stride, const void* qkv,
                                   long long qkv_stride, int qkv_dtype, const float* q_norm_dev,
                                   const float* k_norm_dev, float eps, const float* inv_freq_dev, int rotary_dim,
                                   int rope_half, const int* pos_dev, float qkv_clip, void* stream) {
  PagedAppendArgs a{};
  bool empty = false;
  int rc = check_batch(b, &a.b, &empty);
  if (rc) return rc;
  if (qkv_dtype < 0 || qkv_dtype > 2) return set_error(YB_E_UNSUPPORTED, "qkv must be fp32, fp16 or bf16 (dtype 0, 1, 2)");
  const long long hd = b->head_dim;
  if ((rc = check_rows("q_out", q_out, q_out_stride, b->n_heads * hd, 2, empty))) return rc;
  if ((rc = check_rows("qkv", qkv, qkv_stride, (b->n_heads + 2ll * b->n_kv_heads) * hd, qkv_dtype ? 2 : 4, empty))) return rc;
  if (rotary_dim < 0 || rotary_dim > hd || rotary_dim % 2 || (rope_half && rotary_dim % 8))
    return set_error(YB_E_INVALID, "rotary_dim must be even and <= head_dim (a multiple of 8 for half-split pairs)");
  if (rotary_dim && !inv_freq_dev) return set_error(YB_E_INVALID, "null inv_freq_dev");
  if (!aligned4(q_norm_dev) || !aligned4(k_norm_dev) || !aligned4(inv_freq_dev) || !aligned4(pos_dev))
    return set_error(YB_E_INVALID, "q_norm_dev, k_norm_dev, inv_freq_dev and pos_dev must be 4-byte aligned");
  if (!(eps >= 0.f) || !(qkv_clip > 0.f)) return set_error(YB_E_INVALID, "eps must be >= 0 and qkv_clip > 0");
  if (empty) return 0;
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  rc = check_device(dev, {{"q_out", q_out}, {"qkv", qkv}, {"q_start_dev", b->q_start_dev}, {"kv_len_dev", b->kv_len_dev},
                     {"page_table_dev", b->page_table_dev}, {"k_pages", b->k_pages}, {"v_pages", b->v_pages},
                     {"q_norm_dev", q_norm_dev}, {"k_norm_dev", k_norm_dev}, {"inv_freq_dev", inv_freq_dev},
                     {"pos_dev", pos_dev}});
  if (rc) return rc;
  a.qkv = qkv;
  a.q_out = q_out;
  a.k_pages = b->k_pages;
  a.v_pages = b->v_pages;
  a.qkv_stride = qkv_stride;
  a.q_stride = q_out_stride;
  a.q_norm = q_norm_dev;
  a.k_norm = k_norm_dev;
  a.inv_freq = inv_freq_dev;
  a.pos = pos_dev;
  a.eps = eps;
  a.clip = qkv_clip;
  a.rotary_dim = rotary_dim;
  a.half = rope_half ? 1 : 0;
  YB_CK(paged_append(a, b->head_dim, qkv_dtype, b->dtype, device_sms(dev), static_cast<cudaStream_t>(stream)));
  return 0;
}

extern "C" size_t yb_paged_attention_scratch_bytes(const yb_paged_batch* b) {
  PagedBatch p;
  bool empty;
  if (check_batch(b, &p, &empty)) return 0;
  const int dev = current_device();
  if (check_share(b, p, dev)) return 0;
  return paged_attention_scratch(b->head_dim, device_sms(dev));
}

extern "C" int yb_paged_attention_wait_budget(long long clocks) {
  if (clocks < 0 || clocks > kWaitBudgetCycles) return set_error(YB_E_INVALID, "the wait budget must be 0 (the default) to " +
                                                                                   std::to_string(kWaitBudgetCycles) + " clocks");
  wait_budget.store(clocks ? clocks : kWaitBudgetCycles, std::memory_order_relaxed);
  return 0;
}

extern "C" int yb_paged_attention_dev(const yb_paged_batch* b, void* out, long long out_stride, const void* q,
                                      long long q_stride, float scale, int window, void* scratch_dev, void* stream) {
  PagedAttnArgs a{};
  bool empty = false;
  int rc = check_batch(b, &a.b, &empty);
  if (rc) return rc;
  const long long width = (long long)b->n_heads * b->head_dim;
  if ((rc = check_rows("out", out, out_stride, width, 2, empty)) || (rc = check_rows("q", q, q_stride, width, 2, empty))) return rc;
  if (!(scale > 0.f) || !std::isfinite(scale * 1.4426950408889634f))
    return set_error(YB_E_INVALID, "scale must be positive, and scale * log2(e) finite");
  if (window < 0) return set_error(YB_E_INVALID, "negative window");
  if (!scratch_dev || !aligned16(scratch_dev)) return set_error(YB_E_INVALID, "scratch_dev must be 16-byte aligned memory");
  if (empty) return 0;
  if ((rc = check_share(b, a.b, current_device()))) return rc;
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  rc = check_device(dev, {{"out", out}, {"q", q}, {"q_start_dev", b->q_start_dev}, {"kv_len_dev", b->kv_len_dev},
                     {"page_table_dev", b->page_table_dev}, {"k_pages", b->k_pages}, {"v_pages", b->v_pages},
                     {"scratch_dev", scratch_dev}});
  if (rc) return rc;
  a.q = q;
  a.out = out;
  a.k_pages = b->k_pages;
  a.v_pages = b->v_pages;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.scale = scale;
  a.window = window ? window : INT_MAX;
  a.scratch = scratch_dev;
  a.wait_budget = wait_budget.load(std::memory_order_relaxed);
  YB_CK(paged_attention(a, b->head_dim, b->dtype, dev, device_sms(dev), static_cast<cudaStream_t>(stream)));
  return 0;
}
