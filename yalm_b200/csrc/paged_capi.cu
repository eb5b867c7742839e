// C entry points of the paged KV cache: argument checks and launches.
#include "checks.h"
#include "engine.h"
#include "paged_shared.cuh"

#include <atomic>
#include <climits>
#include <cmath>

using namespace yb;

namespace {

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

// What one of the attention's blocks may have to walk is counted in 31 bits: the units (blocks of up to 2 * (128 /
// query heads per kv head) queries) of every sequence and kv head, with the key tiles of 128 slots of the longest cache
// and 3 more each, shared out over the blocks.
// With `groups` > 0 shared prefixes, which are units of their own, two kernels share the blocks' SMs, by a choice (paged_shared.cu)
// that lets neither take longer than half of the SMs would.  At its rates of 2.2 us a key tile and 0.08 us a step of few rows
// (16 slots, 12 warps a block) a block then has up to twice this count of tiles, a warp up to 4.5 times as many steps.
int check_share(const yb_paged_batch* b, const PagedBatch& p, int dev, int groups = 0) {
  const long long queries = 2 * (128 / (b->n_heads / b->n_kv_heads));
  long long units = b->n_tokens / queries + (b->n_seqs < b->n_tokens ? b->n_seqs : b->n_tokens);
  if (groups) units += b->n_tokens / queries + groups;
  const long long tiles = (((long long)b->max_pages << p.ps_log2) >> 7) + 3;
  if (units * b->n_kv_heads * tiles / paged_attention_grid(device_sms(dev)) >= (groups ? INT_MAX / 5 : INT_MAX))
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

extern "C" int yb_paged_plan_dev(const yb_paged_batch* b, const int* new_len_dev, const int* kv_before_dev,
                                 const int* kept_dev, int* free_pages_dev, const int* n_free_before_dev,
                                 int* n_free_dev, int* pos_dev, long long* slots_dev, int* status_dev, void* stream) {
  PagedBatch p;
  bool empty = false;
  int rc = check_batch(b, &p, &empty);
  if (rc) return rc;
  if (!b->q_start_dev || !free_pages_dev || !n_free_before_dev || !n_free_dev || !status_dev ||
      (b->n_seqs && (!b->kv_len_dev || !b->page_table_dev || !new_len_dev || !kv_before_dev)))
    return set_error(YB_E_INVALID, "null buffer of the plan");
  for (const void* v : {(const void*)b->q_start_dev, (const void*)b->kv_len_dev, (const void*)b->page_table_dev,
                        (const void*)new_len_dev, (const void*)kv_before_dev, (const void*)kept_dev,
                        (const void*)free_pages_dev, (const void*)n_free_before_dev, (const void*)n_free_dev,
                        (const void*)pos_dev, (const void*)status_dev})
    if (!aligned4(v)) return set_error(YB_E_INVALID, "the plan's buffers of ints must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(slots_dev) & 7) return set_error(YB_E_INVALID, "slots_dev must be 8-byte aligned");
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  rc = check_device(dev, {{"q_start_dev", b->q_start_dev}, {"kv_len_dev", b->kv_len_dev},
                          {"page_table_dev", b->page_table_dev}, {"new_len_dev", new_len_dev},
                          {"kv_before_dev", kv_before_dev}, {"kept_dev", kept_dev}, {"free_pages_dev", free_pages_dev},
                          {"n_free_before_dev", n_free_before_dev}, {"n_free_dev", n_free_dev}, {"pos_dev", pos_dev},
                          {"slots_dev", slots_dev}, {"status_dev", status_dev}});
  if (rc) return rc;
  PagedPlanArgs a{};
  a.new_len = new_len_dev;
  a.kv_before = kv_before_dev;
  a.kept = kept_dev;
  a.n_free_before = n_free_before_dev;
  a.q_start = const_cast<int*>(b->q_start_dev);
  a.kv_len = const_cast<int*>(b->kv_len_dev);
  a.page_table = const_cast<int*>(b->page_table_dev);
  a.free_pages = free_pages_dev;
  a.n_free = n_free_dev;
  a.pos = pos_dev;
  a.slots = slots_dev;
  a.status = status_dev;
  a.n_seqs = b->n_seqs;
  a.n_tokens = b->n_tokens;
  a.n_pages = b->n_pages;
  a.max_pages = b->max_pages;
  a.ps_log2 = p.ps_log2;
  YB_CK(paged_plan(a, dev, static_cast<cudaStream_t>(stream)));
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

// What both forms of the attention check before any CUDA call; fills in what they have in common.
static int check_attention(const yb_paged_batch* b, PagedAttnArgs* a, bool* empty, void* out, long long out_stride,
                           const void* q, long long q_stride, float scale, void* scratch_dev) {
  int rc = check_batch(b, &a->b, empty);
  if (rc) return rc;
  const long long width = (long long)b->n_heads * b->head_dim;
  if ((rc = check_rows("out", out, out_stride, width, 2, *empty)) || (rc = check_rows("q", q, q_stride, width, 2, *empty))) return rc;
  if (!(scale > 0.f) || !std::isfinite(scale * 1.4426950408889634f))
    return set_error(YB_E_INVALID, "scale must be positive, and scale * log2(e) finite");
  if (!scratch_dev || !aligned16(scratch_dev)) return set_error(YB_E_INVALID, "scratch_dev must be 16-byte aligned memory");
  a->q = q;
  a->out = out;
  a->k_pages = b->k_pages;
  a->v_pages = b->v_pages;
  a->q_stride = q_stride;
  a->out_stride = out_stride;
  a->scale = scale;
  a->scratch = scratch_dev;
  a->wait_budget = wait_budget.load(std::memory_order_relaxed);
  return 0;
}
static int check_attention_device(int dev, const yb_paged_batch* b, const void* out, const void* q, const void* scratch_dev) {
  return check_device(dev, {{"out", out}, {"q", q}, {"q_start_dev", b->q_start_dev}, {"kv_len_dev", b->kv_len_dev},
                     {"page_table_dev", b->page_table_dev}, {"k_pages", b->k_pages}, {"v_pages", b->v_pages},
                     {"scratch_dev", scratch_dev}});
}

extern "C" int yb_paged_attention_dev(const yb_paged_batch* b, void* out, long long out_stride, const void* q,
                                      long long q_stride, float scale, int window, void* scratch_dev, void* stream) {
  PagedAttnArgs a{};
  bool empty = false;
  int rc = check_attention(b, &a, &empty, out, out_stride, q, q_stride, scale, scratch_dev);
  if (rc) return rc;
  if (window < 0) return set_error(YB_E_INVALID, "negative window");
  if (empty) return 0;
  if ((rc = check_share(b, a.b, current_device()))) return rc;
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  if ((rc = check_attention_device(dev, b, out, q, scratch_dev))) return rc;
  a.window = window ? window : INT_MAX;
  YB_CK(paged_attention(a, b->head_dim, b->dtype, dev, device_sms(dev), static_cast<cudaStream_t>(stream)));
  return 0;
}

static int check_groups(int n_groups) {
  if (n_groups < 0) return set_error(YB_E_INVALID, "negative n_groups");
  if (n_groups > kMaxGroups) return set_error(YB_E_UNSUPPORTED, "at most 2048 groups with a shared prefix");
  return 0;
}

extern "C" size_t yb_paged_attention_shared_scratch_bytes(const yb_paged_batch* b, int n_groups) {
  PagedBatch p;
  bool empty;
  if (check_batch(b, &p, &empty) || check_groups(n_groups)) return 0;
  const int dev = current_device();
  if (check_share(b, p, dev, n_groups)) return 0;
  return paged_shared_scratch(p, n_groups, b->head_dim, device_sms(dev));
}

extern "C" int yb_paged_attention_shared_dev(const yb_paged_batch* b, int n_groups, const int* group_start_dev,
                                             const int* prefix_len_dev, void* out, long long out_stride, const void* q,
                                             long long q_stride, float scale, void* scratch_dev, void* stream) {
  int rc = check_groups(n_groups);
  if (rc) return rc;
  if (n_groups && (!group_start_dev || !prefix_len_dev || !aligned4(group_start_dev) || !aligned4(prefix_len_dev)))
    return set_error(YB_E_INVALID, "group_start_dev and prefix_len_dev must be 4-byte aligned buffers");
  if (n_groups == 0)
    return yb_paged_attention_dev(b, out, out_stride, q, q_stride, scale, 0, scratch_dev, stream);
  PagedAttnArgs a{};
  bool empty = false;
  if ((rc = check_attention(b, &a, &empty, out, out_stride, q, q_stride, scale, scratch_dev))) return rc;
  if (empty) return 0;
  // Where reading a prefix once can save no more than 64 MB (every sequence's whole table but one), the kernels for it
  // cost more than they save.  32 heads of 128 on 8 kv heads, prefix of 4096 and 100 own slots: 4 sequences (50
  // MB) 19.4 us without, 32.9 with; 8 (117 MB) 27.1 and 31.3; 16 (252 MB) 42.9 and 31.5.  8 heads of 64 on 2: 32 (65 MB)
  // 24.3 and 25.2, 64 (132 MB) 37.7 and 25.3.  (Of tables as wide as the sequences: a wider one counts for more than can be
  // saved; with 32768 slots the 4 take 29.5 us.)
  const bool apart = (b->n_seqs - 1.0) * b->max_pages * b->page_size * b->n_kv_heads * b->head_dim * 4.0 >= 64e6;
  if ((rc = check_share(b, a.b, current_device(), apart ? n_groups : 0))) return rc;
  int dev = 0;
  YB_CK(cudaGetDevice(&dev));
  if ((rc = check_attention_device(dev, b, out, q, scratch_dev)) ||
      (rc = check_device(dev, {{"group_start_dev", group_start_dev}, {"prefix_len_dev", prefix_len_dev}})))
    return rc;
  a.window = INT_MAX;
  a.group_start = group_start_dev;
  a.prefix_len = prefix_len_dev;
  a.n_groups = n_groups;
  a.n_sms = device_sms(dev);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  YB_CK(apart ? paged_attention_shared(a, b->head_dim, b->dtype, dev, s)
              : paged_attention(a, b->head_dim, b->dtype, dev, a.n_sms, s));
  return 0;
}
