// Attention of sequences with few rows (up to 8: tokens x query heads of a kv head) over the paged cache, for batches
// with shared prefixes, whose sequences' own slots are mostly few (paged_attn.cu has the prefixes and longer chunks).
//
// What bounds it is the cache's bytes, if starts and ends of many short units cost little: the tensor-core path pays
// 4000 to 5500 clocks of a block for them, which for 3 tiles of own slots is as much as their bytes take.  Here a warp
// works by itself: steps of 16 slots (of one page), whose K and V, 4 KB each for heads of 128, come by a bulk copy into a
// ring of its own, also across units; and from there straight into the operands of mma.m16n8k16, for which the order of
// the dimensions inside a product is chosen so that every lane loads 16 bytes at a time:
//   S^T = K . Q^T   slots x rows; the product over dims takes dims 32c + 8q .. + 7 of lane q's chunk in any order, if K
//                   and Q have the same one
//   O^T += V^T . P^T  dims x rows; P^T is S^T's transpose in registers (movmatrix), V's operand pairs two slots of a
//                   dimension, by byte permutes of two rows' chunks
// Units (sequence, kv head) in order make an axis of steps that warps share out evenly; a unit that is cut leaves
// records, which the join puts together (paged_attn.cu).  It takes as many SMs as the plan gives it, and the tensor-core
// kernel, which is started under it, has the others.  Weights are rounded to the caches' type as there, fp16 with a
// factor 2^7; the rest is fp32.
#include <cuda_bf16.h>

#include <math.h>
#include <type_traits>

#include "launch.h"
#include "paged_shared.cuh"

namespace yb {

namespace {

typedef unsigned long long u64;

// Steps in a sum of the tensor cores: of values of one sign it loses 2^-24 of itself a step, on average over its growth (sums
// of 1024 were 6e-5 too small, a quarter of an fp16 rounding).
constexpr int kFewSum = 256;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Waits for a copy; false, and told, when the clocks have run out.  (Less than the default: without try_wait, which may
// suspend a warp for longer.)
__device__ __forceinline__ bool landed(uint64_t* bar, unsigned parity, long long clocks, unsigned* status) {
  if (mbar_test_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!(clocks < kWaitBudgetCycles ? mbar_test_wait(bar, parity) : mbar_try_wait(bar, parity)))
    if (clock64() - t0 > clocks) {
      atomicOr(status, kStatusMbarTimeout);
      return false;
    }
  return true;
}
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint4 zero4() { return make_uint4(0u, 0u, 0u, 0u); }

template <int HD, typename T>
__global__ void __launch_bounds__(kFewThreads, 1) paged_few_kernel(const __grid_constant__ PagedFewArgs a) {
  constexpr int kC = HD / 32, kJ = HD / 64;  // chunks of 32 dims of K, of 64 of V
  constexpr float kBias = std::is_same<T, __half>::value ? 7.f : 0.f;
  const PagedBatch& b = a.b;
  const int lane = threadIdx.x & 31, g = lane >> 2, q4 = lane & 3;
  const int warp = blockIdx.x * kFewWarps + (threadIdx.x >> 5);
  pdl_wait();
  pdl_trigger();  // the attention kernel beside this one needs no more than the plan, which is there
  // (the search's first round is on its way beside the head)
  const int step0 = (a.shared.n_seqs + 31) / 32, at0 = (lane + 1) * step0;
  const u64 probe0 = at0 < a.shared.n_seqs ? __ldca(&a.shared.seqs[at0].few_begin) : ~0ull;
  const u64 total = __ldca(&a.head->few_total), share = __ldca(&a.head->few_share);
  const int more = __ldca(&a.head->few_more);
  const u64 begin = block_begin(share, more, warp);
  if (begin >= total) return;
  int left = (int)min(share + (warp < more ? 1 : 0), total - begin);
  // the last sequence that begins at or before this warp's part: those without rows here that begin there come earlier
  int seq = __popc(__ballot_sync(0xffffffffu, probe0 <= begin)) * step0;
  for (int hi = min(a.shared.n_seqs, seq + step0); hi - seq > 1;) {
    const int step = (hi - seq + 31) / 32, at = seq + (lane + 1) * step;
    const int n = __popc(__ballot_sync(0xffffffffu, at < hi && __ldca(&a.shared.seqs[at].few_begin) <= begin));
    seq += n * step;
    hi = min(hi, seq + step);
  }
  SharedSeq sq = paged_seq(a.shared, seq);
  int head, off;
  {
    const unsigned length = few_length(sq);
    const u64 rem = begin - sq.few_begin;
    head = (int)quot(rem, length);
    off = (int)(rem - (u64)head * length);
  }
  const int ps = 1 << b.ps_log2;
  // ---- this warp's ring
  constexpr int kStages = few_stages(HD);
  constexpr uint32_t kBytes = kFewSlots * HD * 2;  // of K, and of V
  extern __shared__ __align__(128) unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t s_bars[kFewWarps][kStages];
  const int w = threadIdx.x >> 5;
  const uint32_t ring = smem_u32(smem_raw) + (uint32_t)w * kStages * 2 * kBytes, bars = smem_u32(&s_bars[w][0]);
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init_s(bars + 8 * i, 1);
    mbar_fence_init();
  }
  __syncwarp();
  // The steps of this warp's part in order, copied kStages ahead of those that are worked on.  A wait that runs out ends
  // the warp, once what it has under way has landed.
  struct {
    SharedSeq sq;
    int seq, head, off, left, pages;  // pages: lane i has that of step t with t % 32 == i
    unsigned count, there;            // steps issued; by count % 32, whether the page is there
    bool fresh;
  } ahead{sq, seq, head, off, left, -1, 0, 0, true};
  unsigned done = 0;  // steps worked on
  bool dead = false;
  auto issue = [&] {
    for (;;) {
      if (ahead.left <= 0) return;
      const int steps = few_steps(ahead.sq);
      if (ahead.off < steps) break;
      ahead.left -= steps + kFewUnit - ahead.off;
      if (ahead.left <= 0) return;
      ahead.off = 0;
      ahead.fresh = true;
      if (++ahead.head >= a.K) {
        ahead.head = 0;
        do {
          if (++ahead.seq >= a.shared.n_seqs) {
            ahead.left = 0;
            return;
          }
          ahead.sq = paged_seq(a.shared, ahead.seq);
        } while (ahead.sq.few <= 0);
      }
    }
    const int t = ahead.off, slot = ahead.sq.lo * kKT + t * kFewSlots;
    if (ahead.fresh || (t & 31) == 0) {
      const int at = ahead.sq.lo * kKT + ((t & ~31) + lane) * kFewSlots;
      ahead.pages = at < ahead.sq.kv ? __ldca(b.page_table + (size_t)ahead.sq.table * b.max_pages + (at >> b.ps_log2)) : -1;
      ahead.fresh = false;
    }
    const int page = __shfl_sync(0xffffffffu, ahead.pages, t & 31);
    const bool ok = page >= 0 && page < b.n_pages;
    const unsigned bit = 1u << (ahead.count & 31);
    ahead.there = ok ? ahead.there | bit : ahead.there & ~bit;
    if (ok && lane == 0) {
      const int stage = ahead.count % kStages;
      const size_t from = (((size_t)page * a.K + ahead.head) * ps + (slot & (ps - 1))) * HD;
      const uint32_t to = ring + stage * 2 * kBytes, bar = bars + 8 * stage;
      mbar_arrive_expect_tx_s(bar, 2 * kBytes);
      bulk_g2s_nohint_s(to, static_cast<const T*>(a.k_pages) + from, kBytes, bar);
      bulk_g2s_nohint_s(to + kBytes, static_cast<const T*>(a.v_pages) + from, kBytes, bar);
    }
    ++ahead.count;
    ++ahead.off;
    --ahead.left;
  };
  unsigned phases = 0;  // by stage, the parity that its next copy completes
#pragma unroll
  for (int i = 0; i < kStages; ++i) issue();
  for (;;) {
    // ---- a piece: steps [t0, t1) of the unit
    const int steps = few_steps(sq), length = steps + kFewUnit, t0 = off, t1 = min(steps, off + left);
    if (t0 < t1) {
      const int rows = sq.few * a.gq;  // row r: token r / gq, head r % gq
      const T* qrow = static_cast<const T*>(a.q);
      uint4 qf[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        qf[c] = zero4();
        if (g < rows)
          qf[c] = __ldca(reinterpret_cast<const uint4*>(qrow + (size_t)(sq.row0 + g / a.gq) * a.q_stride +
                                                        (size_t)(head * a.gq + g % a.gq) * HD + 32 * c + 8 * q4));
      }
      // the slots that rows 2 q4 and 2 q4 + 1 see end here
      const int last0 = sq.kv - sq.few + (2 * q4) / a.gq + 1, last1 = sq.kv - sq.few + (2 * q4 + 1) / a.gq + 1;
      const int slot_lo = sq.lo * kKT;
      // The tensor cores' additions cut off what does not fit: a sum of theirs ends after kFewSum of them, and is joined
      // to those before in fp32 (paged_axis.cuh, kSumTiles).
      float had_m[2], had_l[2];  // of those before, whose o this lane has left in the record
      for (int u0 = t0, u1; u0 < t1; u0 = u1) {
        u1 = min(t1, u0 + kFewSum);
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        float o[2 * kC][4];  // o[4 j + i]: dims 64 j + 8 g + 2 i, + 1 of rows 2 q4, 2 q4 + 1
#pragma unroll
        for (int i = 0; i < 2 * kC; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        for (int t = u0; t < u1; ++t) {
          const int slot = slot_lo + t * kFewSlots;
          const int stage = done % kStages;
          const bool here = (ahead.there >> (done & 31)) & 1u;
          ++done;
          if (!here) {
            issue();
            continue;
          }
          if (!__all_sync(0xffffffffu, landed(&s_bars[w][stage], (phases >> stage) & 1u, a.wait_budget, a.status))) {
            dead = true;
            break;
          }
          phases ^= 1u << stage;
          const uint32_t kv = ring + stage * 2 * kBytes, kat = kv + g * (HD * 2) + q4 * 16, vat = kv + kBytes + q4 * (HD * 4) + g * 16;
          float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < kC; ++c) {
            const uint4 k0 = lds16(kat + 64 * c), k1 = lds16(kat + 8 * HD * 2 + 64 * c);
            mma<T>(s, k0.x, k1.x, k0.y, k1.y, qf[c].x, qf[c].y);
            mma<T>(s2, k0.z, k1.z, k0.w, k1.w, qf[c].z, qf[c].w);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) s[k] += s2[k];
          if (slot + kFewSlots > sq.kv - sq.few) {  // an edge
            const int at = slot + g;
            if (at >= last0) s[0] = -INFINITY;
            if (at >= last1) s[1] = -INFINITY;
            if (at + 8 >= last0) s[2] = -INFINITY;
            if (at + 8 >= last1) s[3] = -INFINITY;
          }
          float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
          }
          const float n0 = fmaxf(m0, x0 * a.c), n1 = fmaxf(m1, x1 * a.c);
          const float f0 = n0 == -INFINITY ? 0.f : n0 - kBias, f1 = n1 == -INFINITY ? 0.f : n1 - kBias;
          if (__any_sync(0xffffffffu, n0 > m0 || n1 > m1)) {
            const float r0 = m0 == -INFINITY ? 0.f : ex2(m0 - n0), r1 = m1 == -INFINITY ? 0.f : ex2(m1 - n1);
            l0 *= r0;
            l1 *= r1;
#pragma unroll
            for (int i = 0; i < 2 * kC; ++i) {
              o[i][0] *= r0;
              o[i][1] *= r1;
              o[i][2] *= r0;
              o[i][3] *= r1;
            }
            m0 = n0;
            m1 = n1;
          }
          s[0] = ex2(fmaf(s[0], a.c, -f0));
          s[1] = ex2(fmaf(s[1], a.c, -f1));
          s[2] = ex2(fmaf(s[2], a.c, -f0));
          s[3] = ex2(fmaf(s[3], a.c, -f1));
          l0 += s[0] + s[2];
          l1 += s[1] + s[3];
          const uint32_t p0 = movm_trans(pack(s[0], s[1], T())), p1 = movm_trans(pack(s[2], s[3], T()));
#pragma unroll
          for (int j = 0; j < kJ; ++j) {
            uint32_t w[4][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // slots 2 q4, 2 q4 + 1, 2 q4 + 8, 2 q4 + 9
              const int at = (k & 1) + (k >> 1) * 8;
              uint4 v = lds16(vat + at * (HD * 2) + 128 * j);
              // what lies behind the last slot may be anything, and 0 of it has to be 0
              if (slot + 2 * q4 + at >= sq.kv) v = zero4();
              w[k][0] = v.x, w[k][1] = v.y, w[k][2] = v.z, w[k][3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mma<T>(o[4 * j + i], __byte_perm(w[0][i], w[1][i], 0x5410), __byte_perm(w[0][i], w[1][i], 0x7632),
                     __byte_perm(w[2][i], w[3][i], 0x5410), __byte_perm(w[2][i], w[3][i], 0x7632), p0, p1);
          }
          __syncwarp();  // all have read the stage
          issue();
        }
        if (dead) break;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l0 += __shfl_xor_sync(0xffffffffu, l0, d);
          l1 += __shfl_xor_sync(0xffffffffu, l1, d);
        }
        const bool whole = t0 == 0 && u1 == steps;
        // ---- rows 2 q4 and 2 q4 + 1: the outputs, or a record
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 2 * q4 + e;
          if (r >= rows) continue;
          float m = e ? m1 : m0, l = e ? l1 : l0;
          const int token = r / a.gq, h = head * a.gq + r % a.gq;
          float* const mine = a.recs + (((size_t)warp * 2 + (t0 == 0 ? 1 : 0)) * kFewRows + r) * few_row_floats(HD);
          if (u0 > t0) {  // what the sums before this one have left
            const float mm = fmaxf(m, had_m[e]), f = m == -INFINITY ? 0.f : ex2(m - mm);
            const float fo = had_m[e] == -INFINITY ? 0.f : ex2(had_m[e] - mm);
            m = mm;
            l = l * f + had_l[e] * fo;
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* was = mine + 64 * j + 8 * g + 2 * i;
                o[4 * j + i][e] = o[4 * j + i][e] * f + was[0] * fo;
                o[4 * j + i][2 + e] = o[4 * j + i][2 + e] * f + was[1] * fo;
              }
          }
          had_m[e] = m;
          had_l[e] = l;
          if (whole && sq.part < 0) {
            const float inv = l != 0.f ? 1.f / l : 0.f;
            T* out = static_cast<T*>(a.out) + (size_t)(sq.row0 + token) * a.out_stride + (size_t)h * HD + 8 * g;
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) w[i] = pack(o[4 * j + i][e] * inv, o[4 * j + i][2 + e] * inv, T());
              *reinterpret_cast<uint4*>(out + 64 * j) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            float* rec = whole ? a.parts + ((size_t)(sq.part + token) * b.n_heads + h) * few_row_floats(HD) : mine;
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
              for (int i = 0; i < 4; i += 2)
                *reinterpret_cast<float4*>(rec + 64 * j + 8 * g + 2 * i) =
                    make_float4(o[4 * j + i][e], o[4 * j + i][2 + e], o[4 * j + i + 1][e], o[4 * j + i + 1][2 + e]);
            if (g == 0) *reinterpret_cast<float2*>(rec + HD) = make_float2(m, l);
          }
        }
      }
      if (dead) break;
    }
    // ---- the next unit
    left -= min(length - off, left);
    if (left <= 0) return;
    off = 0;
    if (++head >= a.K) {
      head = 0;
      do {
        if (++seq >= a.shared.n_seqs) return;
        sq = paged_seq(a.shared, seq);
      } while (sq.few <= 0);
    }
  }
  // (only after a wait that ran out) nobody leaves while a copy may still be landing: that of the failed step and later
  for (unsigned i = done - 1; i != ahead.count; ++i)
    if ((ahead.there >> (i & 31)) & 1u) {
      mbar_wait_s(bars + 8 * (i % kStages), (phases >> (i % kStages)) & 1u, a.status);
      phases ^= 1u << (i % kStages);
    }
}

}  // namespace

cudaError_t paged_few(const PagedFewArgs& a, int head_dim, int type, int device, int grid, cudaStream_t s) {
  PagedFewArgs p = a;
  static SmemCap caps[4];
  const int which = (head_dim == 128 ? 2 : 0) + (type == 1 ? 1 : 0);
  const void* const fns[4] = {
      reinterpret_cast<const void*>(&paged_few_kernel<64, __nv_bfloat16>), reinterpret_cast<const void*>(&paged_few_kernel<64, __half>),
      reinterpret_cast<const void*>(&paged_few_kernel<128, __nv_bfloat16>), reinterpret_cast<const void*>(&paged_few_kernel<128, __half>)};
  const size_t smem = (size_t)kFewWarps * few_stages(head_dim) * 2 * kFewSlots * head_dim * 2;
  const cudaError_t e = caps[which].raise(fns[which], device, smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(fns[which], dim3(grid), dim3(kFewThreads), smem, s, true, &p);
}

}  // namespace yb
