// kv_merge.h — the end of a cached-attention row: the wavefronts' partials joined through LDS, and
// the key splits' through the caller's workspace. Shared by the 16/32-bit and the 8-bit caches.
#pragma once

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kMaxMergeSplits = 32;  // upper bound on splits per row (host plan guarantees it)

// A quiet NaN built from its bit pattern (some files are compiled with -fno-honor-nans, under
// which a NaN literal would be undefined); it marks output rows with invalid metadata.
__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7fc00000u); }

// Combines the per-wavefront partials (o[64], m, l per query, in LDS) of one workgroup and
// writes the output rows, or, when the row's keys are split over several workgroups,
// publishes this split's partial and lets the last split to arrive merge them all. SPLIT false: the
// launch splits no row.
template <typename T, int SQ, int kWaves, bool SPLIT = true, typename Args>
__device__ __forceinline__ void kv_finish(const Args& a, int b, int t0, int nq, int sq_stride, int h, int split,
                                          int n_split_b, bool bad, float (&sm_acc)[kWaves][SQ][kHeadDim],
                                          float (&sm_m)[kWaves][SQ], float (&sm_l)[kWaves][SQ]) {
  constexpr int kThreads = kWaves * 64;
  constexpr int EB = ElemBytes<T>::value;
  constexpr int kPart = kHeadDim + 2;  // floats per partial: o[64], m, l
  __shared__ int sm_last;
  const int tid = threadIdx.x;
  auto store_out = [&](int t, int d, float val) {
    char* op = a.o + b * a.os[0] + (t0 + t) * a.os[1] + h * a.os[2];
    if constexpr (EB == 4)
      reinterpret_cast<float*>(op)[d] = val;
    else if constexpr (__is_same(T, Bf16))
      reinterpret_cast<__bf16*>(op)[d] = (__bf16)val;
    else
      reinterpret_cast<_Float16*>(op)[d] = (_Float16)val;
  };
  // This workgroup's (o, m, l) for query t, dim d, from the per-wavefront LDS partials.
  auto wg_partial = [&](int t, int d, float& O, float& M, float& L) {
    M = kNegBig;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sm_m[w][t]);
    L = 0.f;
    O = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(sm_m[w][t] - M);
      L = __builtin_fmaf(sm_l[w][t], f, L);
      O = __builtin_fmaf(sm_acc[w][t][d], f, O);
    }
  };

  if (!SPLIT || n_split_b == 1) {
    for (int idx = tid; idx < nq * kHeadDim; idx += kThreads) {
      const int t = idx / kHeadDim, d = idx % kHeadDim;
      float O, M, L;
      wg_partial(t, d, O, M, L);
      store_out(t, d, bad ? quiet_nan() : O / L);
    }
    return;
  }
  if constexpr (!SPLIT) return;

  // ---- several splits: publish this split's partial; the last split to arrive merges ----
  // Partials are laid out with the workspace's row stride sq_stride (= the launch's query block,
  // which the host sized the workspace for; it can be smaller than SQ).
  const int64_t unit = ((int64_t)b * a.n_qblocks + t0 / sq_stride) * a.H + h;
  float* part = a.ws_part + (unit * a.n_splits) * (sq_stride * kPart);
  for (int idx = tid; idx < nq * kHeadDim; idx += kThreads) {
    const int t = idx / kHeadDim, d = idx % kHeadDim;
    float O, M, L;
    wg_partial(t, d, O, M, L);
    float* pp = part + (split * sq_stride + t) * kPart;
    __hip_atomic_store(pp + d, O, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (d == 0) {
      __hip_atomic_store(pp + kHeadDim, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(pp + kHeadDim + 1, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  // Ordering without cache maintenance: the partial was written with agent-scope atomic
  // stores, which complete at the device coherence point; waiting for them (vmcnt 0) before
  // the counter update makes it visible to whichever split reads the count last. (A C++
  // release fence here would write back the whole L2 of this XCD from every split.)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    const int prev = __hip_atomic_fetch_add(a.ws_count + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_last = prev == n_split_b - 1;
  }
  __syncthreads();
  if (!sm_last) return;
  // The merging workgroup reads the partials with agent-scope atomic loads (coherent, issued
  // only after the counter told it every partial had landed): kMergeBatch splits' o values per
  // (query, dim) into registers and every (m, l) pair into LDS, all in one trip to memory. (One
  // load per split in turn, each waited for: 5 queries over 1500 rows, 12 splits, 18.0 us a launch
  // against 10.9; one query 11.4 against 9.0.)
  constexpr int kMergeBatch = 16;
  constexpr int kItems = (SQ * kHeadDim + kThreads - 1) / kThreads;  // (query, dim) pairs per thread
  float ov[kItems][kMergeBatch];
  auto load_o = [&](int it, int sp0) __attribute__((always_inline)) {
    const int idx = tid + it * kThreads, t = idx / kHeadDim, d = idx % kHeadDim;
#pragma unroll
    for (int u = 0; u < kMergeBatch; ++u) {
      ov[it][u] = 0.f;
      if (sp0 + u < n_split_b && t < nq)
        ov[it][u] = __hip_atomic_load(part + ((sp0 + u) * sq_stride + t) * kPart + d, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT);
    }
  };
#pragma unroll
  for (int it = 0; it < kItems; ++it) load_o(it, 0);
  __shared__ float sm_pm[kMaxMergeSplits * SQ], sm_pl[kMaxMergeSplits * SQ];
  for (int idx = tid; idx < n_split_b * nq; idx += kThreads) {
    const int sp = idx / nq, t = idx % nq;
    float* pp = part + (sp * sq_stride + t) * kPart;
    sm_pm[sp * SQ + t] = __hip_atomic_load(pp + kHeadDim, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_pl[sp * SQ + t] = __hip_atomic_load(pp + kHeadDim + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    pp[kHeadDim] = 0.f;  // consumed: leave the workspace all-zero (see below)
    pp[kHeadDim + 1] = 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    const int idx = tid + it * kThreads, t = idx / kHeadDim, d = idx % kHeadDim;
    if (t >= nq) continue;
    float mm = kNegBig;
    for (int sp = 0; sp < n_split_b; ++sp) mm = fmaxf(mm, sm_pm[sp * SQ + t]);
    float L = 0.f, O = 0.f;
    for (int sp0 = 0; sp0 < n_split_b; sp0 += kMergeBatch) {
      if (sp0) load_o(it, sp0);
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
        if (sp0 + u < n_split_b) {
          const float f = fast_exp2(sm_pm[(sp0 + u) * SQ + t] - mm);
          L = __builtin_fmaf(sm_pl[(sp0 + u) * SQ + t], f, L);
          O = __builtin_fmaf(ov[it][u], f, O);
          part[((sp0 + u) * sq_stride + t) * kPart + d] = 0.f;
        }
      }
    }
    store_out(t, d, O / L);
  }
  // Leave the counter at zero too. Every call returns the whole workspace to all-zero, so the
  // counters of any later call, whatever its shape and therefore its layout, start at zero.
  if (tid == 0) __hip_atomic_store(a.ws_count + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace
}  // namespace wdrz
