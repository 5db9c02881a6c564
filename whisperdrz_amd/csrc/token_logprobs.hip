// token_logprobs.hip — what a step's logits say about its tokens: log probabilities of given tokens, the entropy
// of the distribution and the likeliest alternatives, in one pass over the logits.
//
//   d_i = x_i - M,  Z = sum e^d_i,  log p_i = d_i - ln Z,  H = -sum p_i log p_i = ln Z - sum e^d_i d_i / Z
//
// In the sums the term of the largest token, e^0, stands apart: Z = 1 + r, ln Z = log1p(r), so a row with one likely
// token keeps the digits of its small ln Z. Blocked tokens count as -inf. A row in which nothing is left has log probabilities of -inf, entropy 0 and no
// alternatives (ids -1); NaN or +inf among its tokens makes all of the row NaN. e^d is taken as 2^(d log2 e) of the
// difference, so the terms that count are exact to 2^-22; sums are fp32 in a thread (up to 64 terms of one
// reference) and fp64 across threads.
//
// Alternatives are ordered by logit, equal ones by index: keys of 64 bits, (order of the fp32 bits, ~index), are all
// different. A thread keeps its largest key while it sums. The k-th largest T of the threads' keys bounds the
// k-th largest of all from below, and only the at most k threads whose key is T or above own a key that can be
// among the first k: their tokens alone are read again.
//
// Bound: the bytes of the logits; for few rows launch, a trip to memory, and the counting of keys.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "layernorm.h"
#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kVec = 8;         // tokens a load
constexpr int kBatch = 4;       // loads in flight a thread
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 32;
constexpr int kPerSplit = 65536;  // tokens a workgroup takes at most
constexpr int kMaxSplits = 16;
constexpr int kOwned = kPerSplit / kThreads;  // tokens a thread takes at most
constexpr float kFar = -200.f;    // e^-200 is 0 in fp32, and so are the terms of all logits further down
constexpr int kCounters = 4096;   // rows of a launch that is split: their counters stand before the partials

// Order of fp32 values as unsigned numbers, above 0 for what can be chosen (-inf cannot).
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t u = __float_as_uint(x);
  return x == -INFINITY ? 0u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unorder(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  // +0 and -0 are equal: the lower index wins
  const uint32_t o = order(x + 0.f);
  return o ? (uint64_t)o << 32 | (uint32_t)~i : 0;
}

// The tokens of a part of the row: the largest, m (-inf: none), the sum r of the others' e^(x - m) and the sum w of
// e^(x - m) (x - m). r is NaN where a token is NaN or +inf.
struct Sum {
  double r, w;
  float m;
};
__device__ __forceinline__ void join(Sum& a, float m, double r, double w) {
  if (m == -INFINITY || a.m == -INFINITY) {
    const bool other = a.m == -INFINITY;
    a.r += r;  // one is 0, or NaN
    a.w = other ? w : a.w;
    a.m = other ? m : a.m;
    return;
  }
  const bool up = m > a.m;  // the smaller side's largest token joins the others
  const double d = up ? (double)a.m - m : (double)m - a.m, f = (double)expf((float)d);
  const double less_r = 1. + (up ? a.r : r), less_w = up ? a.w : w;
  a.r = (up ? r : a.r) + less_r * f;
  a.w = (up ? w : a.w) + (less_w + d * less_r) * f;
  a.m = up ? m : a.m;
}

// The k largest of n different keys (0: none), sorted, to out[0 .. k - 1] (0 behind the last). Every thread of the
// workgroup calls it; keys and out in LDS.
__device__ __forceinline__ void largest(const uint64_t* keys, int n, int k, uint64_t* out) {
  for (int i = threadIdx.x; i < k; i += kThreads) out[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > mine;
    if (mine && rank < k) out[rank] = mine;
  }
  __syncthreads();
}

struct Partial {  // one split's sums and keys, in the workspace
  double r, w;
  uint64_t m;  // fp32 bits
  uint64_t key[kMaxTop];
};

template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int EB = ElemBytes<T>::value, kWords = kVec * EB / 4;
  __shared__ uint64_t sm_keys[kMaxTop * (kOwned + kVec)];  // candidates
  __shared__ uint64_t sm_wave[kWaves * kMaxTop], sm_top[kMaxTop];
  __shared__ double sm_r[kWaves], sm_w[kWaves];
  __shared__ float sm_m[kWaves];
  __shared__ int sm_owner[kMaxTop], sm_n, sm_owners, sm_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, split = blockIdx.y, top = a.top;
  const char* lr = static_cast<const char*>(a.logits) + (int64_t)row * a.l_stride * EB;
  const uint8_t* bm = a.blocked ? a.blocked + (int64_t)row * a.m_stride : nullptr;
  // this split's tokens [v0, v1): whole loads, the last V % 8 tokens with the last split
  const int n_vec = a.V / kVec;
  const int c_begin = (int)((int64_t)n_vec * split / a.splits), c_end = (int)((int64_t)n_vec * (split + 1) / a.splits);
  const int tail = split == a.splits - 1 ? a.V - n_vec * kVec : 0;

  float m = -INFINITY, far = -3.402823466e38f, r = 0.f, w = 0.f;
  int at = 0;  // the largest token's index
  auto take = [&](float (&x)[kVec], int i0) __attribute__((always_inline)) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < kVec; ++e) mx = fmaxf(mx, x[e]);
    if (mx > m) {
      const float d = fmaxf(m - mx, kFar), f = fast_exp2(d * kLog2e);
      w = m == -INFINITY ? w : (w + d * (1.f + r)) * f;
      r = m == -INFINITY ? r : (1.f + r) * f;
      m = mx;
      far = mx + kFar;
      int first = 0;
#pragma unroll
      for (int e = kVec - 1; e >= 0; --e)
        if (x[e] == mx) first = e;
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e == first) x[e] = -INFINITY;  // its term stands apart
      at = i0 + first;
    }
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float d = x[e] < far ? kFar : x[e] - m;
      const float p = fast_exp2(d * kLog2e);
      r += p;
      w = __builtin_fmaf(p, d, w);
    }
  };
  // token e of a load of tokens i0 .. i0 + 7
  auto widen = [&](const uint32_t* raw, const u32x2& mask, float (&x)[kVec]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      x[e] = Elem<T>::word(raw, e);
      if (mask[e >> 2] >> (8 * (e & 3)) & 0xffu) x[e] = -INFINITY;
    }
  };
  for (int c0 = c_begin + tid; c0 < c_end; c0 += kBatch * kThreads) {
    uint32_t raw[kBatch][kWords];
    u32x2 mask[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * kThreads;
      mask[u] = u32x2{0, 0};
      if (c < c_end) {
        __builtin_memcpy(raw[u], lr + (int64_t)c * kVec * EB, sizeof(raw[u]));
        if (bm) __builtin_memcpy(&mask[u], bm + (int64_t)c * kVec, 8);
      }
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * kThreads;
      if (c < c_end) {
        float x[kVec];
        widen(raw[u], mask[u], x);
        take(x, c * kVec);
      }
    }
  }
  auto tail_token = [&](float (&x)[kVec], int i) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = -INFINITY;
    if (!(bm && bm[i])) x[0] = Elem<T>::load1(lr, i);
  };
  if (tid < tail) {
    float x[kVec];
    tail_token(x, n_vec * kVec + tid);
    take(x, n_vec * kVec + tid);
  }
  const bool bad = !(r < INFINITY) || !(m < INFINITY);  // NaN among the tokens, or +inf

  // ---- sums over the workgroup ----
  Sum s{(double)r, (double)w, m};
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) join(s, __shfl_xor(s.m, o), __shfl_xor(s.r, o), __shfl_xor(s.w, o));
  if (__any(bad)) s.r = __builtin_nan("");
  if (lane == 0) {
    sm_r[wave] = s.r;
    sm_w[wave] = s.w;
    sm_m[wave] = s.m;
  }
  if (tid == 0) sm_n = sm_owners = 0;

  // ---- alternatives ----
  if (top) {
    const uint64_t mine = key_of(m, at);
    int rank = 0;  // among the wavefront's keys
    for (int i = 0; i < 64; ++i) rank += __shfl(mine, i) > mine;
    if (lane < top) sm_wave[wave * top + lane] = 0;
    __builtin_amdgcn_wave_barrier();
    if (mine && rank < top) sm_wave[wave * top + rank] = mine;
    __syncthreads();
    largest(sm_wave, kWaves * top, top, sm_top);
    const uint64_t least = max(sm_top[top - 1], (uint64_t)1);
    if (mine >= least) sm_owner[atomicAdd(&sm_owners, 1)] = tid;  // at most `top` of them
    __syncthreads();
    const int per = (c_end - c_begin + kThreads - 1) / kThreads + 1;  // an owner's loads, and its tail token
    for (int i = tid; i < sm_owners * per; i += kThreads) {
      const int t = sm_owner[i / per], j = i % per, c = c_begin + t + j * kThreads;
      float x[kVec];
      int i0;
      if (j == per - 1) {
        if (t >= tail) continue;
        i0 = n_vec * kVec + t;
        tail_token(x, i0);
      } else {
        if (c >= c_end) continue;
        uint32_t raw[kWords];
        u32x2 mask = {0, 0};
        __builtin_memcpy(raw, lr + (int64_t)c * kVec * EB, sizeof(raw));
        if (bm) __builtin_memcpy(&mask, bm + (int64_t)c * kVec, 8);
        widen(raw, mask, x);
        i0 = c * kVec;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const uint64_t key = key_of(x[e], i0 + e);
        if (key >= least) sm_keys[atomicAdd(&sm_n, 1)] = key;
      }
    }
    __syncthreads();
    largest(sm_keys, sm_n, top, sm_top);
  } else {
    __syncthreads();
  }
  if (wave == 0) {  // every lane the same
    s = Sum{sm_r[0], sm_w[0], sm_m[0]};
    for (int i = 1; i < kWaves; ++i) join(s, sm_m[i], sm_r[i], sm_w[i]);
  }

  if (a.splits > 1) {
    // every split publishes its sums and keys at the device's coherence point; the last to arrive joins them
    Partial* const parts = reinterpret_cast<Partial*>(static_cast<char*>(a.ws) + kCounters * 4) + (int64_t)row * a.splits;
    int* const count = static_cast<int*>(a.ws) + row;
    if (tid == 0) {
      __hip_atomic_store(&parts[split].r, s.r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&parts[split].w, s.w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(&parts[split].m, (uint64_t)__float_as_uint(s.m), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (tid < top) __hip_atomic_store(&parts[split].key[tid], sm_top[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0) sm_last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.splits - 1;
    __syncthreads();
    if (!sm_last) return;
    if (tid == 0) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    if (wave == 0) {
      s = Sum{0., 0., -INFINITY};
      if (lane < a.splits) {
        s.r = __hip_atomic_load(&parts[lane].r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s.w = __hip_atomic_load(&parts[lane].w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s.m = __uint_as_float((uint32_t)__hip_atomic_load(&parts[lane].m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
      }
      const bool nan = __any(!(s.r < INFINITY));
#pragma unroll
      for (int o = kMaxSplits / 2; o >= 1; o >>= 1) join(s, __shfl_xor(s.m, o), __shfl_xor(s.r, o), __shfl_xor(s.w, o));
      s = Sum{__shfl(s.r, 0), __shfl(s.w, 0), __shfl(s.m, 0)};  // for the lanes behind the splits too
      if (nan) s.r = __builtin_nan("");
    }
    if (top) {
      for (int i = tid; i < a.splits * top; i += kThreads)
        sm_keys[i] = __hip_atomic_load(&parts[i / top].key[i % top], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      largest(sm_keys, a.splits * top, top, sm_top);
    }
  }
  // ---- results, by the first wavefront ----
  if (wave != 0) return;
  const bool nan = !(s.r < INFINITY), none = !nan && s.m == -INFINITY;
  const float fnan = __builtin_nanf("");
  const double lz = nan || none ? 0. : log1p(s.r);
  if (lane == 0) {
    a.entropy[row] = nan ? fnan : none ? 0.f : (float)(lz - s.w / (1. + s.r));
    const int64_t t = a.tokens[row];
    float lp = fnan;  // a token out of range
    if (!nan && t >= 0 && t < a.V) {
      const float x = bm && bm[t] ? -INFINITY : Elem<T>::load1(lr, (int)t);
      lp = none || x == -INFINITY ? -INFINITY : (float)((double)x - s.m - lz);
    }
    a.logprob[row] = lp;
  }
  if (lane < top) {
    const uint64_t key = sm_top[lane];
    a.top_id[(int64_t)row * top + lane] = nan || !key ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
    a.top_logprob[(int64_t)row * top + lane] =
        nan ? fnan : !key ? -INFINITY : (float)((double)unorder((uint32_t)(key >> 32)) - s.m - lz);
  }
}

int plan_splits(int64_t rows, int64_t V) {
  const int64_t least = (V + kPerSplit - 1) / kPerSplit;
  int64_t want = 1;
  if (rows <= 64) want = std::min<int64_t>(V / (kVec * kThreads), 512 / rows);
  return (int)std::min<int64_t>(std::max<int64_t>(std::max<int64_t>(want, 1), least), kMaxSplits);
}

}  // namespace

size_t logprobs_workspace_bytes(int64_t rows, int64_t V, int64_t top) {
  (void)top;
  const int s = plan_splits(rows, V);
  return s == 1 ? 0 : kCounters * 4 + (size_t)std::min<int64_t>(rows, kCounters) * s * sizeof(Partial);
}

hipError_t launch_token_logprobs(int dtype, LogprobArgs a, hipStream_t stream) {
  const int64_t rows = a.rows, most = plan_splits(rows, a.V) > 1 ? kCounters : rows;
  const int eb = dtype == 0 ? 4 : 2;
  a.splits = plan_splits(rows, a.V);
  for (int64_t r0 = 0; r0 < rows; r0 += most) {
    LogprobArgs b = a;
    b.rows = (int)std::min(most, rows - r0);
    b.logits = static_cast<const char*>(a.logits) + r0 * a.l_stride * eb;
    if (a.blocked) b.blocked = a.blocked + r0 * a.m_stride;
    b.tokens = a.tokens + r0;
    b.logprob = a.logprob + r0;
    b.entropy = a.entropy + r0;
    if (a.top) {
      b.top_logprob = a.top_logprob + r0 * a.top;
      b.top_id = a.top_id + r0 * a.top;
    }
    const dim3 grid((unsigned)b.rows, (unsigned)b.splits);
    if (dtype == 2) hipLaunchKernelGGL((token_logprobs_kernel<Bf16>), grid, dim3(kThreads), 0, stream, b);
    else if (dtype == 1) hipLaunchKernelGGL((token_logprobs_kernel<F16>), grid, dim3(kThreads), 0, stream, b);
    else hipLaunchKernelGGL((token_logprobs_kernel<F32>), grid, dim3(kThreads), 0, stream, b);
  }
  return hipGetLastError();
}

}  // namespace wdrz
