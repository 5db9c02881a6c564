// token_logprobs.hip — what a step's logits say about its tokens: log probabilities of given tokens, the entropy
// of the distribution and the likeliest alternatives, in one pass over the logits.
//
//   d_i = x_i - M,  Z = sum e^d_i,  log p_i = d_i - ln Z,  H = -sum p_i log p_i = ln Z - sum e^d_i d_i / Z
//
// In the sums the term of the largest token, e^0, stands apart: Z = 1 + r, ln Z = log1p(r), so a row with one likely
// token keeps the digits of its small ln Z. Blocked tokens count as -inf. A row in which nothing is left has log
// probabilities of -inf, entropy 0 and no alternatives (ids -1); NaN or +inf among its tokens makes all of the row
// NaN. e^d is taken as 2^(d log2 e) of the difference, so the terms that count are exact to 2^-22; sums are fp32 in a
// wavefront and fp64 above it.
//
// Alternatives are ordered by logit, equal ones by index: keys of 64 bits, (order of the fp32 bits, ~index), are all
// different. A thread keeps its largest key while it sums. The k-th largest of the keys of 16 or 64 groups of threads
// bounds the k-th largest of all from below. A workgroup of one load a thread lists its tokens that are no smaller, a
// few more than k; one of more loads lists such threads, and reads the tokens of the k first again, which alone can own
// a key among the first k. Where a list grows beyond a wavefront it is ranked in full.
//
// Bound: VALU issue, 17 instructions a token (two of them the exponential's, five the largest term's, which some lane of a
// wavefront moves at most loads), near the bytes of the logits; for few rows launch, two trips to memory and a handful of
// barriers. 3584 x 51866 bf16 with 3 alternatives 85 us, 4.4 TB/s (a copy 5.2; 93 us with the masks' instructions where
// there is no mask; logits without a likely token, whose largest moves more often, 102, with a mask 120); one row of 51866
// fp32 in 26 workgroups 11.4 us. 3 or 8 loads in flight a thread 84 and 87 us.
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
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 32;
constexpr int kList = kThreads * kVec + kVec + kMaxTop;  // tokens listed at most, with those of the round before
constexpr float kFar = -200.f;    // e^-200 is 0 in fp32, and so are the terms of all logits further down
constexpr int kCounters = 4096;   // of rows that are split (512 at most, each over two workgroups or more), before their partials

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

// Maximum of different keys over the wavefront's first N lanes (N a power of two); every one of them gets it.
template <int N> __device__ __forceinline__ uint64_t key_max(uint64_t k) {
#pragma unroll
  for (int o = N / 2; o >= 1; o >>= 1) {
    const uint64_t other = __shfl_xor(k, o);
    k = other > k ? other : k;
  }
  return k;
}
// The rank of this lane's key among the wavefront's first n (0: the largest).
__device__ __forceinline__ int key_rank(uint64_t k, int n) {
  int rank = 0;
  for (int i = 0; i < n; ++i) {
    const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), i) << 32 |
                           (uint32_t)__builtin_amdgcn_readlane((int)k, i);
    rank += other > k;
  }
  return rank;
}
// The nth largest of the wavefront's first n keys, whose ranks are given; 1, below every key, where there are fewer.
__device__ __forceinline__ uint64_t nth_key(uint64_t k, int rank, int n, int nth) {
  const uint64_t lanes = __ballot((int)(threadIdx.x & 63) < n && rank == nth - 1 && k != 0);
  if (!lanes) return 1;
  const int src = __ffsll((unsigned long long)lanes) - 1;
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), src) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)k, src);
}
__device__ __forceinline__ float key_value(uint64_t k) { return k ? unorder((uint32_t)(k >> 32)) : -INFINITY; }

// The tokens of a part of the row: the largest key, the sum r of the others' e^(x - m) and the sum w of e^(x - m)
// (x - m), m the largest logit. Sums over the wavefront's first N lanes, every part with a largest key of its own.
template <int N, typename F> __device__ __forceinline__ void join(uint64_t key, F& r, F& w, uint64_t& top_key) {
  top_key = key_max<N>(key);
  const float m = key_value(key), to = key_value(top_key);
  const float d = m == -INFINITY ? kFar : fmaxf(m - to, kFar);
  const F f = key == 0 ? F(0) : F(expf(d)), others = key == top_key ? r : r + F(1);
  w = (w + F(d) * others) * f;
  r = key == 0 ? r : others * f;  // r without a key: 0, or NaN
#pragma unroll
  for (int o = N / 2; o >= 1; o >>= 1) {
    r += __shfl_xor(r, o);
    w += __shfl_xor(w, o);
  }
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

// The same for the first wavefront alone where they fit it; it may read `out` afterwards, the others behind a barrier.
__device__ __forceinline__ void sort_top(const uint64_t* keys, int n, int k, uint64_t* out) {
  if (n > 64) {
    largest(keys, n, k, out);
    return;
  }
  if (threadIdx.x >= 64) return;
  const int lane = threadIdx.x;
  const uint64_t mine = lane < n ? keys[lane] : 0;
  const int rank = key_rank(mine, n);
  if (lane < k) out[lane] = 0;
  __builtin_amdgcn_wave_barrier();
  if (mine && rank < k) out[rank] = mine;
  __builtin_amdgcn_wave_barrier();
}

static_assert(2 * kMaxSplits * kMaxTop <= kList, "the splits' keys and those of them that count");
struct Partial {  // one split's sums and keys, in the workspace
  double r, w;
  uint64_t top;
  uint64_t key[kMaxTop];
};

template <typename T>
__global__ __launch_bounds__(kThreads) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int EB = ElemBytes<T>::value, kWords = kVec * EB / 4;
  __shared__ uint64_t sm_keys[kList];
  __shared__ uint64_t sm_list[kWaves * kMaxTop], sm_top[kMaxTop], sm_group[64], sm_wave[kWaves];
  __shared__ double sm_r[kWaves], sm_w[kWaves];
  __shared__ int sm_n, sm_listed, sm_last;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = blockIdx.x, split = blockIdx.y, top = a.top;
  const char* lr = static_cast<const char*>(a.logits) + (int64_t)row * a.l_stride * EB;
  const uint8_t* bm = a.blocked ? a.blocked + (int64_t)row * a.m_stride : nullptr;
  // this split's tokens [v0, v1): whole loads, the last V % 8 tokens with the last split
  const int n_vec = a.V / kVec;
  const int c_begin = (int)((int64_t)n_vec * split / a.splits), c_end = (int)((int64_t)n_vec * (split + 1) / a.splits);
  const int tail = split == a.splits - 1 ? a.V - n_vec * kVec : 0;

  float m = -INFINITY, ref = 0.f, r = 0.f, w = 0.f;  // the largest logit, the same or 0 while there is none
  int at = 0;  // its index
  auto take = [&](float (&x)[kVec], int i0) __attribute__((always_inline)) {
    float mx = x[0];
#pragma unroll
    for (int e = 1; e < kVec; ++e) mx = fmaxf(mx, x[e]);
    if (mx > m) {
      const float d = fmaxf(m - mx, kFar), f = fast_exp2(d * kLog2e);
      w = m == -INFINITY ? w : (w + d * kLog2e * (1.f + r)) * f;
      r = m == -INFINITY ? r : (1.f + r) * f;
      m = ref = mx;
      int first = 0;
#pragma unroll
      for (int e = kVec - 1; e >= 0; --e)
        if (x[e] == mx) first = e;
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (e == first) x[e] = -INFINITY;  // its term stands apart
      at = i0 + first;
    }
    float p[kVec], u = 0.f;  // a load's sums first: a thread's grow by one term a load
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const float t = (x[e] - ref) * kLog2e;
      p[e] = fast_exp2(t);
      u = __builtin_fmaf(p[e], fmaxf(t, kFar), u);  // in units of ln 2; 0 times the far ones is 0
    }
    r += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    w += u;
  };
  // token e of a load of tokens i0 .. i0 + 7
  auto widen = [&](const uint32_t* raw, const u32x2& mask, float (&x)[kVec]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) x[e] = Elem<T>::word(raw, e);
    if (bm) {
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (mask[e >> 2] >> (8 * (e & 3)) & 0xffu) x[e] = -INFINITY;
    }
  };
  uint32_t raw[kBatch][kWords];
  u32x2 mask[kBatch];
  for (int c0 = c_begin + tid; c0 < c_end; c0 += kBatch * kThreads) {
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
  if (!(m < INFINITY)) r = __builtin_nanf("");  // +inf among the tokens

  // ---- sums over the wavefront, then the workgroup (in the first wavefront) ----
  const uint64_t mine = key_of(m, at);
  const int groups = top <= 8 ? 16 : 64, lanes = kThreads / groups;  // of threads, for the bound of the alternatives
  if (tid == 0) sm_n = sm_listed = 0;
  {
    uint64_t k = mine, wave_key;
    for (int o = 1; o < lanes; o <<= 1) {
      const uint64_t other = __shfl_xor(k, o);
      k = other > k ? other : k;
    }
    if (tid % lanes == 0) sm_group[tid / lanes] = k;
    float wr = r, ww = w * 0.69314718055994531f;
    join<64>(mine, wr, ww, wave_key);
    if (lane == 0) {
      sm_wave[wave] = wave_key;
      sm_r[wave] = wr;
      sm_w[wave] = ww;
    }
  }
  __syncthreads();
  double sr = 0., sw = 0.;
  uint64_t best = 0;
  if (wave == 0) {
    if (lane < kWaves) {
      sr = sm_r[lane];
      sw = sm_w[lane];
    }
    join<kWaves>(lane < kWaves ? sm_wave[lane] : 0, sr, sw, best);
  }

  // ---- alternatives ----
  if (top) {
    auto list = [&](const float (&x)[kVec], int first, uint64_t least) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const uint64_t key = key_of(x[e], first + e);
        if (key >= least) sm_keys[atomicAdd(&sm_n, 1)] = key;
      }
    };
    const uint64_t gk = sm_group[lane & (groups - 1)];
    uint64_t least = nth_key(gk, key_rank(gk, groups), groups, top);
    if (c_end - c_begin <= kThreads) {  // every token is still here
      float x[kVec];
      if (c_begin + tid < c_end) {
        widen(raw[0], mask[0], x);
        list(x, (c_begin + tid) * kVec, least);
      }
      if (tid < tail) {
        tail_token(x, n_vec * kVec + tid);
        list(x, n_vec * kVec + tid, least);
      }
      __syncthreads();
    } else {
      if (mine >= least) {
        const int i = atomicAdd(&sm_listed, 1);
        if (i < 64) sm_list[i] = mine;
      }
      __syncthreads();
      const int listed = sm_listed;
      if (listed > 64) {
        __syncthreads();
        const int rank = key_rank(mine, 64);
        if (lane < top) sm_list[wave * top + lane] = 0;
        __builtin_amdgcn_wave_barrier();
        if (mine && rank < top) sm_list[wave * top + rank] = mine;
        __syncthreads();
        largest(sm_list, kWaves * top, top, sm_top);
      }
      const int n = listed > 64 ? top : listed;  // different keys, some of them 0
      const uint64_t k = lane < n ? (listed > 64 ? sm_top[lane] : sm_list[lane]) : 0;
      least = nth_key(k, key_rank(k, n), n, top);
      const uint64_t own = __ballot(k != 0 && k >= least);  // lanes whose key's thread is read again: `top` at most
      // thread t's loads are c_begin + t, + kThreads, .., and the tail token n_vec * kVec + t
      const int owners = __popcll(own), per = (c_end - c_begin + kThreads - 1) / kThreads + 1;
      for (int i0 = 0; i0 < owners * per; i0 += kThreads) {
        const int i = i0 + tid, j = i % per;
        int src = 0;
        uint64_t left = own;
        for (int o = min(i / per, owners - 1); o > 0; --o) left &= left - 1;
        src = __ffsll((unsigned long long)left) - 1;
        const int index = (int)~(uint32_t)__shfl(k, src);  // of its largest token
        const int t = index >= n_vec * kVec ? index - n_vec * kVec : (index / kVec - c_begin) % kThreads, c = c_begin + t + j * kThreads;
        float x[kVec];
        if (i < owners * per && j == per - 1 && t < tail) {
          tail_token(x, n_vec * kVec + t);
          list(x, n_vec * kVec + t, least);
        } else if (i < owners * per && j < per - 1 && c < c_end) {
          uint32_t again[kWords];
          u32x2 m8 = {0, 0};
          __builtin_memcpy(again, lr + (int64_t)c * kVec * EB, sizeof(again));
          if (bm) __builtin_memcpy(&m8, bm + (int64_t)c * kVec, 8);
          widen(again, m8, x);
          list(x, c * kVec, least);
        }
        __syncthreads();
        if (i0 + kThreads < owners * per) {  // room for the next round: the first `top` so far
          largest(sm_keys, sm_n, top, sm_top);
          if (tid < top) sm_keys[tid] = sm_top[tid];
          if (tid == 0) sm_n = top;
          __syncthreads();
        }
      }
      if (owners == 0) __syncthreads();
    }
    sort_top(sm_keys, sm_n, top, sm_top);
  }

  if (a.splits > 1) {
    // every split publishes its sums and keys at the device's coherence point; the last to arrive joins them
    Partial* const parts = reinterpret_cast<Partial*>(static_cast<char*>(a.ws) + kCounters * 4) + (int64_t)row * a.splits;
    int* const count = static_cast<int*>(a.ws) + row;
    if (wave == 0) {
      if (lane == 0) {
        __hip_atomic_store(&parts[split].r, sr, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&parts[split].w, sw, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(&parts[split].top, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      if (lane < top) __hip_atomic_store(&parts[split].key[lane], sm_top[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0) sm_last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.splits - 1;
    __syncthreads();
    if (!sm_last) return;
    if (tid == 0) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    if (wave == 0) {
      uint64_t key = 0;
      sr = sw = 0.;
      if (lane < a.splits) {
        sr = __hip_atomic_load(&parts[lane].r, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sw = __hip_atomic_load(&parts[lane].w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        key = __hip_atomic_load(&parts[lane].top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      join<kMaxSplits>(key, sr, sw, best);
    }
    if (top) {
      const int n = a.splits * top;
      for (int i = tid; i < n; i += kThreads)
        sm_keys[i] = __hip_atomic_load(&parts[i / top].key[i % top], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (tid == 0) sm_n = 0;
      __syncthreads();
      if (n <= 64) {
        sort_top(sm_keys, n, top, sm_top);
      } else {
        // the splits' keys are sorted: the first few of each bound the `top`-th of all
        const int first = a.splits * ((top + a.splits - 1) / a.splits);  // 64 at most
        const uint64_t k = lane < first ? sm_keys[lane % a.splits * top + lane / a.splits] : 0;
        const uint64_t least = nth_key(k, key_rank(k, first), first, top);
        for (int i = tid; i < n; i += kThreads)
          if (sm_keys[i] >= least) sm_keys[kMaxSplits * kMaxTop + atomicAdd(&sm_n, 1)] = sm_keys[i];
        __syncthreads();
        sort_top(sm_keys + kMaxSplits * kMaxTop, sm_n, top, sm_top);
      }
    }
  }
  // ---- results, by the first wavefront ----
  if (wave != 0) return;
  sr = __shfl(sr, 0);
  best = __shfl(best, 0);
  const float m_row = key_value(best);
  const bool nan = !(sr < INFINITY), none = !nan && best == 0;
  const float fnan = __builtin_nanf("");
  const double lz = nan || none ? 0. : log1p(sr);
  if (lane == 0) {
    a.entropy[row] = nan ? fnan : none ? 0.f : (float)(lz - sw / (1. + sr));
    const int64_t t = a.tokens[row];
    float lp = fnan;  // a token out of range
    if (!nan && t >= 0 && t < a.V) {
      const float x = bm && bm[t] ? -INFINITY : Elem<T>::load1(lr, (int)t);
      lp = none || x == -INFINITY ? -INFINITY : (float)((double)x - m_row - lz);
    }
    a.logprob[row] = lp;
  }
  if (lane < top) {
    const uint64_t key = sm_top[lane];
    a.top_id[(int64_t)row * top + lane] = nan || !key ? -1 : (int64_t)(uint32_t)~(uint32_t)key;
    a.top_logprob[(int64_t)row * top + lane] = nan ? fnan : !key ? -INFINITY : (float)((double)key_value(key) - m_row - lz);
  }
}

// Workgroups a row.
int plan_splits(int64_t rows, int64_t V) {
  const int64_t one = (V / kVec + kThreads - 1) / kThreads;  // of one load a thread
  return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(one, 1024 / rows), kMaxSplits));
}

}  // namespace

size_t logprobs_workspace_bytes(int64_t rows, int64_t V, int64_t top) {
  (void)top;
  const int s = plan_splits(rows, V);
  return s == 1 ? 0 : kCounters * 4 + (size_t)rows * s * sizeof(Partial);
}

hipError_t launch_token_logprobs(int dtype, LogprobArgs a, hipStream_t stream) {
  a.splits = plan_splits(a.rows, a.V);
  const dim3 grid((unsigned)a.rows, (unsigned)a.splits);
  if (dtype == 2) hipLaunchKernelGGL((token_logprobs_kernel<Bf16>), grid, dim3(kThreads), 0, stream, a);
  else if (dtype == 1) hipLaunchKernelGGL((token_logprobs_kernel<F16>), grid, dim3(kThreads), 0, stream, a);
  else hipLaunchKernelGGL((token_logprobs_kernel<F32>), grid, dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace wdrz
