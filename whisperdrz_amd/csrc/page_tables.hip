// page_tables.hip — the bookkeeping of a paged key/value cache, on the GPU: which pages a request's new tokens
// go to, and the writes of their keys and values.
//
// A stream s holds `lens[s]` positions in `counts[s]` pages, tables[s][0 .. counts[s] - 1] in order; the pages
// that nobody holds are the first n_free entries of a stack. Request i adds m_i tokens to stream s_i. With P
// positions a page it needs
//     need_i = max(0, ceil((lens + m_i) / P) - counts),   off_i = need_0 + .. + need_(i-1)
// more pages, and gets the stack's entries n_free - 1 - off_i, n_free - 2 - off_i, ..; token t of it stands at
// position lens + t, slot tables[s][position / P] * P + position % P. Requests are served in their order while
// pages last: one whose off_i + need_i is above n_free gets nothing, which then holds for all behind it that need pages (the
// sums depend on no answer, and nobody overtakes a long prompt); nor does one that names no stream, a stream that an
// earlier one named, or a length that the table cannot hold.
//
// Bound: launch and a chain of four dependent trips to memory (stream -> its length -> the stack -> the table).
// One workgroup does the scan, since every request's pages depend on all before it. Plan and truncation of 8 streams 3.5 and
// 2.5 us on the GPU (13 us a pair of calls: the host's side), of 1000 prompts 12.3 (and 4.6 for 168000 tokens' slots) and 8.3:
// one CU's scattered reads and writes of lengths and tables. Up to 256 requests and tokens take the small form: a pair of calls for
// 52 streams of 4 tokens 6.9 us in a graph, of 5 (260 tokens, the large form, whose tokens find their request in memory) 10.2.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kSmallThreads = 256;  // threads of the workgroup, for up to as many requests and tokens; else
constexpr int kPlanThreads = 1024;
constexpr int kLdsSums = 2048;  // requests whose sums the tokens' workgroups keep in LDS

// Exclusive sums of two values over the workgroup's threads, and the totals. `sm` is free to use afterwards.
// The first are capped at `cap` (sums of 2^30 and more would leave 32 bits).
template <int kW>
__device__ __forceinline__ void scan2(int& a, int& b, int cap, int& total_a, int& total_b, int64_t (&sm_a)[kW], int (&sm_b)[kW]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t sa = a;
  int sb = b;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t ua = __shfl_up(sa, o);
    const int ub = __shfl_up(sb, o);
    if (lane >= o) {
      sa += ua;
      sb += ub;
    }
  }
  if (lane == 63) {
    sm_a[wave] = sa;
    sm_b[wave] = sb;
  }
  __syncthreads();
  int64_t base_a = 0, sum_a = 0;
  int base_b = 0;
  total_b = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    base_a += w < wave ? sm_a[w] : 0;
    base_b += w < wave ? sm_b[w] : 0;
    sum_a += sm_a[w];
    total_b += sm_b[w];
  }
  __syncthreads();
  a = (int)min(base_a + sa - a, (int64_t)cap);
  total_a = (int)min(sum_a, (int64_t)cap);
  b = base_b + sb - b;
}

constexpr int kMostPages = 1 << 29;  // sums of pages are held at it: with a round's 1024 x 2^20 behind they stay in 31 bits

// The first request that names each stream, in claims[n_streams] (LDS); the others count as naming none.
__device__ __forceinline__ void claim_streams(const PageArgs& a, int* claims) {
  for (int s = threadIdx.x; s < a.n_streams; s += blockDim.x) claims[s] = 0x7fffffff;
  __syncthreads();
  for (int i = threadIdx.x; i < a.B; i += blockDim.x) {
    const int s = a.streams[i];
    if (s >= 0 && s < a.n_streams) atomicMin(claims + s, i);
  }
  __syncthreads();
}

// Request i's stream with its length and pages; false where it names none (or not first, or the state is not one).
__device__ __forceinline__ bool request(const PageArgs& a, const int* claims, int i, int& s, int& len, int& count) {
  s = a.streams ? a.streams[i] : i;
  if (s < 0 || s >= a.n_streams) return false;
  len = a.lens[s];
  count = a.counts[s];
  if (a.streams && claims[s] != i) return false;
  return len >= 0 && len <= a.max_len && count >= 0 && count <= a.max_pages;
}

// The pages of a round of requests, one a thread: n of stream s, entries `first` and on of its table, last - off and down in
// the stack; off ascends by their n, and entries [begin, end) are all that there are (s < 0: left out). To the tables, or
// (kBack) to the stack, which leaves -1 in the tables. Every thread of the workgroup calls it. Where some request has
// several, the threads take consecutive entries whoever's they are: a long request does not wait for one thread, and
// lines of memory are shared, of which the CU passes one at a time. Plan and truncation, us, a thread a request / so: one
// stream of 32768 positions in pages of 16 340 / 32; 64 of 4000 74 / 72; 700 of 448 61 / 39; 2500 of 448 193 / 112.
template <int kThreads> struct Moves {
  int off[kThreads], stream[kThreads], delta[kThreads];  // delta: first - off
};
template <bool kBack, int kThreads>
__device__ __forceinline__ void move_pages(const PageArgs& a, Moves<kThreads>& sm, int n, int s, int first, int off, int begin, int end, int last) {
  const int tid = threadIdx.x;
  auto get = [&](int64_t at, int from) { return kBack ? a.tables[at] : a.free_pages[from]; };
  auto put = [&](int64_t at, int from, int32_t page) {
    if (!kBack) {
      a.tables[at] = page;
      return;
    }
    if (from >= 0 && from < a.n_pages) a.free_pages[from] = page;  // counts that are not the state's own stay in bounds
    a.tables[at] = -1;
  };
  sm.off[tid] = off;
  sm.stream[tid] = s;
  sm.delta[tid] = first - off;
  if (!__syncthreads_or(n > 1)) {
    const int64_t at = (int64_t)s * a.max_pages + first;
    if (n == 1) put(at, last - off, get(at, last - off));
    return;
  }
  constexpr int kTrips = 4;
  for (int e0 = begin; e0 < end; e0 += kThreads * kTrips) {
    int64_t at[kTrips];
    int32_t page[kTrips];
#pragma unroll
    for (int u = 0; u < kTrips; ++u) {
      const int e = e0 + kThreads * u + tid;
      int src = 0;  // the last request whose entries begin at e or before
#pragma unroll
      for (int o = kThreads / 2; o >= 1; o >>= 1)
        if (sm.off[src + o] <= e) src += o;
      at[u] = e < end && sm.stream[src] >= 0 ? (int64_t)sm.stream[src] * a.max_pages + sm.delta[src] + e : -1;
      if (at[u] >= 0) page[u] = get(at[u], last - e);
    }
#pragma unroll
    for (int u = 0; u < kTrips; ++u)
      if (at[u] >= 0) put(at[u], last - (e0 + kThreads * u + tid), page[u]);
  }
}

// Slot and position of token t from the finished tables. cu: the B + 1 sums, starts: the positions before them.
__device__ __forceinline__ void emit_token(const PageArgs& a, const int* cu, const int* starts, int t) {
  int64_t slot = -1, pos = 0;
  if (t < cu[a.B]) {
    int lo = 0, hi = a.B;  // the last request that begins at t or before
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int start = starts[lo];
    if (start >= 0) {
      pos = (int64_t)start + t - cu[lo];
      const int s = a.streams ? a.streams[lo] : lo;
      const int page = a.tables[(int64_t)s * a.max_pages + (pos >> a.shift)];
      slot = ((int64_t)page << a.shift) + (pos & ((1 << a.shift) - 1));
    }
  }
  a.slots[t] = slot;
  a.positions[t] = pos;
}

template <int kThreads>
__global__ __launch_bounds__(kThreads) void page_plan_kernel(PageArgs a) {
  extern __shared__ int sm_dyn[];
  __shared__ int64_t sm_a[kThreads / 64];
  // the small form keeps the tokens' sums; the large one's LDS holds the claims of all streams
  constexpr int kSums = kThreads == kSmallThreads ? kThreads : 0;
  __shared__ int sm_b[kThreads / 64], sm_taken, sm_cu[kSums + 1], sm_starts[kSums + 1];
  __shared__ Moves<kThreads> sm_moves;
  int* const claims = sm_dyn;
  const int tid = threadIdx.x;
  if (tid == 0) sm_taken = 0;
  const int top = min(max(*a.n_free, 0), a.n_pages);
  if (a.streams) claim_streams(a, claims);
  else __syncthreads();
  int base_new = 0, base_need = 0, taken = 0;
  for (int i0 = 0; i0 < a.B; i0 += kThreads) {
    const int i = i0 + tid;
    int s = 0, len = 0, count = 0, m = 0, need = 0;
    bool ok = false;
    if (i < a.B) {
      m = a.new_lens ? a.new_lens[i] : a.new_all;
      ok = request(a, claims, i, s, len, count) && m >= 0 && m <= a.max_len - len;
      if (ok) need = max(0, ((len + m + (1 << a.shift) - 1) >> a.shift) - count);
    }
    int cu = min(max(m, 0), a.total), off = need, all_new, all_need;
    scan2(cu, off, a.total, all_new, all_need, sm_a, sm_b);
    cu = min(cu + base_new, a.total);
    off += base_need;
    const int first_need = base_need;
    base_new = min(base_new + all_new, a.total);
    base_need = min(base_need + all_need, kMostPages);
    if (i < a.B) {
      ok = ok && (need == 0 || off + need <= top);
      a.cu[i] = cu;
      a.starts[i] = ok ? len : -1;
      if (kSums) {
        sm_cu[tid] = cu;
        sm_starts[tid] = ok ? len : -1;
      }
      if (ok) {
        if (need) {
          a.counts[s] = count + need;
          taken = off + need;  // ascending over a thread's requests
        }
        a.lens[s] = len + m;
      }
    }
    move_pages<false>(a, sm_moves, ok ? need : 0, ok ? s : -1, count, off, first_need, min(first_need + all_need, top), top - 1);
  }
  if (taken) atomicMax(&sm_taken, taken);
  if (tid == 0) {
    a.cu[a.B] = base_new;
    if (a.B <= kSums) sm_cu[a.B] = base_new;
  }
  __syncthreads();  // this workgroup's writes are visible to it
  if (tid == 0 && sm_taken) *a.n_free = top - sm_taken;
  if (a.emit)
    for (int t = tid; t < a.total; t += kThreads) {
      if (a.B <= kSums) emit_token(a, sm_cu, sm_starts, t);
      else emit_token(a, a.cu, a.starts, t);
    }
}

__global__ __launch_bounds__(256) void page_slots_kernel(PageArgs a) {
  __shared__ int sm_cu[kLdsSums + 1], sm_starts[kLdsSums];
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (a.B > kLdsSums) {
    if (t < a.total) emit_token(a, a.cu, a.starts, t);
    return;
  }
  for (int i = threadIdx.x; i < a.B; i += 256) {
    sm_cu[i] = a.cu[i];
    sm_starts[i] = a.starts[i];
  }
  if (threadIdx.x == 0) sm_cu[a.B] = a.cu[a.B];
  __syncthreads();
  if (t < a.total) emit_token(a, sm_cu, sm_starts, t);
}

// Streams set back to lens_new: the pages behind go back to the stack, in the order that gives the stack of
// before where the plan took them in one call of the same requests.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void page_truncate_kernel(PageArgs a) {
  extern __shared__ int sm_dyn[];
  __shared__ int64_t sm_a[kThreads / 64];
  __shared__ int sm_b[kThreads / 64];
  __shared__ Moves<kThreads> sm_moves;
  int* const claims = sm_dyn;
  const int tid = threadIdx.x;
  const int top = min(max(*a.n_free, 0), a.n_pages);
  if (a.streams) claim_streams(a, claims);
  else __syncthreads();
  auto gone_of = [&](int i, int& s, int& keep) {
    int len, count;
    if (i >= a.B || !request(a, claims, i, s, len, count)) return -1;
    const int n = a.new_lens ? a.new_lens[i] : a.new_all;
    if (n < 0 || n > len) return -1;
    keep = (n + (1 << a.shift) - 1) >> a.shift;
    return max(0, count - keep);
  };
  int total = 0;
  // the sum of all first, where one round of the scan does not hold them
  for (int pass = a.B <= kThreads ? 1 : 0; pass < 2; ++pass) {
    int base = 0;
    for (int i0 = 0; i0 < a.B; i0 += kThreads) {
      int s = 0, keep = 0;
      const int gone = gone_of(i0 + tid, s, keep);
      int unused = 0, off = max(gone, 0), none, all;
      scan2(unused, off, 0, none, all, sm_a, sm_b);
      off += base;
      const int first = base;
      base = min(base + all, kMostPages);
      if (a.B <= kThreads) total = base;
      if (pass == 1) move_pages<true>(a, sm_moves, max(gone, 0), gone >= 0 ? s : -1, keep, off, first, first + all, top + total - 1);
      if (pass == 1 && gone >= 0) {
        a.lens[s] = a.new_lens ? a.new_lens[i0 + tid] : a.new_all;
        if (gone) a.counts[s] = keep;
      }
    }
    total = base;
  }
  if (tid == 0) *a.n_free = min(top + total, a.n_pages);
}

// ---- writes: row t's keys and values to slot slots[t] of every head's page ------------------------------
// A thread moves 16 bytes of a key and of a value; rows whose slot lies outside the cache are left out. Bound: bytes, read and
// written once: 39 us for 21500 rows of 20 heads of 64, 5.6 TB/s, as fast as a large copy.
__global__ __launch_bounds__(256) void page_write_kernel(PageWriteArgs a) {
  const int pieces = a.D / 8;
  const int64_t n = (int64_t)a.T * a.Hk * pieces;
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (idx >= n) return;
  const int p = (int)(idx % pieces);
  const int64_t row = idx / pieces;
  const int h = (int)(row % a.Hk);
  const int64_t t = row / a.Hk;
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= ((int64_t)a.n_pages << a.shift)) return;
  const int64_t page = slot >> a.shift, in = slot & ((1 << a.shift) - 1);
  const int64_t to = (((page * a.Hk + h) << a.shift) + in) * a.D * 2 + p * 16;
  const u32x4 kv = load16(a.k + t * a.ks[0] + h * a.ks[1] + p * 16), vv = load16(a.v + t * a.vs[0] + h * a.vs[1] + p * 16);
  store16(a.k_pages + to, kv);
  store16(a.v_pages + to, vv);
}

}  // namespace

hipError_t launch_page_plan(PageArgs a, hipStream_t stream) {
  const size_t lds = a.streams ? (size_t)a.n_streams * 4 : 0;
  a.emit = a.total <= kPlanThreads;
  if (a.B <= kSmallThreads && a.total <= kSmallThreads) {
    hipLaunchKernelGGL((page_plan_kernel<kSmallThreads>), dim3(1), dim3(kSmallThreads), lds, stream, a);
  } else {
    hipLaunchKernelGGL((page_plan_kernel<kPlanThreads>), dim3(1), dim3(kPlanThreads), lds, stream, a);
    if (!a.emit) hipLaunchKernelGGL(page_slots_kernel, dim3((unsigned)((a.total + 255) / 256)), dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_page_truncate(const PageArgs& a, hipStream_t stream) {
  const size_t lds = a.streams ? (size_t)a.n_streams * 4 : 0;
  if (a.B <= kSmallThreads) hipLaunchKernelGGL((page_truncate_kernel<kSmallThreads>), dim3(1), dim3(kSmallThreads), lds, stream, a);
  else hipLaunchKernelGGL((page_truncate_kernel<kPlanThreads>), dim3(1), dim3(kPlanThreads), lds, stream, a);
  return hipGetLastError();
}

hipError_t launch_page_write(const PageWriteArgs& a, hipStream_t stream) {
  const int64_t n = (int64_t)a.T * a.Hk * (a.D / 8);
  if (n == 0) return hipSuccess;
  hipLaunchKernelGGL(page_write_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace wdrz
