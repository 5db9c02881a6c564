// kv_pages.hip — attention of new tokens over a paged key/value cache, with grouped heads.
//
// o[t, h] = sum_j p_j v_j / sum_j p_j, p_j = 2^(c q[t, h] k_j - m), c = scale log2(e), over the positions j that
// query t sees: j <= n + t behind n cached positions where the call appends its rows, j < n where it only reads.
// Position j of a stream is row j % P of page tables[stream][j / P]; pages are [head][P][D].
//
// A workgroup takes one key/value head of one batch row and up to 16 (query, head of the group) rows, which share
// every key and value: one tile of the 16-row matrix instructions. A wavefront takes 32 positions at a time (two
// tiles of 16, each inside one page, since pages hold a multiple of 16):
//   S^T[key, row] = K Q^T     lane (li, g) = (lane % 16, lane / 16) loads 16 bytes of key 16 t + li, and gets the
//                             scores of keys 16 t + 4 g + 0..3 for row li;
//   O^T[dim, row] += V^T P^T  with the sum's index 8 g + 4 t + r standing for key 16 t + 4 g + r, the scores are the
//                             operand as they lie, and V^T is made in registers: lane (li, g) loads D / 16
//                             consecutive dims of its eight keys, whole rows by 16 lanes, and one v_perm_b32 pairs
//                             two keys of a dim. Nothing goes through LDS before the wavefronts' sums.
// Probabilities are two 16-bit operands (value and remainder, 2^-17 relative), since the matrix cores idle anyway.
// A softmax reference is moved only when a score exceeds it by 2^15. The next block's keys are requested when this one's
// have been used, its values when this one's have been: one block of registers, and loads under way at all times.
// Bound: the bytes of keys and values, for short rows launch and the chain metadata -> table -> keys. One token, bf16,
// in a graph: 52 streams of 224 to 448 positions, 20 heads of 64, 20 us (4.5 TB/s; a large copy reaches 5.2); 4 of 16384 to
// 32768, 32/8 heads of 128, 83 us (4.8 TB/s); one stream of 200 8 us, of which the launch and its host side are most.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kRows = 16;           // (query, group head) rows a workgroup
constexpr int kBlock = 32;          // positions a wavefront takes at a time
constexpr int kLeast = 16;          // positions of the smallest page
constexpr int kPagesMaxSplits = 64;  // workgroups that a row's keys are cut into at most
// A row's reference lies 2^7 below its largest probability, so that the two fp16 operands hold small ones too (2^-32 of
// the largest), and is moved where one exceeds it by 2^15: none leaves fp16.
constexpr float kBelow = 7.f, kMove = 15.f;

template <typename T> struct Pg;
template <> struct Pg<Bf16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u, kNan = 0x7fc07fc0u;
};
template <> struct Pg<F16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return f16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return f16_hi(w); }
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u, kNan = 0x7e007e00u;
};

// Maximum and sum over the lanes li, li + 16, li + 32, li + 48 (every lane gets it).
__device__ __forceinline__ float quarters_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float quarters_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

template <int D> struct VRow;  // D / 16 consecutive dims of a row
template <> struct VRow<64> { typedef u32x2 type; };
template <> struct VRow<128> { typedef u32x4 type; };

template <typename T, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, D == 64 ? 3 : 2) void pages_attn_kernel(PagesArgs a) {
  constexpr int KS = D / 32, NJ = D / 16, kThreads = 64 * kWaves, kRow = D * 2;
  typedef typename VRow<D>::type vrow_t;
  extern __shared__ __attribute__((aligned(16))) float sm_o[];  // [kWaves][rows of the launch][D]
  __shared__ float sm_m[kWaves][kRows], sm_l[kWaves][kRows];
  __shared__ float sm_pm[kPagesMaxSplits][kRows], sm_pl[kPagesMaxSplits][kRows];
  __shared__ int sm_bad, sm_last;

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  // row tiles of one (b, head) next to each other, on one XCD: they read the same keys
  const int unit = a.n_rt > 1 ? remap_xcd((int)blockIdx.x, (int)gridDim.x) : (int)blockIdx.x;
  const int rt = unit % a.n_rt, hk = unit / a.n_rt % a.Hk, b = unit / a.n_rt / a.Hk;
  const int split = blockIdx.y;
  const int r0 = rt * kRows, rows = min(kRows, a.sq * a.G - r0);
  const int row_stride = min(kRows, a.sq * a.G);  // rows of a partial in LDS and the workspace

  const bool has_new = a.kn != nullptr;
  const int stream = a.streams ? a.streams[b] : b;
  const int n = a.seqlens[b];
  const int capacity = a.max_pages << a.shift;
  bool bad = stream < 0 || stream >= a.n_streams || n < 0 || n > capacity - (has_new ? a.sq : 0);
  if (has_new && a.streams) {  // a stream named twice: its rows would read what others write
    bool twice = false;
    for (int i = lane; i < a.B; i += 64) twice = twice || (i != b && a.streams[i] == stream);
    bad = bad || __any(twice);
  }
  auto out_row = [&](int r) {  // r: row of the tile
    const int t = (r0 + r) / a.G, h = hk * a.G + (r0 + r) % a.G;
    return a.o + (int64_t)b * a.os[0] + (int64_t)t * a.os[1] + (int64_t)h * a.os[2];
  };
  if (bad) {
    if (split == 0)
      for (int i = tid; i < rows * (D / 8); i += kThreads)
        store16(out_row(i / (D / 8)) + (i % (D / 8)) * 16, u32x4{Pg<T>::kNan, Pg<T>::kNan, Pg<T>::kNan, Pg<T>::kNan});
    return;
  }
  const int32_t* table = a.tables + (int64_t)stream * a.max_pages;
  const char* knew = has_new ? a.kn + (int64_t)b * a.kns[0] + (int64_t)hk * a.kns[2] : nullptr;
  const char* vnew = has_new ? a.vn + (int64_t)b * a.vns[0] + (int64_t)hk * a.vns[2] : nullptr;
  const int mask = (1 << a.shift) - 1;

  // keys that some row of the tile sees, and this split's part of them
  const int lim_hi = has_new ? n + (r0 + rows - 1) / a.G + 1 : n;
  const int lim_lo = has_new ? n + r0 / a.G + 1 : n;
  const int parts = a.n_splits == 1 ? 1 : min(a.n_splits, max(1, (lim_hi + a.min_chunk - 1) / a.min_chunk));
  const int chunk = ((lim_hi + parts - 1) / parts + kBlock - 1) / kBlock * kBlock;  // whole blocks: there may be fewer parts
  const int n_split_b = max(1, (lim_hi + chunk - 1) / max(chunk, 1));
  if (split >= n_split_b) return;
  const int k0 = split * chunk, k1 = min(lim_hi, k0 + chunk);
  if (tid == 0) sm_bad = 0;

  // the new rows to their pages; every workgroup takes them from the call's own rows
  if (has_new && rt == 0 && split == 0) {
    for (int i = tid; i < a.sq * (D / 8); i += kThreads) {
      const int t = i / (D / 8), p = i % (D / 8), pos = n + t;
      const int page = table[pos >> a.shift];
      if (page < 0 || page >= a.n_pages) continue;
      const int64_t to = ((((int64_t)page * a.Hk + hk) << a.shift) + (pos & mask)) * kRow + p * 16;
      store16(a.k_pages + to, load16(knew + (int64_t)t * a.kns[1] + p * 16));
      store16(a.v_pages + to, load16(vnew + (int64_t)t * a.vns[1] + p * 16));
    }
  }

  // queries: the B operand of S^T
  u32x4 q[KS];
  {
    const int r = r0 + li, t = r / a.G, h = hk * a.G + r % a.G;
    const char* p = a.q + (int64_t)b * a.qs[0] + (int64_t)t * a.qs[1] + (int64_t)h * a.qs[2] + g * 16;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = li < rows ? load16(p + s * 64) : u32x4{0, 0, 0, 0};
  }
  const int lim = has_new ? n + min(r0 + li, r0 + rows - 1) / a.G + 1 : n;  // keys that row li sees

  bool bad_page = false;
  struct Block {
    u32x4 k[2][KS];
    vrow_t v[2][4];
  };
  // Blocks of this wavefront: kb0, kb0 + kWaves, ..; the first n_whole hold cached rows alone, which every row of the tile
  // sees. Lane l holds the page of tile l % 2 of the (l / 2)-th of them from a multiple of 32 on (0 for one behind the
  // keys): the loads of keys wait for no table entry.
  const int kb_end = (k1 + kBlock - 1) / kBlock, kb0 = k0 / kBlock + wave;
  const int n_blocks = kb0 < kb_end ? (kb_end - kb0 + kWaves - 1) / kWaves : 0;
  const int whole_end = min(n, k1) / kBlock, n_whole = kb0 < whole_end ? (whole_end - kb0 + kWaves - 1) / kWaves : 0;
  int ids = 0, ids_at = -1;
  auto places = [&](int i, const char* (&kp)[2], const char* (&vp)[2]) __attribute__((always_inline)) {
    if (i >> 5 != ids_at) {
      ids_at = i >> 5;
      const int pos = (kb0 + (ids_at * 32 + (lane >> 1)) * kWaves) * kBlock + 16 * (lane & 1);
      ids = pos < min(lim_hi, kb_end * kBlock) ? table[pos >> a.shift] : 0;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      int page = __builtin_amdgcn_readlane(ids, (i & 31) * 2 + t);
      if (page < 0 || page >= a.n_pages) {
        bad_page = true;
        page = 0;
      }
      const int64_t at = ((((int64_t)page * a.Hk + hk) << a.shift) + (((kb0 + i * kWaves) * kBlock + 16 * t) & mask)) * kRow;
      kp[t] = a.k_pages + at;
      vp[t] = a.v_pages + at;
    }
  };
  const uint32_t k_off = li * kRow + g * 16, v_off = 4 * g * kRow + li * (D / 8);
  Block x;
  const char* vp[2];  // of the block of the last load_keys
  // Cached rows; behind them the call's own, then none (zeros: what stands there does not count).
  auto load_keys = [&](int i) __attribute__((always_inline)) {
    const char* kp[2];
    places(i, kp, vp);
    if (i < n_whole) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int s = 0; s < KS; ++s) x.k[t][s] = load16(kp[t] + k_off + s * 64);
      return;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = (kb0 + i * kWaves) * kBlock + 16 * t + li;
      const char* p = (key < n ? kp[t] + li * kRow : knew + (int64_t)(key - n) * a.kns[1]) + g * 16;
#pragma unroll
      for (int s = 0; s < KS; ++s) x.k[t][s] = u32x4{0, 0, 0, 0};
      if (key < lim_hi)
#pragma unroll
        for (int s = 0; s < KS; ++s) x.k[t][s] = load16(p + s * 64);
    }
  };
  auto load_values = [&](int i) __attribute__((always_inline)) {  // behind load_keys(i)
    if (i < n_whole) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x.v[t][r] = *reinterpret_cast<const vrow_t*>(vp[t] + v_off + r * kRow);
      return;
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = (kb0 + i * kWaves) * kBlock + 16 * t + 4 * g + r;
        const char* p = (key < n ? vp[t] + (4 * g + r) * kRow : vnew + (int64_t)(key - n) * a.vns[1]) + li * (D / 8);
        x.v[t][r] = vrow_t{};
        if (key < lim_hi) x.v[t][r] = *reinterpret_cast<const vrow_t*>(p);
      }
  };

  f32x4 acc[NJ];  // [j][r]: row li, dim (D / 4) g + (D / 16) r + j
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, mu = 0.f, l = 0.f;  // reference, the same or 0 while there is none, this lane's sum
  auto values = [&](int j, uint32_t low, uint32_t high) __attribute__((always_inline)) {  // dims j, j + NJ, .. of V^T
    u32x4 vt;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        vt[2 * t + i] = __builtin_amdgcn_perm(x.v[t][2 * i + 1][j / 2], x.v[t][2 * i][j / 2], j & 1 ? high : low);
    return vt;
  };
  constexpr uint32_t kLow = 0x05040100u, kHigh = 0x07060302u;  // the low, the high halves of two words

  // The keys of the next block are requested when this one's have been used, its values when this one's have been.
  auto compute = [&](int i) __attribute__((always_inline)) {
    const bool mixed = (kb0 + i * kWaves + 1) * kBlock > lim_lo;  // some rows do not see some keys of the block
    const int sees = lim - (kb0 + i * kWaves) * kBlock - 4 * g;   // key 16 t + r of this lane's: where below
    float p[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < KS; ++e) s = Pg<T>::mfma(x.k[t][e], q[e], s);
#pragma unroll
      for (int r = 0; r < 4; ++r) p[t][r] = 16 * t + r >= sees ? -INFINITY : s[r] * a.c;
    }
    if (i + 1 < n_blocks) load_keys(i + 1);
    const float mx = quarters_max(fmaxf(fmaxf(fmaxf(p[0][0], p[0][1]), fmaxf(p[0][2], p[0][3])),
                                        fmaxf(fmaxf(p[1][0], p[1][1]), fmaxf(p[1][2], p[1][3]))));
    if (__any(mx > m + kMove)) {
      const float to = fmaxf(m, mx - kBelow);
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - to);
      m = to;
      mu = to == -INFINITY ? 0.f : to;
      l *= f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
    }
    u32x4 hi, lo;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float p0 = fast_exp2(p[t][2 * e] - mu), p1 = fast_exp2(p[t][2 * e + 1] - mu);
        l += p0 + p1;
        const uint32_t w = Pg<T>::pack(p0, p1);
        hi[2 * t + e] = w;
        lo[2 * t + e] = Pg<T>::pack(p0 - Pg<T>::lo(w), p1 - Pg<T>::hi(w));
      }
    bool odd = false;
    if (mixed && has_new && a.sq > 1) {
      // 0 times an infinity or NaN that a row does not see would count in the products: such values are taken out
      // of V, and given to the rows that see them. 0 times each value first: 0, or NaN where there is such a one.
      uint32_t low = kLow, high = kHigh;
      asm("" : "+s"(low), "+s"(high));  // made anew below: kept from here they would take the loop's registers
      f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) zero = Pg<T>::mfma(values(j, low, high), u32x4{0, 0, 0, 0}, zero);
      const float any = (zero[0] + zero[1]) + (zero[2] + zero[3]);
      odd = __any(any != any);
    }
    if (odd) {
      u32x4 seen;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) seen[2 * t + e] = Pg<T>::pack(16 * t + 2 * e < sees ? 1.f : 0.f, 16 * t + 2 * e + 1 < sees ? 1.f : 0.f);
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        u32x4 vt = values(j, kLow, kHigh);
#pragma unroll 1
        for (int kind = 0; kind < 3; ++kind) {  // inf, -inf, NaN, as ones
          u32x4 ones;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w = 0;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t u = vt[e] >> (16 * half) & 0xffffu;
              const bool is = kind == 2 ? (u & 0x7fffu) > Pg<T>::kExp : u == (Pg<T>::kExp | (kind ? 0x8000u : 0u));
              w |= is ? Pg<T>::kOne << (16 * half) : 0u;
            }
            ones[e] = w;
          }
          const f32x4 count = Pg<T>::mfma(ones, seen, f32x4{0.f, 0.f, 0.f, 0.f});
          const float value = kind == 2 ? __builtin_nanf("") : kind ? -INFINITY : INFINITY;
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][r] += count[r] > 0.f ? value : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((vt[e] & Pg<T>::kExp) == Pg<T>::kExp) vt[e] &= 0xffff0000u;
          if ((vt[e] >> 16 & Pg<T>::kExp) == Pg<T>::kExp) vt[e] &= 0xffffu;
        }
        acc[j] = Pg<T>::mfma(vt, hi, acc[j]);
        acc[j] = Pg<T>::mfma(vt, lo, acc[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const u32x4 vt = values(j, kLow, kHigh);
        acc[j] = Pg<T>::mfma(vt, hi, acc[j]);
        acc[j] = Pg<T>::mfma(vt, lo, acc[j]);
      }
    }
    if (i + 1 < n_blocks) load_values(i + 1);
  };

  if (n_blocks) {
    load_keys(0);
    load_values(0);
  }
  for (int i = 0; i < n_blocks; ++i) compute(i);
  l = quarters_sum(l);

  // ---- the wavefronts' sums ----
  __syncthreads();  // sm_bad
  if (bad_page && lane == 0) sm_bad = 1;
  if (li < rows) {
    float* o = sm_o + (wave * row_stride + li) * D + (D / 4) * g;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < NJ; j += 4)
        *reinterpret_cast<f32x4*>(o + NJ * r + j) = f32x4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
    if (g == 0) {
      sm_m[wave][li] = m;
      sm_l[wave][li] = l;
    }
  }
  __syncthreads();
  const bool nan = sm_bad != 0;
  auto joined = [&](int r, int d, float& M, float& L) {
    M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, sm_m[w][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(sm_m[w][r] - ref);
      L = __builtin_fmaf(sm_l[w][r], f, L);
      o += *reinterpret_cast<const f32x4*>(sm_o + (w * row_stride + r) * D + d) * f;
    }
    if (nan) L = __builtin_nanf("");
    return o;
  };
  int odd = 0;  // bit u: this thread's u-th dims have NaN that their row's sum has not
  auto put = [&](int i, f32x4 o, float L) __attribute__((always_inline)) {
    const float any = (o[0] + o[1]) + (o[2] + o[3]);
    odd |= any != any && L == L ? 1 << i / kThreads : 0;
    const float f = L == 0.f ? 0.f : 1.f / L;  // a row that sees nothing is 0
    *reinterpret_cast<u32x2*>(out_row(i / (D / 4)) + i % (D / 4) * 8) =
        u32x2{Pg<T>::pack(o[0] * f, o[1] * f), Pg<T>::pack(o[2] * f, o[3] * f)};
  };
  // An infinite value times a probability's two parts, of which the second may be 0 or of the other sign, has become NaN: such
  // dims again, from the values that their row sees, each of which has weight.
  auto infinite = [&]() __attribute__((always_inline)) {
    for (; odd; odd &= odd - 1) {
      // the arguments anew, so that the loop above holds none of them for this
      typedef const __attribute__((address_space(4))) PagesArgs* args_t;
      args_t ap = (args_t)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(ap));
      const int n0 = ap->seqlens[b], stream0 = ap->streams ? ap->streams[b] : b, shift = ap->shift;
      const int32_t* table0 = ap->tables + (int64_t)stream0 * ap->max_pages;
      const int i = tid + (__ffs(odd) - 1) * kThreads, r = i / (D / 4), d = i % (D / 4) * 4;
      const char* vn = ap->kn ? ap->vn + (int64_t)b * ap->vns[0] + (int64_t)hk * ap->vns[2] + d * 2 : nullptr;
      const int seen = ap->kn ? n0 + (r0 + r) / ap->G + 1 : n0;
      uint32_t kinds = 0;  // bits 8 e and on of dim d + e: inf, -inf, NaN
#pragma unroll 1
      for (int key0 = 0; key0 < seen; key0 += kLeast) {  // inside one page
        const char* vp = ap->v_pages + ((((int64_t)table0[key0 >> shift] * ap->Hk + hk) << shift) + (key0 & ((1 << shift) - 1))) * kRow + d * 2;
        u32x2 x[kLeast];
#pragma unroll
        for (int u = 0; u < kLeast; ++u) {
          x[u] = u32x2{0, 0};
          if (key0 + u < seen) x[u] = *reinterpret_cast<const u32x2*>(key0 + u < n0 ? vp + u * kRow : vn + (int64_t)(key0 + u - n0) * ap->vns[1]);
        }
#pragma unroll
        for (int u = 0; u < kLeast; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = x[u][e / 2] >> (16 * (e & 1)) & 0xffffu;
            if ((v & Pg<T>::kExp) == Pg<T>::kExp) kinds |= ((v & 0x7fffu) > Pg<T>::kExp ? 4u : v >> 15 ? 2u : 1u) << (8 * e);
          }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t is = kinds >> (8 * e) & 7u;
        if (is == 1u || is == 2u) *reinterpret_cast<uint16_t*>(out_row(r) + (d + e) * 2) = (uint16_t)(Pg<T>::kExp | (is == 2u ? 0x8000u : 0u));
      }
    }
  };
  if (n_split_b == 1) {
    for (int i = tid; i < rows * (D / 4); i += kThreads) {
      float M, L;
      const f32x4 o = joined(i / (D / 4), i % (D / 4) * 4, M, L);
      put(i, o, L);
    }
    infinite();
    return;
  }
  // ---- several workgroups a row: each publishes its sums, the last to arrive joins them ----
  // Agent-scope stores complete at the device's coherence point; every thread waits for its own (the counter may
  // be seen by another XCD before a store that still travels), then one counts the arrival. No cache is flushed.
  constexpr int kPart = D + 2;  // o[D], reference, sum
  float* part = a.ws_part + (int64_t)unit * a.n_splits * row_stride * kPart;
  for (int i = tid; i < rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float M, L;
    const f32x4 o = joined(r, d, M, L);
    float* pp = part + (split * row_stride + r) * kPart;
#pragma unroll
    for (int e = 0; e < 4; ++e) __hip_atomic_store(pp + d + e, o[e], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (d == 0) {
      __hip_atomic_store(pp + D, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __hip_atomic_store(pp + D + 1, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
  __syncthreads();
  if (tid == 0) sm_last = __hip_atomic_fetch_add(a.ws_count + unit, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n_split_b - 1;
  __syncthreads();
  if (!sm_last) return;
  for (int i = tid; i < n_split_b * rows; i += kThreads) {
    const int s = i / rows, r = i % rows;
    const float* pp = part + (s * row_stride + r) * kPart + D;
    sm_pm[s][r] = __hip_atomic_load(pp, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sm_pl[s][r] = __hip_atomic_load(pp + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  constexpr int kBatch = 8;
  for (int i = tid; i < rows * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < n_split_b; ++s) M = fmaxf(M, sm_pm[s][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < n_split_b; s0 += kBatch) {
      f32x4 x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (s0 + u < n_split_b)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            x[u][e] = __hip_atomic_load(part + ((s0 + u) * row_stride + r) * kPart + d + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (s0 + u < n_split_b) {
          const float f = fast_exp2(sm_pm[s0 + u][r] - ref);
          L = __builtin_fmaf(sm_pl[s0 + u][r], f, L);
          o += x[u] * f;
        }
    }
    put(i, o, L);
  }
  infinite();
  if (tid == 0) __hip_atomic_store(a.ws_count + unit, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
}

template <typename T, int D, int kWaves>
void launch_w(const PagesArgs& a, hipStream_t stream) {
  const size_t lds = (size_t)kWaves * std::min(kRows, a.sq * a.G) * D * 4;
  hipLaunchKernelGGL((pages_attn_kernel<T, D, kWaves>), dim3((unsigned)(a.B * a.Hk * a.n_rt), (unsigned)a.n_splits), dim3(64 * kWaves), lds,
                     stream, a);
}
template <typename T, int D>
void launch_d(const PagesArgs& a, hipStream_t stream) {
  if constexpr (D == 64)
    if (a.waves == 8) return launch_w<T, D, 8>(a, stream);
  if (a.waves == 2) launch_w<T, D, 2>(a, stream);
  else launch_w<T, D, 4>(a, stream);
}

}  // namespace

// How many workgroups a row's keys are cut into (n_splits at most, each of min_chunk keys or more, even parts of the
// row's own length) and the wavefronts of one. Joining costs about 2 us; a workgroup walks 1000 keys in 5 us. So rows are
// cut until there is one workgroup a CU, and further only to hold the time of a long row among short ones. One token, bf16,
// cold caches in a graph, all rows of the same length, us, unsplit / parts of 1024, 512, 256 keys:
//   20 heads of 64: 1 stream of 447 positions 8.8 / - / - / 9.5 (two parts), 1000 11.5 / - / 11.0 / 9.9, 2000 16.9 / 13.8 /
//   11.5 / 10.7; 8 of 4000 35.2 / 38.6 / 37.1 / 40.2 (two parts, the rule's, 38.9); 32 of 4000 125 / 126 / 123 / 128;
//   32/8 heads of 128: 1 of 32000 390 / 34.8 / 40.0 / -; 4 of 32000 412 / 102 / 109 / - (eight parts 95, 5.5 TB/s); 16 of 2000
//   34.4 / 29.8 / 30.2 / 31.4; 32 of 2000 50.5 / 53.0 / 54.3 / 60.6.
// Wavefronts, rows of 440, us of 2 / 4 / 8: 160 workgroups 13.2 / 10.6 / 10.1, 260 16.0 / 13.9 / 17.5, 520 18.4 / 18.7 / 25.4,
// 800 23.7 / 26.7 / 33.9, 1280 33.0 / 35.1 / 44.4.
constexpr int64_t kCus = 256;
void pages_plan(int64_t B, int64_t sq, int64_t H, int64_t Hk, int64_t D, int64_t max_len, PagesArgs* a) {
  a->G = (int)(H / Hk);
  a->n_rt = (int)((sq * a->G + kRows - 1) / kRows);
  const int64_t units = B * Hk * a->n_rt;
  int64_t least = max_len, splits = 1;
  if (units <= kPagesCounters && max_len > 512) {
    least = units >= kCus ? std::max<int64_t>(4096, (max_len + kPagesMaxSplits - 1) / kPagesMaxSplits) : 256;
    splits = (max_len + least - 1) / least;
    if (units < kCus) splits = std::min<int64_t>(std::min<int64_t>(splits, (kCus + units - 1) / units), kPagesMaxSplits / 2);
  }
  a->n_splits = (int)splits;
  a->min_chunk = (int)least;
  a->waves = units * splits <= 160 && D == 64 ? 8 : units * splits < 768 ? 4 : 2;
}

size_t pages_workspace_bytes(int64_t B, int64_t sq, int64_t H, int64_t Hk, int64_t D, int64_t max_len) {
  PagesArgs a{};
  pages_plan(B, sq, H, Hk, D, max_len, &a);
  if (a.n_splits == 1) return 0;
  return kPagesCounters * 4 + (size_t)B * Hk * a.n_rt * a.n_splits * std::min<int64_t>(kRows, sq * a.G) * (D + 2) * 4;
}

hipError_t launch_pages(int dtype, int D, const PagesArgs& a, hipStream_t stream) {
  if (D == 64) {
    if (dtype == 2) launch_d<Bf16, 64>(a, stream);
    else launch_d<F16, 64>(a, stream);
  } else {
    if (dtype == 2) launch_d<Bf16, 128>(a, stream);
    else launch_d<F16, 128>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace wdrz
