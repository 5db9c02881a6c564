// linear4.hip — linears with 4-bit weights: Y = act(X (s Q)^T + b).
//
// Q holds whole numbers -7..7, s one 16-bit scale for each output feature and group of G inputs (G 32, 64
// or 128). For the decode step's few rows the product is bound by reading the weights, here a quarter of
// the 16-bit ones and their scales.
//
// Weights are laid out once as the matrix cores take them: tile (16 features, 128 inputs) is 64 lanes x
// 16 bytes, lane l = 16 g + n holding feature n; its dword s holds inputs 32 s + 8 g .. + 7, byte i of
// it input i in the low half and input 4 + i in the high half, each as sign and magnitude. So a
// wavefront reads a tile with one fully coalesced load a lane, and a dword becomes one 16x16x32 operand:
// the magnitudes are looked up as e4m3 bytes (one v_perm_b32 for four), the sign is bit 7, and two bytes
// an instruction widen to bf16 or fp16, exactly. Scales stand as [feature tile][group][16]; each group's
// product is summed in fp32 from zero and then multiplied by its scale in fp32, so nothing is rounded
// before the one rounding of the result.
//
// Bound: few rows, launch and one trip to memory (1 row of 1280 x 5120 4.2-4.7 us for 3.5 MB; in turn
// instead of together the trips took 6.6); a large vocabulary, the weights' stream (1 row of 1280 x 51866
// 12.4 us, 2.8 TB/s); many rows, matrix products and lookups issued in turn (3584 rows of 5120 x 1280 59 us at groups
// of 128, 800 TFLOP/s; 66 at 64, whose sums are scaled twice as often, 84 at 32; the 16-bit library product 53-59).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

template <typename T> struct L4;
template <> struct L4<Bf16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
template <> struct L4<F16> {
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t widen(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  }
  static __device__ __forceinline__ float lo(uint32_t w) { return f16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return f16_hi(w); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
};

// e4m3 of 0..7: 0x00 0x38 0x40 0x44 | 0x48 0x4a 0x4c 0x4e
constexpr uint32_t kMag03 = 0x44403800u, kMag47 = 0x4e4c4a48u;

// Eight weights of one packed dword as a 16-bit matrix operand.
template <typename T>
__device__ __forceinline__ u32x4 unpack8(uint32_t w) {
  const uint32_t hi = w >> 4;
  const uint32_t a = __builtin_amdgcn_perm(kMag47, kMag03, w & 0x07070707u) | ((w << 4) & 0x80808080u);
  const uint32_t b = __builtin_amdgcn_perm(kMag47, kMag03, hi & 0x07070707u) | (w & 0x80808080u);
  return u32x4{L4<T>::widen(a, false), L4<T>::widen(a, true), L4<T>::widen(b, false), L4<T>::widen(b, true)};
}

__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }

// The bias of features nb .. nb + 3, in fp32 (requested with the operands: at the end each would be a
// trip to memory of its own).
template <typename T>
__device__ __forceinline__ f32x4 bias4(const Linear4Args& a, int nb) {
  const uint16_t* B = static_cast<const uint16_t*>(a.bias);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (!B) return v;
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = L4<T>::lo(B[min(nb + r, a.N - 1)]);
  return v;
}

// Features nb .. nb + 3 of row m: bias and activation in fp32, one rounding; or fp32 sums of split z.
template <typename T, int ACT, bool PART>
__device__ __forceinline__ void put4(const Linear4Args& a, int z, int64_t m, int nb, f32x4 v, f32x4 bias) {
  if constexpr (PART) {
    float* p = a.part + (z * (int64_t)a.M + m) * a.N + nb;
    if (a.vec) {
      *reinterpret_cast<f32x4*>(p) = v;
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nb + r < a.N) p[r] = v[r];
  } else {
    uint16_t* y = static_cast<uint16_t*>(a.y) + m * a.y_stride + nb;
    v += bias;
    if constexpr (ACT != 0)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = gelu(v[r]);
    const u32x2 w = {L4<T>::pack(v[0], v[1]), L4<T>::pack(v[2], v[3])};
    if (a.vec) {
      *reinterpret_cast<u32x2*>(y) = w;
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (nb + r < a.N) y[r] = (uint16_t)(w[r >> 1] >> (16 * (r & 1)));
  }
}

// ---- few rows -------------------------------------------------------------------------------------
// A workgroup takes 16 NT features and 16 MT rows; its wavefronts take the 128-input chunks in turn and
// add up through LDS. NB chunks' weights, activations and scales are requested together, so a short K
// is one trip to memory. GS: 32-input steps a group. PART: the chunks of split z only, fp32 sums to
// part[z][m][n].
template <typename T, int ACT, bool PART, int GS, int MT, int NT, int NB, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void linear4_rows_kernel(Linear4Args a) {
  __shared__ f32x4 red[kWaves][NT * MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt0 = blockIdx.x * NT, m0 = blockIdx.y * 16 * MT;
  const int li = lane & 15, g = lane >> 4;
  const int steps = a.K / 32, chunks = (a.K + 127) / 128, groups = steps / GS, tiles = (a.N + 15) / 16;
  const int c0 = PART ? (int)((int64_t)chunks * blockIdx.z / a.n_split) : 0;
  const int c1 = PART ? (int)((int64_t)chunks * (blockIdx.z + 1) / a.n_split) : chunks;
  const u32x4* w[NT];
  const uint16_t* sc[NT];
  f32x4 bias[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {  // tiles past N re-read the last one and are not stored
    const int64_t nt = NT == 1 ? nt0 : min(nt0 + j, tiles - 1);
    w[j] = static_cast<const u32x4*>(a.w) + nt * chunks * 64 + lane;
    sc[j] = static_cast<const uint16_t*>(a.scales) + nt * groups * 16 + 4 * g;
    bias[j] = bias4<T>(a, (int)nt * 16 + 4 * g);
  }
  const uint16_t* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    x[t] = static_cast<const uint16_t*>(a.x) + (int64_t)min(m0 + 16 * t + li, a.M - 1) * a.x_stride + 8 * g;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int cb = c0 + wave; cb < c1; cb += kWaves * NB) {
    u32x4 wq[NB][NT], xv[NB][4][MT];
    uint2 sq[NB][NT][4 / GS];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = cb + i * kWaves;
      if (c < c1)
#pragma unroll
        for (int j = 0; j < NT; ++j) wq[i][j] = load16_stream(w[j] + (int64_t)c * 64);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = cb + i * kWaves;
      if (c < c1) {  // steps past K re-read its last one and are left out below
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int t = 0; t < MT; ++t) xv[i][s][t] = load16(x[t] + min(4 * c + s, steps - 1) * 32);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 4 / GS; ++q)
            sq[i][j][q] = *reinterpret_cast<const uint2*>(sc[j] + (int64_t)min(c * (4 / GS) + q, groups - 1) * 16);
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = cb + i * kWaves;
      if (c < c1) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          f32x4 part[MT];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            if (4 * c + s < steps) {
              const u32x4 wop = unpack8<T>(wq[i][j][s]);
#pragma unroll
              for (int t = 0; t < MT; ++t)
                part[t] = L4<T>::mfma(wop, xv[i][s][t], s % GS == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[t]);
              if (s % GS == GS - 1) {
                const uint2 q = sq[i][j][s / GS];
                const float f[4] = {L4<T>::lo(q.x), L4<T>::hi(q.x), L4<T>::lo(q.y), L4<T>::hi(q.y)};
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                  for (int r = 0; r < 4; ++r) acc[j][t][r] = __builtin_fmaf(f[r], part[t][r], acc[j][t][r]);
              }
            }
          }
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) red[wave][j * MT + t][lane] = acc[j][t];
  __syncthreads();
  // red[w][j MT + t][lane][r]: feature 16 j + 4 g + r, row 16 t + li, over wavefront w's chunks
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if ((j * MT + t) % kWaves != wave || nt0 + j >= tiles) continue;
      f32x4 s = red[0][j * MT + t][lane];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) s += red[v][j * MT + t][lane];
      const int m = m0 + 16 * t + li;
      if (m < a.M) put4<T, ACT, PART>(a, blockIdx.z, m, (nt0 + j) * 16 + 4 * g, s, bias[j]);
    }
}

// ---- many rows --------------------------------------------------------------------------------------
// A workgroup takes 64 WM rows and 16 WN NT features; each of its wavefronts 64 rows, 16 NT features and
// every KH-th chunk of 128 inputs, so that a SIMD has wavefronts to overlap (one's lookups with another's
// matrix products) even where there are no more tiles than CUs. A stage is KH chunks: the activations go
// from memory into one of two LDS buffers without passing through registers while the other is computed,
// each wavefront's weights of the next stage into the registers that this one's leave. The KH sums of an
// output are added through LDS at the end.
// LDS rows are 16 KH pieces of 16 bytes, piece p of row r at place p ^ (r % 16): the 16 rows that a
// quarter wavefront reads a piece of lie in different banks.
template <int WM, int WN, int KH, int NT>
constexpr int tile_lds() {
  const int x = 2 * 64 * WM * 256 * KH, red = (KH - 1) * WM * WN * NT * 4 * 64 * 16;
  return x > red ? x : red;
}

// 16 bytes a lane from memory to LDS, lane l to `to` + 16 l (`to` the same in every lane).
__device__ __forceinline__ void load16_lds(const void* from, char* to) {
#if __HIP_DEVICE_COMPILE__
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(uintptr_t)from,
                                   (__attribute__((address_space(3))) void*)(uint32_t)(uintptr_t)to, 16, 0, 0);
#else
  (void)from, (void)to;
#endif
}

template <typename T, int ACT, bool PART, int GS, int WM, int WN, int KH, int NT>
__global__ __launch_bounds__(64 * WM * WN * KH) void linear4_tile_kernel(Linear4Args a) {
  constexpr int kWaves = WM * WN * KH, kRows = 64 * WM, kPitch = 256 * KH, kBuf = kRows * kPitch;
  constexpr int kLoads = kBuf / (1024 * kWaves);
  __shared__ __attribute__((aligned(1024))) char smem[tile_lds<WM, WN, KH, NT>()];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int li = lane & 15, g = lane >> 4;
  const int nw = wave % WN, mw = wave / WN % WM, kh = wave / (WN * WM);
  const int steps = a.K / 32, chunks = (a.K + 127) / 128, groups = steps / GS, tiles = (a.N + 15) / 16;
  const int c0 = PART ? (int)((int64_t)chunks * blockIdx.z / a.n_split) : 0;
  const int c1 = PART ? (int)((int64_t)chunks * (blockIdx.z + 1) / a.n_split) : chunks;
  // feature blocks fastest, neighbours on one XCD: they share the activations in its L2
  const int n_blocks = (tiles + WN * NT - 1) / (WN * NT);
  const int id = remap_xcd((int)blockIdx.x, (int)gridDim.x);
  const int m0 = id / n_blocks * kRows, nt0 = (id % n_blocks * WN + nw) * NT;

  const char* xb0 = static_cast<const char*>(a.x) + (int64_t)m0 * a.x_stride * 2;
  const int x_step = (int)(a.x_stride * 2), m_last = a.M - 1 - m0;  // 128 rows' bytes fit 31 bits (launcher)
  auto fetch_x = [&](int c, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int at = (i * kWaves + wave) * 1024;
      const int r = (at + lane * 16) / kPitch, p = (at + lane * 16) % kPitch / 16 ^ (r & 15);
      load16_lds(xb0 + min(r, m_last) * x_step + min(c * 128 + p * 8, a.K - 8) * 2, smem + buf * kBuf + at);
    }
  };
  u32x4 wq[NT];
  uint2 ws[NT][4 / GS];
  auto fetch_w = [&](int c, int j) __attribute__((always_inline)) {  // tiles past N re-read the last one, not stored
    const int64_t t = min(nt0 + j, tiles - 1);
    c = min(c + kh, chunks - 1);
    wq[j] = load16(static_cast<const char*>(a.w) + (t * chunks + c) * 1024 + lane * 16);
#pragma unroll
    for (int q = 0; q < 4 / GS; ++q)
      ws[j][q] = *reinterpret_cast<const uint2*>(static_cast<const char*>(a.scales) +
                                                 (t * groups + min(c * (4 / GS) + q, groups - 1)) * 32 + g * 8);
  };
  f32x4 acc[NT][4];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  // One stage. LAST: nothing is fetched, and chunks and inputs past the end are left out (the activations
  // there are copies of others, and 0 times an infinity would count).
  auto stage = [&](int c, int buf, auto last) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last)::value;
    const char* from = smem + buf * kBuf + (mw * 64 + li) * kPitch;
    u32x4 xb[4][4];
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        xb[s][t] = *reinterpret_cast<const u32x4*>(from + 16 * t * kPitch + (kh * 16 + ((4 * s + g) ^ li)) * 16);
    __builtin_amdgcn_sched_barrier(0);  // before the fetch: reads behind it would wait for it
    if (!LAST) fetch_x(c + KH, buf ^ 1);
    // the next tile's lookups between this one's products; no further ahead, or they take all registers
    // (nor at all where 32-input groups' scales need them: 5 tiles would spill)
    constexpr bool AHEAD = GS > 1 || NT < 5;
    u32x4 wop[2][4];
    if (AHEAD) {
#pragma unroll
      for (int s = 0; s < 4; ++s) wop[0][s] = unpack8<T>(wq[0][s]);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      f32x4 part[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (!AHEAD) wop[j & 1][s] = unpack8<T>(wq[j][s]);
        if (!LAST || 4 * (c + kh) + s < min(steps, 4 * c1)) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
            part[t] = L4<T>::mfma(wop[j & 1][s], xb[s][t], s % GS == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : part[t]);
          if (s % GS == GS - 1) {
            const uint2 q = ws[j][s / GS];
            const float f[4] = {L4<T>::lo(q.x), L4<T>::hi(q.x), L4<T>::lo(q.y), L4<T>::hi(q.y)};
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[j][t][r] = __builtin_fmaf(f[r], part[t][r], acc[j][t][r]);
          }
        }
        if (AHEAD && j + 1 < NT) wop[(j + 1) & 1][s] = unpack8<T>(wq[j + 1][s]);
      }
      if (!LAST) fetch_w(c + KH, j);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (!LAST) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wavefront's part of the next stage is in LDS
      __syncthreads();
    }
  };
  if (c0 < c1) {
    fetch_x(c0, 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) fetch_w(c0, j);
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
    int c = c0, buf = 0;
    for (; c + KH < c1; c += KH, buf ^= 1) stage(c, buf, std::false_type{});
    stage(c, buf, std::true_type{});
  }
  if (KH > 1) __syncthreads();
  if constexpr (KH > 1) {
    f32x4* red = reinterpret_cast<f32x4*>(smem) + ((mw * WN + nw) * (KH - 1) * NT * 4) * 64 + lane;
    if (kh > 0) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) red[(((kh - 1) * NT + j) * 4 + t) * 64] = acc[j][t];
    }
    __syncthreads();
    if (kh > 0) return;
#pragma unroll
    for (int z = 0; z < KH - 1; ++z)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) acc[j][t] += red[((z * NT + j) * 4 + t) * 64];
  }
  f32x4 bias[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) bias[j] = bias4<T>(a, (nt0 + j) * 16 + 4 * g);
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int m = m0 + mw * 64 + 16 * t + li;
      if (m < a.M && nt0 + j < tiles) put4<T, ACT, PART>(a, blockIdx.z, m, (nt0 + j) * 16 + 4 * g, acc[j][t], bias[j]);
    }
}

template <typename T, int ACT, bool PART, int GS, int WM, int WN, int KH, int NT>
void launch_tile(const Linear4Args& a, hipStream_t stream) {
  const int64_t m = (a.M + 64 * WM - 1) / (64 * WM), n = ((a.N + 15) / 16 + WN * NT - 1) / (WN * NT);
  const dim3 grid((unsigned)(m * n), 1, (unsigned)(PART ? a.n_split : 1));
  hipLaunchKernelGGL((linear4_tile_kernel<T, ACT, PART, GS, WM, WN, KH, NT>), grid, dim3(64 * WM * WN * KH), 0, stream, a);
}

template <typename T, int ACT, bool PART, int GS, int MT, int NT, int NB, int W>
void launch_rows(const Linear4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)),
                  (unsigned)(PART ? a.n_split : 1));
  hipLaunchKernelGGL((linear4_rows_kernel<T, ACT, PART, GS, MT, NT, NB, W>), grid, dim3(64 * W), 0, stream, a);
}

// Time of a tile launch in us, from how many workgroups run at once and how long one takes over `chunks`
// chunks: `step` a chunk beside `fixed` for start, sum and stores; `both`: two workgroups fit a CU. The constants are
// fits to K of 1280 and 5120. Held against all three tiles at 44 shapes (136 to 3584 rows, 384 to 5120 inputs and
// features, every group) the choice was the fastest or within 3% of it in 40, within 7% in the others.
double tile_cost(int64_t wgs, double fixed, double step, double chunks, bool both) {
  const double t = fixed + step * chunks;
  if (!both) return (double)((wgs + 255) / 256) * t;
  const int64_t rem = wgs % 512;
  return (double)(wgs / 512) * 1.25 * t + (rem == 0 ? 0. : rem <= 256 ? t : 1.45 * t);
}

// Which kernel, by what it takes at these sizes (bf16, cold weights in a graph, us):
//   * up to 16 rows: one row tile; eight wavefronts share a short K, sixteen a long one (1 row: 1280 x 1280
//     3.7, 1280 x 5120 4.4-5.0, 5120 x 1280 5.5-6.4). From some 450 tiles of features on a workgroup takes two
//     of them, and above 2048 four, which share its activations (1 / 16 rows, one tile a workgroup of four
//     wavefronts, then as here: 2560 x 7680 6.6 / 8.9, 6.5 / 7.2; 1280 x 24576 8.9 / 13.9, 7.9 / 9.8;
//     1280 x 51866 13.2 / 23.6, 12.4 / 16.4). Below, two cost more: 1280 x 3840 4.3, and 5.4 with two;
//   * blocks of 32 rows while the launch has about as many workgroups as CUs, up to twice as many for a
//     short K: 52 rows 1280 x 1280 5.2, x 3840 7.2, 5120 x 1280 12.4; 128 rows of 5120 x 1280 (320
//     workgroups) 23.4, and 18.8 in tiles; 64 rows of 1280 x 5120 (640) 10.9, and 8.0 in tiles;
//   * tiles of 64 x 64, 64 x 128 or 128 x 160, by the sum of their rounds. A round over 10 / 40 chunks, groups
//     of 128: 64 x 64 8.0 / 19.3, 64 x 128 13.3 / 36.7, 128 x 160 20 / 59; of 32: 9 / 23, 17.4 / 56, 26 / 83.
//     3584 rows: 1280 x 5120 121 / 75 / 79, 5120 x 1280 87 / 77 / 60 (784 TFLOP/s; in 32-row blocks 360).
template <typename T, int ACT, bool PART, int GS>
void launch_g(const Linear4Args& a, hipStream_t stream) {
  const int64_t tiles = (a.N + 15) / 16, splits = PART ? a.n_split : 1;
  const int chunks = (int)((a.K + 127) / 128 / splits);
  if (a.M <= 16) {
    const int64_t wgs = tiles * splits;
    if (wgs > 2048) launch_rows<T, ACT, PART, GS, 1, 4, 1, 4>(a, stream);
    else if (wgs > 1024) launch_rows<T, ACT, PART, GS, 1, 2, 2, 4>(a, stream);
    else if (wgs > 448) launch_rows<T, ACT, PART, GS, 1, 2, 2, 8>(a, stream);
    else if (chunks <= 16) launch_rows<T, ACT, PART, GS, 1, 1, 3, 8>(a, stream);
    else launch_rows<T, ACT, PART, GS, 1, 1, 3, 16>(a, stream);
    return;
  }
  const int64_t blocks32 = (a.M + 31) / 32 * tiles * splits;
  // a tile's rows are addressed by 31-bit offsets
  if (blocks32 <= 256 || (blocks32 <= 512 && a.K <= 2048) || a.x_stride > (1 << 22)) {
    launch_rows<T, ACT, PART, GS, 2, 1, 2, 8>(a, stream);
    return;
  }
  auto wgs = [&](int rows, int feats) { return (int64_t)((a.M + rows - 1) / rows) * ((a.N + feats - 1) / feats) * splits; };
  const double c5 = tile_cost(wgs(64, 64), 4.2, GS == 1 ? 0.47 : GS == 2 ? 0.40 : 0.38, chunks, false);
  const double c4 = tile_cost(wgs(64, 128), 5.0, GS == 1 ? 1.28 : GS == 2 ? 0.88 : 0.79, chunks, true);
  const double c1 = tile_cost(wgs(128, 160), 7.0, GS == 1 ? 1.90 : GS == 2 ? 1.46 : 1.29, chunks, false);
  if (c5 <= c4 && c5 <= c1) launch_tile<T, ACT, PART, GS, 1, 2, 4, 2>(a, stream);
  else if (c4 <= c1) launch_tile<T, ACT, PART, GS, 1, 2, 2, 4>(a, stream);
  else launch_tile<T, ACT, PART, GS, 2, 2, 2, 5>(a, stream);
}

template <typename T, int ACT, bool PART>
void launch_p(const Linear4Args& a, hipStream_t stream) {
  if (a.group == 32) launch_g<T, ACT, PART, 1>(a, stream);
  else if (a.group == 64) launch_g<T, ACT, PART, 2>(a, stream);
  else launch_g<T, ACT, PART, 4>(a, stream);
}

template <typename T>
void launch_t(const Linear4Args& a, hipStream_t stream) {
  if (a.part) launch_p<T, 0, true>(a, stream);
  else if (a.act) launch_p<T, 1, false>(a, stream);
  else launch_p<T, 0, false>(a, stream);
}

}  // namespace

hipError_t launch_linear4(int dtype, Linear4Args a, hipStream_t stream) {
  a.vec = a.N % 16 == 0 && (a.part || (a.y_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0));
  if (dtype == 2) launch_t<Bf16>(a, stream);
  else launch_t<F16>(a, stream);
  return hipGetLastError();
}

}  // namespace wdrz
