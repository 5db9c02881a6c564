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
#include <hip/hip_runtime.h>
#include <stdint.h>

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
  static __device__ __forceinline__ uint16_t round(float v) { return (uint16_t)pack_bf16x2(v, 0.f); }
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
  static __device__ __forceinline__ uint16_t round(float v) { return (uint16_t)pack_f16x2(v, 0.f); }
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

// Features nb .. nb + 3 of row m: bias and activation in fp32, one rounding.
template <typename T, int ACT>
__device__ __forceinline__ void store4(const Linear4Args& a, int64_t m, int nb, f32x4 acc) {
  const uint16_t* B = static_cast<const uint16_t*>(a.bias);
  uint16_t* y = static_cast<uint16_t*>(a.y) + m * a.y_stride + nb;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (nb + r >= a.N) break;
    float s = acc[r];
    if (B) s += L4<T>::lo(B[nb + r]);
    y[r] = L4<T>::round(ACT ? gelu(s) : s);
  }
}

constexpr int kWaves = 4;

// A workgroup takes 16 features and 16 MT rows; its wavefronts take the 128-input chunks in turn and
// add up through LDS. PART: the chunks of split z only, fp32 sums to part[z][m][n].
template <typename T, int ACT, int MT, bool PART>
__global__ __launch_bounds__(64 * kWaves) void linear4_rows_kernel(Linear4Args a) {
  __shared__ f32x4 red[kWaves][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nt = blockIdx.x, m0 = blockIdx.y * 16 * MT;
  const int li = lane & 15, g = lane >> 4;
  const int chunks = (a.K + 127) / 128;
  const int c0 = PART ? (int)((int64_t)chunks * blockIdx.z / a.n_split) : 0;
  const int c1 = PART ? (int)((int64_t)chunks * (blockIdx.z + 1) / a.n_split) : chunks;
  const u32x4* w = static_cast<const u32x4*>(a.w) + (int64_t)nt * chunks * 64 + lane;
  const int groups = a.K / a.group, gsteps = a.group / 32;  // 32-input steps a group
  const uint16_t* sc = static_cast<const uint16_t*>(a.scales) + (int64_t)nt * groups * 16 + 4 * g;
  const uint16_t* x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    x[t] = static_cast<const uint16_t*>(a.x) + (int64_t)min(m0 + 16 * t + li, a.M - 1) * a.x_stride + 8 * g;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int c = c0 + wave; c < c1; c += kWaves) {
    const u32x4 wq = load16_stream(w + (int64_t)c * 64);
    f32x4 part[MT];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int step = 4 * c + s;
      if (step * 32 >= a.K) break;
      const u32x4 wop = unpack8<T>(wq[s]);
      const bool first = step % gsteps == 0, last = (step + 1) % gsteps == 0;
#pragma unroll
      for (int t = 0; t < MT; ++t)
        part[t] = L4<T>::mfma(wop, load16(x[t] + step * 32), first ? f32x4{0.f, 0.f, 0.f, 0.f} : part[t]);
      if (last) {
        const uint2 q = *reinterpret_cast<const uint2*>(sc + (int64_t)(step / gsteps) * 16);
        const float f[4] = {L4<T>::lo(q.x), L4<T>::hi(q.x), L4<T>::lo(q.y), L4<T>::hi(q.y)};
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[t][r] = __builtin_fmaf(f[r], part[t][r], acc[t][r]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  // red[w][t][lane][r]: feature 4 g + r, row 16 t + li, over wavefront w's chunks
  for (int t = wave; t < MT; t += kWaves) {
    f32x4 s = red[0][t][lane];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) s += red[v][t][lane];
    const int m = m0 + 16 * t + li, nb = nt * 16 + 4 * g;
    if (m >= a.M) continue;
    if constexpr (PART) {
      float* p = a.part + ((int64_t)blockIdx.z * a.M + m) * a.N + nb;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (nb + r < a.N) p[r] = s[r];
    } else {
      store4<T, ACT>(a, m, nb, s);
    }
  }
}

template <typename T, int MT>
void launch_rows(const Linear4Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)), (unsigned)(a.part ? a.n_split : 1));
  if (a.part) hipLaunchKernelGGL((linear4_rows_kernel<T, 0, MT, true>), grid, dim3(64 * kWaves), 0, stream, a);
  else if (a.act) hipLaunchKernelGGL((linear4_rows_kernel<T, 1, MT, false>), grid, dim3(64 * kWaves), 0, stream, a);
  else hipLaunchKernelGGL((linear4_rows_kernel<T, 0, MT, false>), grid, dim3(64 * kWaves), 0, stream, a);
}

template <typename T>
void launch_t(const Linear4Args& a, hipStream_t stream) {
  if (a.M <= 16) launch_rows<T, 1>(a, stream);
  else if (a.M <= 32) launch_rows<T, 2>(a, stream);
  else launch_rows<T, 4>(a, stream);
}

}  // namespace

hipError_t launch_linear4(int dtype, const Linear4Args& a, hipStream_t stream) {
  if (dtype == 2) launch_t<Bf16>(a, stream);
  else launch_t<F16>(a, stream);
  return hipGetLastError();
}

}  // namespace wdrz
