// packed.hip — attention of packed sequences of different lengths, with grouped heads: no padding between them.
//
// Sequence i is rows cu_q[i] .. cu_q[i + 1] - 1 of the queries and cu_k[i] .. cu_k[i + 1] - 1 of the keys and values.
// Its query t sees all its keys, or under the causal mask those at t + (keys - queries) and before; a query that
// sees none gives zeros. Query head h reads key/value head h / (H / Hk).
//
// A workgroup takes 128 QB queries of one head, a wavefront 32 QB of them (QB blocks of 32), over tiles of 64 keys
// that pass through registers into one of two LDS buffers while the other is computed. As in the encoder's
// attention the products are transposed, S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 matrix instructions, with
// the keys' rows permuted so that the scores of a lane are already the operand of the second product, and V^T is
// read from row-major V by transposing LDS reads.
//
// Softmax: p = 2^(c s - m) in fp32 with a reference m per query, taken from the first 32 keys and moved only
// where a lane's 16 probabilities sum to more than 2^10 (some exceeds 2^6): no maximum is taken otherwise. Every
// query that sees any key sees the first, so the first keys give a reference.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kTile = 64;           // keys a stage
constexpr int kSub = 32;            // keys a step
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kSumLimit = 1024.f;

template <typename T> struct Pk;
template <> struct Pk<Bf16> {
  typedef bf16x8 op_t;
  static __device__ __forceinline__ f32x16 mfma(op_t a, op_t b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float one(uint16_t w) { return bf16_lo(w); }
  static constexpr uint32_t kExp = 0x7f80u;
};
template <> struct Pk<F16> {
  typedef f16x8 op_t;
  static __device__ __forceinline__ f32x16 mfma(op_t a, op_t b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ float one(uint16_t w) { return f16_lo(w); }
  static constexpr uint32_t kExp = 0x7c00u;
};

// max of x over the two 32-lane halves of the wavefront (every lane gets the result)
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Within each 16-lane group, lane i gets element i % 4 of the 8-byte pieces that lanes 4 c + i / 4 (c = 0..3) of
// its group point at: row-major [key][dim] rows become the dim-major operand. p points into LDS.
__device__ __forceinline__ u32x2 read_tr(const uint16_t* p) {
#if __HIP_DEVICE_COMPILE__
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uint32_t)(uintptr_t)p));
#else
  (void)p;
  return u32x2{0, 0};
#endif
}

// Sequence and query block of the work item `idx`, blocks of a sequence counted from its end (under the mask the
// last needs the most keys), sequences from the last; false where there is none. Every lane of a wavefront calls it.
struct Item {
  int q0, nq, k0, nk, block;
};
__device__ __forceinline__ bool find_item(const PackedArgs& a, int rows, int idx, Item& it) {
  const int lane = threadIdx.x & 63;
  for (int i0 = 0; i0 < a.B; i0 += 64) {
    const int i = a.B - 1 - i0 - lane;
    int c0 = 0, c1 = 0;
    if (i >= 0) {
      c0 = min(max(a.cu_q[i], 0), a.T);  // sums that are not ascending or in range stay in bounds
      c1 = min(max(a.cu_q[i + 1], c0), a.T);
    }
    const int n = (c1 - c0 + rows - 1) / rows;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(sum, o);
      if (lane >= o) sum += u;
    }
    const int total = __shfl(sum, 63);
    if (idx < total) {
      const uint64_t here = __ballot(idx < sum);
      const int src = __ffsll((unsigned long long)here) - 1;
      const int s = __builtin_amdgcn_readfirstlane(a.B - 1 - i0 - src);
      it.q0 = __builtin_amdgcn_readfirstlane(__shfl(c0, src));
      it.nq = __builtin_amdgcn_readfirstlane(__shfl(c1, src)) - it.q0;
      it.block = __builtin_amdgcn_readfirstlane(__shfl(sum, src) - 1 - idx);
      it.k0 = min(max(a.cu_k[s], 0), a.Tk);
      it.nk = min(max(a.cu_k[s + 1], it.k0), a.Tk) - it.k0;
      return true;
    }
    idx -= total;
  }
  return false;
}

template <typename T, int D, int QB>
__global__ __launch_bounds__(kThreads, 2) void packed_attn_kernel(PackedArgs a) {
  typedef typename Pk<T>::op_t op_t;
  typedef uint16_t e_t;
  constexpr int kBM = 32 * QB * kWaves, kPitch = D + 8, KS = D / 16, DB = D / 32;
  constexpr int kPieces = kTile * D / 8 / kThreads;  // 16-byte pieces a thread and tile
  __shared__ __attribute__((aligned(16))) e_t sK[2][kTile * kPitch];
  __shared__ __attribute__((aligned(16))) e_t sV[2][kTile * kPitch];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  // heads fastest, the heads of different groups side by side: with a multiple of eight groups a group's heads run
  // on one XCD and share its L2
  const int hid = (int)blockIdx.x % a.H, idx = (int)blockIdx.x / a.H;
  const int hk = hid % a.Hk, h = hk * (a.H / a.Hk) + hid / a.Hk;
  Item it;
  if (!find_item(a, kBM, idx, it)) return;

  const int q_wg = it.block * kBM, q_wave = q_wg + wave * 32 * QB;
  const int shift = a.causal ? it.nk - it.nq : 0;  // query t sees the keys up to t + shift
  const int k_lim = a.causal ? max(0, min(it.nk, min(q_wg + kBM, it.nq) + shift)) : it.nk;
  const int n_tiles = (k_lim + kTile - 1) / kTile;
  const int w_lim = a.causal ? max(0, min(k_lim, q_wave + 32 * QB + shift)) : it.nk;  // keys of this wavefront
  const int n_sub = (w_lim + kSub - 1) / kSub;

  const char* Q = a.q + (int64_t)it.q0 * a.qs[0] + (int64_t)h * a.qs[1];
  const char* K = a.k + (int64_t)it.k0 * a.ks[0] + (int64_t)hk * a.ks[1];
  const char* V = a.v + (int64_t)it.k0 * a.vs[0] + (int64_t)hk * a.vs[1];

  op_t q[QB][KS];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int t = min(q_wave + qb * 32 + l32, it.nq - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) q[qb][s] = __builtin_bit_cast(op_t, load16(Q + (int64_t)t * a.qs[0] + s * 32 + hl * 16));
  }

  u32x4 rk[kPieces], rv[kPieces];
  auto fetch = [&](int tile) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = tid + i * kThreads, row = piece / (D / 8), p = piece % (D / 8), key = tile * kTile + row;
      rk[i] = rv[i] = u32x4{0, 0, 0, 0};  // behind the sequence: another's rows, which must not count
      if (key < it.nk) {
        rk[i] = load16(K + (int64_t)key * a.ks[0] + p * 16);
        rv[i] = load16(V + (int64_t)key * a.vs[0] + p * 16);
      }
    }
  };
  auto stage = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = tid + i * kThreads, row = piece / (D / 8), p = piece % (D / 8);
      *reinterpret_cast<u32x4*>(&sK[buf][row * kPitch + p * 8]) = rk[i];
      *reinterpret_cast<u32x4*>(&sV[buf][row * kPitch + p * 8]) = rv[i];
    }
  };

  // K operand: key row 8 i + 4 j + e of a step stands at row 16 (i / 2) + 8 j + 4 (i % 2) + e, so that score x of a
  // lane is key 16 (x / 8) + 8 hl + x % 8
  const int k_off = (16 * (l32 >> 4) + 8 * ((l32 >> 2) & 1) + 4 * ((l32 >> 3) & 1) + (l32 & 3)) * kPitch + hl * 8;
  const int g16 = lane >> 4, j16 = lane & 15;
  const int v_off = (8 * (g16 >> 1) + (j16 >> 2)) * kPitch + 16 * (g16 & 1) + 4 * (j16 & 3);

  f32x16 acc[DB][QB];  // O^T: query l32 of block qb, dim 32 db + 8 (x / 4) + 4 hl + x % 4
  float m[QB], l[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m[qb] = l[qb] = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[db][qb][x] = 0.f;
  }

  auto step = [&](int s, int buf) __attribute__((always_inline)) {
    const int base = s * kSub;
    const e_t* kb = &sK[buf][(s & 1) * kSub * kPitch + k_off];
    const e_t* vb = &sV[buf][(s & 1) * kSub * kPitch + v_off];
    const bool edge = base + kSub > (a.causal ? min(it.nk, q_wave + shift + 1) : it.nk);
    f32x16 sc[QB];
#pragma unroll
    for (int i = 0; i < KS; ++i) {
      const op_t k = __builtin_bit_cast(op_t, *reinterpret_cast<const u32x4*>(kb + i * 16));
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) sc[qb] = Pk<T>::mfma(k, q[qb][i], i == 0 ? f32x16{} : sc[qb]);
    }
    if (edge) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const int lim = a.causal ? min(it.nk, q_wave + qb * 32 + l32 + shift + 1) : it.nk;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (base + 16 * (x >> 3) + 8 * hl + (x & 7) >= lim) sc[qb][x] = -INFINITY;
      }
    }
    op_t p[QB][2];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float st;
      auto exps = [&]() __attribute__((always_inline)) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(__builtin_fmaf(sc[qb][8 * ch + 2 * e], a.c, -m[qb]));
            const float p1 = fast_exp2(__builtin_fmaf(sc[qb][8 * ch + 2 * e + 1], a.c, -m[qb]));
            w[e] = Pk<T>::pack(p0, p1);
            part[e] += p0 + p1;
          }
          p[qb][ch] = __builtin_bit_cast(op_t, w);
        }
        st = (part[0] + part[1]) + (part[2] + part[3]);
      };
      if (s != 0) exps();
      if (s == 0 || __any(!(st <= kSumLimit))) {
        asm volatile("" ::: "memory");  // rare: stays a branch
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < 16; ++x) mx = fmaxf(mx, sc[qb][x]);
        mx = halves_max(mx) * a.c;
        const float to = s == 0 ? (mx == -INFINITY ? 0.f : mx) : fmaxf(m[qb], mx);
        const float f = fast_exp2(m[qb] - to);
        m[qb] = to;
        if (s != 0) {
          l[qb] *= f;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[db][qb][x] *= f;
        }
        exps();
      }
      l[qb] += st;
    }
    op_t v[2][DB];
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const e_t* at = vb + ch * 16 * kPitch + db * 32;
        const u32x2 lo = read_tr(at), hi = read_tr(at + 4 * kPitch);
        v[ch][db] = __builtin_bit_cast(op_t, u32x4{lo[0], lo[1], hi[0], hi[1]});
      }
    if (edge && a.causal) {
      // Some query of the block sees some key of it and not others: 0 times an infinity or NaN behind the mask
      // would count in the products, so such keys are added one by one.
      bool odd = false;
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = __builtin_bit_cast(u32x4, v[ch][db])[e];
            odd = odd || (w & Pk<T>::kExp) == Pk<T>::kExp || ((w >> 16) & Pk<T>::kExp) == Pk<T>::kExp;
          }
      if (__any(odd)) {
        const e_t* rows = &sV[buf][(s & 1) * kSub * kPitch];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          const int lim = min(it.nk, q_wave + qb * 32 + l32 + shift + 1);
#pragma unroll 1
          for (int kk = 0; kk < kSub; ++kk) {
            // key 16 ch + 8 half + e: element e of operand ch in the lane of that half
            const u32x4 w0 = __builtin_bit_cast(u32x4, p[qb][0]), w1 = __builtin_bit_cast(u32x4, p[qb][1]);
            const int e = (kk & 7) >> 1;
            uint32_t w = kk & 16 ? (e & 2 ? (e & 1 ? w1[3] : w1[2]) : (e & 1 ? w1[1] : w1[0]))
                                 : (e & 2 ? (e & 1 ? w0[3] : w0[2]) : (e & 1 ? w0[1] : w0[0]));
            w = __shfl(w, l32 + 32 * ((kk >> 3) & 1));
            const float pk = Pk<T>::one((uint16_t)(kk & 1 ? w >> 16 : w & 0xffffu));
            if (base + kk >= lim) continue;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
              for (int x = 0; x < 16; ++x)
                acc[db][qb][x] = __builtin_fmaf(pk, Pk<T>::one(rows[kk * kPitch + 32 * db + 8 * (x >> 2) + 4 * hl + (x & 3)]), acc[db][qb][x]);
          }
        }
        return;
      }
    }
#pragma unroll
    for (int ch = 0; ch < 2; ++ch)
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) acc[db][qb] = Pk<T>::mfma(v[ch][db], p[qb][ch], acc[db][qb]);
  };

  if (n_tiles > 0) {
    fetch(0);
    stage(0);
    __syncthreads();
    for (int t = 0; t < n_tiles; ++t) {
      const int buf = t & 1;
      if (t + 1 < n_tiles) fetch(t + 1);
      if (2 * t < n_sub) step(2 * t, buf);
      if (2 * t + 1 < n_sub) step(2 * t + 1, buf);
      if (t + 1 < n_tiles) {
        stage(buf ^ 1);  // its last readers passed the barrier of the tile before
        __syncthreads();
      }
    }
  }

#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float sum = l[qb] + __shfl_xor(l[qb], 32);
    const float f = sum == 0.f ? 0.f : 1.f / sum;  // a query that sees no key is 0
    const int t = q_wave + qb * 32 + l32;
    if (t >= it.nq) continue;
    char* o = a.o + (int64_t)(it.q0 + t) * a.os[0] + (int64_t)h * a.os[1];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x16& r = acc[db][qb];
        *reinterpret_cast<u32x2*>(o + (32 * db + 8 * i + 4 * hl) * 2) =
            u32x2{Pk<T>::pack(r[4 * i] * f, r[4 * i + 1] * f), Pk<T>::pack(r[4 * i + 2] * f, r[4 * i + 3] * f)};
      }
  }
}

template <typename T, int D, int QB>
void launch_q(const PackedArgs& a, hipStream_t stream) {
  constexpr int kBM = 32 * QB * kWaves;
  const int64_t blocks = a.T / kBM + std::min(a.B, a.T);  // at most: every sequence's last block is part full
  hipLaunchKernelGGL((packed_attn_kernel<T, D, QB>), dim3((unsigned)(blocks * a.H)), dim3(kThreads), 0, stream, a);
}

}  // namespace

hipError_t launch_packed(int dtype, int D, const PackedArgs& a, hipStream_t stream) {
  if (D == 64) {
    if (dtype == 2) launch_q<Bf16, 64, 2>(a, stream);
    else launch_q<F16, 64, 2>(a, stream);
  } else {
    if (dtype == 2) launch_q<Bf16, 128, 1>(a, stream);
    else launch_q<F16, 128, 1>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace wdrz
