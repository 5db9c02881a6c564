// packed.hip — attention of packed sequences of different lengths, with grouped heads: no padding between them.
//
// Sequence i is rows cu_q[i] .. cu_q[i + 1] - 1 of the queries and cu_k[i] .. cu_k[i + 1] - 1 of the keys and values.
// Its query t sees all its keys, or under the causal mask those at t + (keys - queries) and before; a query that
// sees none gives zeros. Query head h reads key/value head h / (H / Hk).
//
// A wavefront takes 32 queries of one head; a workgroup of 4 (64 dims) or 8 (128 dims) holds as many heads of a group as
// divide both, which read the same keys, and blocks of 32 queries beside each other; where blocks are few two wavefronts
// share one, each with half of every tile's keys, and join at the end. Tiles of 64 keys and values go from memory to
// one of 3 or 4 LDS buffers past the registers, the next ones while one is computed; a tile's rows are swizzled so that neither operand's reads meet in a bank. As in the encoder's attention the products are transposed,
// S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 matrix instructions, with the keys' rows permuted so that the scores of
// a lane are already the operand of the second product, and V^T is read from row-major V by transposing LDS reads. Work
// items, the longest first, are found from the sums by every workgroup: the host does not know them.
//
// Softmax: p = 2^(c s - m) in fp32 with a reference m per query, taken from the first 32 keys of which one has weight (a score
// above -inf) and moved only where a lane's 16 probabilities sum to more than 2^15: no maximum is taken otherwise. Sums are of the fp32 probabilities. The products take them in the
// operands' type, one rounding of half a step (2^-8 or 2^-11 of each), as the encoder and long prompts into slots do; the
// attention over pages and short prompts into slots, whose matrix cores idle, take two operands, the rounded value and what is
// left. Results in bf16 are 0.0022 (relative, 2-norm) from 64 bits, those of a plain form in fp32, rounded once, 0.0016. Here
// the second product and the remainders cost, us: 13 tokens 4.63 / 4.76, 1 x 128 over 1500 keys 19.0 / 22.1, the cases below 41 / 53 and
// 700 / 948, 64 prompts with their writes 108 / 118.
//
// Bound: at 128 dims the matrix cores, at 64 the exponentials, the operands' reads from LDS, of which each feeds one matrix
// instruction of a wavefront's 32 queries (the encoder's form, with 64, has half as many), and with few blocks the chain of a step. 2 x 8192 tokens of 32/8 heads of 128, causal: 680 .. 715 us, 1.0 PFLOP/s of the
// 1.39 that a library product of 8192^3 reaches; 16 prompts over 1500 keys of 20 heads of 64: 41 us, 390 TFLOP/s.
// Measured, us, at 64 dims (long batch with its write / cross) and 128:
//   4 wavefronts, 3 buffers, 3 a SIMD     110 / 41.6    the form taken: other wavefronts of the SIMD fill the softmax's time
//     4 buffers, next scores ahead, 2     127 / 47.8      2 buffers, 4 a SIMD 112 / 41.9; 3 buffers, ahead, 3 a SIMD 114 / 42.2
//   8 wavefronts, 4 buffers, ahead, 2     154 / 51.7      685 at 128, the form taken (registers allow 2 a SIMD)
//     3 buffers, not ahead                691 at 128      4 wavefronts 1169
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kTile = 64;           // keys a stage
constexpr int kSub = 32;            // keys a step
// A query's reference lies 2^8 below its largest probability, so that fp16 operands hold those down to 2^-22 of it with
// all digits, and is moved where a lane's 16 sum to more than 2^15: none leaves fp16.
constexpr float kBelow = 8.f, kSumLimit = 32768.f;

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// A buffer resource over [base, base + bytes): loads past the end return zero.
__device__ __forceinline__ i32x4 rsrc(const void* base, uint32_t bytes) {
  const uint64_t p = (uint64_t)(uintptr_t)base;
  i32x4 r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)p);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32) & 0xffff);  // stride 0
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;  // 32-bit data format
  return r;
}

template <typename T> struct Pk;
template <> struct Pk<Bf16> {
  typedef bf16x8 op_t;
  static __device__ __forceinline__ f32x16 mfma(op_t a, op_t b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static constexpr uint32_t kExp = 0x7f80u, kOne = 0x3f80u;
};
template <> struct Pk<F16> {
  typedef f16x8 op_t;
  static __device__ __forceinline__ f32x16 mfma(op_t a, op_t b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static constexpr uint32_t kExp = 0x7c00u, kOne = 0x3c00u;
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

// Work items: the query blocks of the sequences, counted from a sequence's end (under the mask the last needs the most
// keys), sequences from the last. Every lane of a wavefront calls these.
struct Item {
  int q0, nq, k0, nk, block;
};
// 64 sequences from B - 1 - i0 down, one a lane: its rows and the items up to it.
struct Chunk {
  int c0, c1, sum, total;
};
__device__ __forceinline__ Chunk scan_items(const PackedArgs& a, int rows, int i0) {
  const int lane = threadIdx.x & 63, i = a.B - 1 - i0 - lane;
  Chunk c = {0, 0, 0, 0};
  if (i >= 0) {
    c.c0 = min(max(a.cu_q[i], 0), a.T);  // sums that are not ascending or in range stay in bounds
    c.c1 = min(max(a.cu_q[i + 1], c.c0), a.T);
  }
  c.sum = (c.c1 - c.c0 + rows - 1) / rows;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(c.sum, o);
    if (lane >= o) c.sum += u;
  }
  c.total = __builtin_amdgcn_readlane(c.sum, 63);
  return c;
}
// The item `idx` of the chunk's `total`.
__device__ __forceinline__ Item pick_item(const PackedArgs& a, const Chunk& c, int i0, int idx) {
  const int src = __ffsll((unsigned long long)__ballot(idx < c.sum)) - 1, s = a.B - 1 - i0 - src;
  Item it;
  it.q0 = __builtin_amdgcn_readlane(c.c0, src);
  it.nq = __builtin_amdgcn_readlane(c.c1, src) - it.q0;
  it.block = __builtin_amdgcn_readlane(c.sum, src) - 1 - idx;
  it.k0 = min(max(a.cu_k[s], 0), a.Tk);
  it.nk = min(max(a.cu_k[s + 1], it.k0), a.Tk) - it.k0;
  return it;
}
// This workgroup's item, and its group of heads in `sub`; false where it has none. Items of a group of heads are next to
// each other, on one XCD: those of a sequence read the same keys. The host launches as many workgroups as there may be
// items; where one chunk holds all sequences their number is known, the first workgroups take them and the CUs get
// equally many. 20 heads of 64, us, with the empty ones in between / so: 64 prompts of 448 tokens 103 / 100, of 30 12.4 / 11.0;
// 64 tokens over 1500 keys each, 8 prompts 28.4 / 21.3, 16 42.7 / 34.8.
__device__ __forceinline__ bool find_item(const PackedArgs& a, int rows, int& sub, Item& it) {
  const int n_wg = (int)gridDim.x, groups = a.H / a.nh;
  Chunk c = scan_items(a, rows, 0);
  if (a.B <= 64) {
    const int n = (int)min((int64_t)c.total * groups, (int64_t)n_wg);
    if ((int)blockIdx.x >= n) return false;
    const int unit = remap_xcd((int)blockIdx.x, n);
    sub = unit / c.total;
    it = pick_item(a, c, 0, unit % c.total);
    return sub < groups;
  }
  const int unit = remap_xcd((int)blockIdx.x, n_wg), n_idx = n_wg / groups;
  sub = unit / n_idx;
  int idx = unit % n_idx;
  for (int i0 = 0;;) {
    if (idx < c.total) {
      it = pick_item(a, c, i0, idx);
      return true;
    }
    idx -= c.total;
    if ((i0 += 64) >= a.B) return false;
    c = scan_items(a, rows, i0);
  }
}

// 16 bytes a lane from memory to LDS, lane l to byte `to` + 16 l, without passing through registers; zeros where the
// offset lies behind the resource. The compiler does not know of it: waits are written out below.
__device__ __forceinline__ void load_lds(i32x4 from, uint32_t offset, uint32_t to) {
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(from), "s"(to) : "m0", "memory");
#else
  (void)from, (void)offset, (void)to;
#endif
}
template <int N> __device__ __forceinline__ void landed_barrier() {  // all but the last N loads, of every wavefront
#if __HIP_DEVICE_COMPILE__
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
#endif
}

// AHEAD: the next step's scores run under this step's softmax; else the other wavefronts of the SIMD (SIMD_WAVES) fill it.
// HALVES 2: two wavefronts share a query block, each takes one half of every tile's keys.
template <typename T, int D, int NW, int NBUF, bool AHEAD, int SIMD_WAVES, int HALVES>
__global__ __launch_bounds__(64 * NW, SIMD_WAVES) void packed_attn_kernel(PackedArgs a) {
  typedef typename Pk<T>::op_t op_t;
  typedef uint16_t e_t;
  constexpr int KS = D / 16, DB = D / 32, kRow = D * 2, kPiece = kRow / 16, kHalf = kTile * kRow, kBuf = 2 * kHalf;
  constexpr int kLoads = kHalf / 1024 / NW;  // a wavefront's loads of a tile's keys (and of its values)
  __shared__ __attribute__((aligned(1024))) char smem[NBUF * kBuf];  // tiles: keys, then values

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hl = lane >> 5, l32 = lane & 31;
  const int nqb = NW / HALVES / a.nh;  // query blocks a head
  int sub;
  Item it;
  if (!find_item(a, 32 * nqb, sub, it)) return;
  const int hk = sub / (a.H / a.Hk / a.nh);
  // wavefronts w and w + 4 share a SIMD: under the mask the later blocks of one half meet the earlier ones of the other
  const int slot = wave % (NW / HALVES), half = wave / (NW / HALVES);
  const int qbi = slot < 4 || NW == 4 ? slot / a.nh : nqb - 1 - (slot - 4) / a.nh;
  const int h = sub * a.nh + slot % a.nh;
  const int q_wg = it.block * 32 * nqb, q_wave = q_wg + qbi * 32;
  const int shift = a.causal ? it.nk - it.nq : 0;  // query t sees the keys up to t + shift
  const int k_lim = a.causal ? max(0, min(it.nk, min(q_wg + 32 * nqb, it.nq) + shift)) : it.nk;
  const int n_tiles = (k_lim + kTile - 1) / kTile;
  const int w_lim = q_wave >= it.nq ? 0 : a.causal ? max(0, min(k_lim, q_wave + 32 + shift)) : it.nk;  // keys of this wavefront
  const int n_sub = (w_lim + kSub - 1) / kSub;
  const int lim = a.causal ? min(it.nk, q_wave + l32 + shift + 1) : it.nk;        // keys that this lane's query sees
  const int lim_lo = a.causal ? min(it.nk, q_wave + shift + 1) : it.nk;           // keys that every query sees

  const char* Q = a.q + (int64_t)it.q0 * a.qs[0] + (int64_t)h * a.qs[1];
  const char* K = a.k + (int64_t)it.k0 * a.ks[0] + (int64_t)hk * a.ks[1];
  const char* V = a.v + (int64_t)it.k0 * a.vs[0] + (int64_t)hk * a.vs[1];

  // Tiles lie in LDS as rows of kPiece 16-byte pieces, piece p of row r at place p ^ swizzle(r): the 16 rows of a K
  // operand's piece and the 4 rows x 64 bytes of a V^T operand's lie in different banks.
  auto swizzle = [](int r) { return D == 64 ? ((r >> 1 & 1) << 2) | (r >> 2 & 3) : ((r & 3) << 2) | (r >> 2 & 3); };
  uint32_t k_from[kLoads], v_from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = (i * NW + wave) * (1024 / kRow) + lane / kPiece, p = (lane % kPiece) ^ swizzle(r);
    k_from[i] = (uint32_t)(r * (int)a.ks[0] + p * 16);  // 64 rows fit 31 bits (checked by the caller)
    v_from[i] = (uint32_t)(r * (int)a.vs[0] + p * 16);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)smem;
  auto issue = [&](int t) __attribute__((always_inline)) {
    const int rows = min(it.nk - t * kTile, kTile);  // rows behind the sequence come as zeros: another's, which must not count
    const i32x4 kr = rsrc(K + (int64_t)t * kTile * a.ks[0], rows > 0 ? (uint32_t)((rows - 1) * (int)a.ks[0] + kRow) : 0u);
    const i32x4 vr = rsrc(V + (int64_t)t * kTile * a.vs[0], rows > 0 ? (uint32_t)((rows - 1) * (int)a.vs[0] + kRow) : 0u);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (uint32_t)(t % NBUF) * kBuf + wave * 1024);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_lds(kr, k_from[i], to + i * NW * 1024);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_lds(vr, v_from[i], to + kHalf + i * NW * 1024);
  };

  f32x16 acc[DB];  // O^T: query l32, dim 32 db + 8 (x / 4) + 4 hl + x % 4
  float m = -INFINITY, l = 0.f;  // reference (-inf: no key had weight yet), this lane's sum
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int x = 0; x < 16; ++x) acc[db][x] = 0.f;

  if (n_tiles > 0) {
    issue(0);
    u32x4 q[KS];
    {
      const char* row = Q + (int64_t)min(q_wave + l32, it.nq - 1) * a.qs[0] + hl * 16;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[s] = load16(row + s * 32);
#pragma unroll
      for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(q[s]));  // here, not behind the next tiles
    }
#pragma unroll
    for (int t = 1; t < NBUF - 1; ++t) issue(t);
    if (AHEAD) landed_barrier<2 * kLoads * (NBUF - 2)>();

    // K operand: key row 8 i + 4 j + e of a step stands at row 16 (i / 2) + 8 j + 4 (i % 2) + e, so that score x of a
    // lane is key 16 (x / 8) + 8 hl + x % 8. Piece 2 s + hl of it: the place of piece hl, ^ 2 s.
    const int k_row = 16 * (l32 >> 4) + 8 * (l32 >> 2 & 1) + 4 * (l32 >> 3 & 1) + (l32 & 3);
    const uint32_t k_at = k_row * kRow + ((hl ^ swizzle(k_row)) << 4);
    // V^T operand: rows 8 hl + j / 4 (j = lane % 16) and those 4 further, dims 16 (lane / 16 % 2) + 4 (j % 4) of a block
    const int j16 = lane & 15, v_row = 8 * hl + (j16 >> 2);
    const uint32_t v_at = v_row * kRow + (((2 * (lane >> 4 & 1) + (j16 >> 1 & 1)) ^ swizzle(v_row)) << 4) + (j16 & 1) * 8;
    op_t k[KS], v[2][DB];
    auto read_k = [&](int s) __attribute__((always_inline)) {
      const uint32_t at = k_at + ((s >> 1) % NBUF) * kBuf + (s & 1) * kSub * kRow;
#pragma unroll
      for (int i = 0; i < KS; ++i) k[i] = __builtin_bit_cast(op_t, *reinterpret_cast<const u32x4*>(smem + (at ^ (i << 5))));
    };
    auto read_v = [&](int s) __attribute__((always_inline)) {
      const uint32_t at = v_at + ((s >> 1) % NBUF) * kBuf + kHalf + (s & 1) * kSub * kRow;
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const u32x2 lo = read_tr(reinterpret_cast<const e_t*>(smem + (at ^ (db << 6)) + ch * 16 * kRow));
          const u32x2 hi = read_tr(reinterpret_cast<const e_t*>(smem + (at ^ (db << 6) ^ 16) + (ch * 16 + 4) * kRow));
          v[ch][db] = __builtin_bit_cast(op_t, u32x4{lo[0], lo[1], hi[0], hi[1]});
        }
    };
    auto scores = [&](f32x16& sc) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < KS; ++i) sc = Pk<T>::mfma(k[i], __builtin_bit_cast(op_t, q[i]), i == 0 ? f32x16{} : sc);
    };
    // One step: the next step's scores and this one's V^T operands are under way while the softmax runs.
    auto step = [&](int s, f32x16& sc, f32x16& next) __attribute__((always_inline)) {
      const int base = s * kSub;
      const bool edge = base + kSub > lim_lo;
      if (AHEAD) {
        read_v(s);
        if (s + 1 < n_sub) scores(next);
      } else {
        read_k(s);
        scores(sc);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (edge) {
        const int sees = lim - base - 8 * hl;
#pragma unroll
        for (int x = 0; x < 16; ++x)
          if (16 * (x >> 3) + (x & 7) >= sees) sc[x] = -INFINITY;
      }
      op_t p[2];
      float st;
      auto exps = [&](float ref) __attribute__((always_inline)) {
        float part[4];
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p0 = fast_exp2(__builtin_fmaf(sc[8 * ch + 2 * e], a.c, -ref));
            const float p1 = fast_exp2(__builtin_fmaf(sc[8 * ch + 2 * e + 1], a.c, -ref));
            w[e] = Pk<T>::pack(p0, p1);
            part[e] = ch == 0 ? p0 + p1 : part[e] + p0 + p1;
          }
          p[ch] = __builtin_bit_cast(op_t, w);
        }
        st = (part[0] + part[1]) + (part[2] + part[3]);
      };
      const bool first = s == half;
      if (!first) exps(m);
      if (first || __any(!(st <= kSumLimit))) {  // without a reference st is infinite or NaN
        asm volatile("" ::: "memory");  // rare: stays a branch
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < 16; ++x) mx = fmaxf(mx, sc[x]);
        mx = halves_max(mx) * a.c;
        const float to = fmaxf(m, mx - kBelow);
        if (!first) {
          const float f = to == m ? 1.f : fast_exp2(m - to);
          l *= f;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[db][x] *= f;
        }
        m = to;
        exps(m == -INFINITY ? 0.f : m);
      }
      l += st;
      if (!AHEAD) read_v(s);
      __builtin_amdgcn_sched_barrier(0);
      // Where some query sees some key of the step and not others, 0 times an infinity or NaN behind the mask would
      // count in the products: such values are taken out of V, and given to the queries that see them.
      if (edge) {
        f32x16 zero = {};  // 0 times each value: 0, or NaN where there is such a one
#pragma unroll
        for (int ch = 0; ch < 2; ++ch)
#pragma unroll
          for (int db = 0; db < DB; ++db) zero = Pk<T>::mfma(v[ch][db], op_t{}, zero);
        float any = 0.f;
#pragma unroll
        for (int x = 0; x < 16; ++x) any += zero[x];
        const bool odd = any != any;
        if (__any(odd)) {
          op_t sees[2];
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = base + 16 * ch + 8 * hl + 2 * e;
              w[e] = Pk<T>::pack(key < lim ? 1.f : 0.f, key + 1 < lim ? 1.f : 0.f);
            }
            sees[ch] = __builtin_bit_cast(op_t, w);
          }
          // the values of one kind (inf, -inf, NaN) as ones
          auto ones = [&](op_t x, int kind) __attribute__((always_inline)) {
            u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t r = 0;
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const uint32_t u = w[e] >> (16 * half) & 0xffffu;
                const bool is = kind == 2 ? (u & 0x7fffu) > Pk<T>::kExp : u == (Pk<T>::kExp | (kind ? 0x8000u : 0u));
                r |= is ? Pk<T>::kOne << (16 * half) : 0u;
              }
              w[e] = r;
            }
            return __builtin_bit_cast(op_t, w);
          };
#pragma unroll
          for (int db = 0; db < DB; ++db) {
#pragma unroll 1
            for (int kind = 0; kind < 3; ++kind) {
              f32x16 n = Pk<T>::mfma(ones(v[0][db], kind), sees[0], f32x16{});
              n = Pk<T>::mfma(ones(v[1][db], kind), sees[1], n);
              const float value = kind == 2 ? __builtin_nanf("") : kind ? -INFINITY : INFINITY;
#pragma unroll
              for (int x = 0; x < 16; ++x) acc[db][x] += n[x] > 0.f ? value : 0.f;
            }
#pragma unroll
            for (int ch = 0; ch < 2; ++ch) {
              u32x4 w = __builtin_bit_cast(u32x4, v[ch][db]);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if ((w[e] & Pk<T>::kExp) == Pk<T>::kExp) w[e] &= 0xffff0000u;
                if ((w[e] >> 16 & Pk<T>::kExp) == Pk<T>::kExp) w[e] &= 0xffffu;
              }
              v[ch][db] = __builtin_bit_cast(op_t, w);
            }
          }
        }
      }
      if (AHEAD) read_k(s + 2);
#pragma unroll
      for (int ch = 0; ch < 2; ++ch)
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = Pk<T>::mfma(v[ch][db], p[ch], acc[db]);
      __builtin_amdgcn_sched_barrier(0);
    };

    f32x16 s0, s1;
    if (AHEAD) {
      read_k(0);
      scores(s0);
      read_k(1);
    }
    for (int t = 0; t < n_tiles; ++t) {
      // the last tile that this one's steps read (AHEAD: the next one's keys) is there; nobody reads tile t - 1 any more
      landed_barrier<2 * kLoads * (NBUF - (AHEAD ? 3 : 2))>();
      issue(t + NBUF - 1);
      if (HALVES == 2) {
        if (2 * t + half < n_sub) step(2 * t + half, s0, s1);
        continue;
      }
      if (2 * t < n_sub) step(2 * t, s0, s1);
      if (2 * t + 1 < n_sub) {
        if (AHEAD) step(2 * t + 1, s1, s0);
        else step(2 * t + 1, s0, s1);
      }
    }
  }

  // O^T through LDS, so that memory sees whole rows: the wavefront's 32 rows in its own part
  landed_barrier<0>();
  float sum = l + __shfl_xor(l, 32);
  constexpr int kPart = HALVES == 1 ? 32 * kRow : (DB * 16 + 2) * 64 * 4;  // a query block's part of the LDS
  if (HALVES == 2) {  // the second half's sums to the first's wavefront
    float* part = reinterpret_cast<float*>(smem + slot * kPart) + lane;
    if (half) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int x = 0; x < 16; ++x) part[(db * 16 + x) * 64] = acc[db][x];
      part[DB * 16 * 64] = m;
      part[(DB * 16 + 1) * 64] = sum;
    }
    __syncthreads();
    if (half) return;
    const float m1 = part[DB * 16 * 64], sum1 = part[(DB * 16 + 1) * 64];
    const float M = sum == 0.f ? m1 : sum1 == 0.f ? m : fmaxf(m, m1);  // a half that sees nothing has no reference
    const float f0 = sum == 0.f ? 0.f : fast_exp2(m - M), f1 = sum1 == 0.f ? 0.f : fast_exp2(m1 - M);
    sum = sum * f0 + sum1 * f1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int x = 0; x < 16; ++x) acc[db][x] = acc[db][x] * f0 + part[(db * 16 + x) * 64] * f1;
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum;  // a query that sees no key is 0
  char* mine = smem + slot * kPart;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x16& r = acc[db];
      const int at = l32 * kRow + (((4 * db + i) ^ swizzle(l32)) << 4) + hl * 8;
      *reinterpret_cast<u32x2*>(mine + at) = u32x2{Pk<T>::pack(r[4 * i] * f, r[4 * i + 1] * f), Pk<T>::pack(r[4 * i + 2] * f, r[4 * i + 3] * f)};
    }
  __builtin_amdgcn_wave_barrier();
  char* o = a.o + (int64_t)(it.q0 + q_wave) * a.os[0] + (int64_t)h * a.os[1];
#pragma unroll
  for (int i = 0; i < 32 * kPiece / 64; ++i) {
    const int r = i * (64 / kPiece) + lane / kPiece, p = lane % kPiece;
    const u32x4 w = *reinterpret_cast<const u32x4*>(mine + r * kRow + ((p ^ swizzle(r)) << 4));
    if (q_wave + r < it.nq) store16(o + (int64_t)r * a.os[0] + p * 16, w);
  }
}

// A query block's chain of steps takes 530 ns for 32 keys however few there are: with up to 1.5 blocks a SIMD, and keys enough
// to make up for the join, two wavefronts take half of it each. 20 heads of 64 over 1500 keys, us, one / two wavefronts, by
// prompts of 128 tokens: 1 26.7 / 18.4, 8 29.4 / 25.7, 16 37.1 / 32.5, 24 41.3 / 44.9, 64 118.6 / 135.7; 8 over 150 keys 7.8 / 8.2.
constexpr int64_t kFewBlocks = 1536;
constexpr int kWaves64 = 4, kWaves128 = 8;  // wavefronts a workgroup, by the head's dims

// How a call is cut: wavefronts to a query block, heads of a group in a workgroup (as many as divide the group and the
// workgroup's query blocks), workgroups.
struct Cut {
  int halves, nh, rows;
  int64_t blocks;
};
Cut cut_of(int64_t T, int64_t Tk, int64_t B, int64_t H, int64_t Hk, int64_t D) {
  Cut c;
  c.halves = D == 64 && T / 32 * H <= kFewBlocks && Tk >= 256 * B ? 2 : 1;
  const int slots = (D == 64 ? kWaves64 : kWaves128) / c.halves;
  c.nh = 1;
  while (c.nh < slots && H / Hk % (2 * c.nh) == 0) c.nh *= 2;
  c.rows = 32 * slots / c.nh;
  c.blocks = (T / c.rows + std::min(B, T)) * (H / c.nh);  // at most: every sequence's last block is part full
  return c;
}

template <typename T, int D, int NW, int NBUF, bool AHEAD, int SIMD_WAVES, int HALVES>
void launch_q(PackedArgs a, const Cut& c, hipStream_t stream) {
  a.nh = c.nh;
  hipLaunchKernelGGL((packed_attn_kernel<T, D, NW, NBUF, AHEAD, SIMD_WAVES, HALVES>), dim3((unsigned)c.blocks), dim3(64 * NW), 0, stream, a);
}
template <typename T> void launch_t(int D, const PackedArgs& a, hipStream_t stream) {
  const Cut c = cut_of(a.T, a.Tk, a.B, a.H, a.Hk, D);
  if (D == 128) launch_q<T, 128, kWaves128, 4, true, 2, 1>(a, c, stream);
  else if (c.halves == 2) launch_q<T, 64, kWaves64, 3, false, 3, 2>(a, c, stream);
  else launch_q<T, 64, kWaves64, 3, false, 3, 1>(a, c, stream);
}

}  // namespace

int64_t packed_blocks(int64_t T, int64_t Tk, int64_t B, int64_t H, int64_t Hk, int64_t D) { return cut_of(T, Tk, B, H, Hk, D).blocks; }

hipError_t launch_packed(int dtype, int D, const PackedArgs& a, hipStream_t stream) {
  if (dtype == 2) launch_t<Bf16>(D, a, stream);
  else launch_t<F16>(D, a, stream);
  return hipGetLastError();
}

}  // namespace wdrz
