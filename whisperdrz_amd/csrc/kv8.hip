// kv8.hip — the slot cache held in 8 bits: its writes and the cached attention over it (gfx950).
//
// Storage of one cache (wdrz_kv8 in include/wdrz_attn.h). Positions are held in blocks of 32. A complete
// block of one (slot, head) is 32 x 64 codes (e4m3) with one scale for its keys and one for its values:
//   2^e, e the least whole number of [-100, 100] under which the block's largest finite value is at
//   most 448; code = round_to_nearest_even(clamp(x 2^-e, -448, 448)), what is not finite becomes NaN.
// e4m3 is a floating type, so a power of two loses nothing against a finer scale, x 2^-e is exact and the
// code is x rounded once; a code times its scale is exact in bf16 as in fp32.
// A cache that is appended to also keeps its newest positions as they came, in a ring of 64 rows a
// (slot, head): position p in row p % 64, of the last complete block and the one behind it. The block
// that is not complete is read from there. So a position is rounded once, when its block completes, a
// block never changes afterwards, and how the tokens were cut into calls changes no bit of the cache.
//
// Attention. A call that appends reads positions below c0 = 32 floor(len / 32) as codes, [c0, len) from
// the ring and its own new rows as they are. What it writes, ring rows of [len, len + sq) and the codes
// of the block that they complete, nobody reads in the same launch: with sq <= 32 the positions
// [c0, len + sq) are at most 63, so no new row shares a ring row with an old one that is still read,
// and the append rides in the attention launch. Longer prompts append in a launch of their own behind it.
//
// One wavefront takes a block of 32 keys and up to 16 queries a step, as kv_mq_kernel does:
//   S^T (32 keys x 16 queries) = K Q^T with 4 v_mfma_f32_16x16x32, O^T (64 dims x 16 queries) += V^T P^T
// with 8 more, P in two 16-bit parts. Codes become bf16 (fp16 queries: fp16 for K, whose products are
// then exact too) two an instruction; the keys' scale multiplies the scores in fp32, the values' scale
// is the conversion's own, exact in bf16. A lane's 16-byte load is 16 dimensions of one key: the matrix
// product sums over the dimensions in that order, for K and Q alike. V goes through an LDS tile and
// comes back transposed.
#include <algorithm>

#include "kv_merge.h"
#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kBlk = 32;                  // positions a scale covers
constexpr int kRing = 64;                 // ring rows
constexpr int kRowBytes16 = kHeadDim * 2;
constexpr int kVPitch = kHeadDim + 8;     // V tile row pitch (16-bit elements)
constexpr float kTau = 8.0f;              // lazy-rescale threshold (log2 units)

template <typename T> struct Ops;
template <> struct Ops<Bf16> {
  typedef bf16x8 op_t;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(op_t, a), __builtin_bit_cast(op_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
  static constexpr uint32_t kExp = 0x7f80u;  // exponent bits: all set in what is not finite
};
template <> struct Ops<F16> {
  typedef f16x8 op_t;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(op_t, a), __builtin_bit_cast(op_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_f16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return f16_lo(w); }
  static __device__ __forceinline__ float hi(uint32_t w) { return f16_hi(w); }
  static constexpr uint32_t kExp = 0x7c00u;
};

// Eight e4m3 codes as eight 16-bit values of type T, times a power of two (exact in bf16; fp16 holds
// the codes alone).
template <typename T> __device__ __forceinline__ u32x4 widen8(uint32_t a, uint32_t b, float scale);
template <> __device__ __forceinline__ u32x4 widen8<Bf16>(uint32_t a, uint32_t b, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, scale, true))};
}
template <> __device__ __forceinline__ u32x4 widen8<F16>(uint32_t a, uint32_t b, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, scale, true))};
}

// ---- rows of one call that name the same slot -------------------------------------------------
// They have to agree on its length; then the last of them gives the new rows for all (a decode graph's
// padding repeats a slot with that slot's own length). Rows that do not agree are invalid: reading one
// row's positions while another rewrites them has no defined result.
struct SlotRows {
  int src;        // the last row naming this slot
  bool conflict;  // a row names it with another start
};
// Every lane active; the same result in every lane and wavefront.
template <typename Id, typename Start>
__device__ __forceinline__ SlotRows slot_rows(int B, int64_t slot, int start, Id id, Start start_of) {
  SlotRows r{-1, false};
  const int lane = threadIdx.x & 63;
  bool differ = false;
  for (int base = 0; base < B; base += 64) {
    const int i = min(base + lane, B - 1);
    const bool same = id(i) == slot && base + lane < B;
    differ = differ || (same && start_of(i) != start);
    const uint64_t m = __ballot(same);
    if (m) r.src = base + 63 - __clzll((long long)m);
  }
  r.conflict = __ballot(differ) != 0ull;
  return r;
}

// ---- one block into codes -----------------------------------------------------------------------
// Threads 0..255 hold the block, thread i the 8 dimensions 8 (i % 8).. of row i / 8, of K and of V;
// rows that are not there are zeros. Every thread of the workgroup calls it.
template <typename T>
__device__ __forceinline__ void quantize_block(u32x4 kw, u32x4 vw, uint8_t* kc, uint8_t* vc, float* ks, float* vs,
                                               uint32_t (&red)[2][4]) {
  const int tid = threadIdx.x;
  Slice<T> x[2];
  x[0].from_raw(kw);
  x[1].from_raw(vw);
  uint32_t top[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    top[n] = 0;  // magnitudes compare as their bits do
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t m = __float_as_uint(x[n].v[i]) & 0x7fffffffu;
      top[n] = max(top[n], m < 0x7f800000u ? m : 0u);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top[n] = max(top[n], (uint32_t)__shfl_xor((int)top[n], off));
    if (tid < 256 && (tid & 63) == 0) red[n][tid >> 6] = top[n];
  }
  __syncthreads();
  if (tid < 256) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const uint32_t t = max(max(red[n][0], red[n][1]), max(red[n][2], red[n][3]));
      // t = m 2^E with m in [1, 2), 448 = 1.75 * 2^8
      int e = (int)(t >> 23) - 127 - 8 + ((t & 0x7fffffu) > 0x600000u);
      e = min(max(e, -100), 100);
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
      uint32_t w[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[n].v[4 * q + i] * inv, -448.f, 448.f);
        uint32_t c = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], c, true);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if ((__float_as_uint(x[n].v[4 * q + i]) & 0x7fffffffu) >= 0x7f800000u) c |= 0x7fu << (8 * i);
        w[q] = c;
      }
      *reinterpret_cast<uint2*>((n ? vc : kc) + (tid >> 3) * kHeadDim + (tid & 7) * 8) = make_uint2(w[0], w[1]);
      if (tid == 0) *(n ? vs : ks) = __uint_as_float((uint32_t)(e + 127) << 23);
    }
  }
}

// Where the buffers of (slot, head) start.
__device__ __forceinline__ int64_t slot_head(const Kv8Cache& c, int64_t slot, int h) { return slot * c.H + h; }

// ---- writes: one workgroup a block of 32 positions of (row, head) ------------------------------
// fill: every block is closed, the last one with zeros behind its rows. Otherwise (append) complete
// blocks become codes and the rows of the last two blocks go to the ring. Ring rows of the first block's
// old positions are read here too, so this block's workgroup also writes the later rows that take
// their place (those of the later block of the same parity), after it has read them.
template <typename T, typename Id>
__global__ __launch_bounds__(256) void kv8_write_kernel(Kv8Cache c, Kv8WriteArgs a, const Id* slots) {
  __shared__ uint32_t red[2][4];
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t slot = slots ? (int64_t)slots[b] : b;
  const int start = a.starts ? a.starts[b] : a.start;
  if (slot < 0 || slot >= c.n_slots || start < 0 || start > c.Lk - a.T) return;
  if (slots) {
    const SlotRows r = slot_rows(a.B, slot, start, [&](int i) { return (int64_t)slots[i]; },
                                 [&](int i) { return a.starts ? a.starts[i] : start; });
    if (r.conflict || r.src != b) return;
  }
  const int end = start + a.T, first = start / kBlk, last = (end - 1) / kBlk;
  const int blk = first + (int)blockIdx.x;
  if (blk > last) return;
  const int tid = threadIdx.x, row = tid >> 3, ch = tid & 7;
  const int64_t sh = slot_head(c, slot, h);
  char* rings[2] = {c.kr + sh * (kRing * kRowBytes16) + ch * 16, c.vr + sh * (kRing * kRowBytes16) + ch * 16};
  const char* src[2] = {a.k + b * a.ks[0] + h * a.ks[2] + ch * 16, a.v + b * a.vs[0] + h * a.vs[2] + ch * 16};
  const int64_t step[2] = {a.ks[1], a.vs[1]};
  const int p = blk * kBlk + row;
  u32x4 w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (p < end) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
      w[n] = p >= start ? load16_stream(src[n] + (int64_t)(p - start) * step[n])
             : c.kr     ? load16(rings[n] + (p % kRing) * kRowBytes16)
                        : w[n];
  }
  const bool closed = !c.kr || (blk + 1) * kBlk <= end;
  if (closed) {
    const int64_t code = (sh * c.n_blk + blk) * (kBlk * kHeadDim);
    quantize_block<T>(w[0], w[1], c.kc + code, c.vc + code, c.ks + sh * c.n_blk + blk, c.vs + sh * c.n_blk + blk, red);
  }
  if (!c.kr) return;
  const int keep = end / kBlk - 1;  // blocks from here on stand in the ring
  if (blk >= keep && p >= start && p < end && (blk == first || (blk - first) % 2 != 0)) {
#pragma unroll
    for (int n = 0; n < 2; ++n) store16(rings[n] + (p % kRing) * kRowBytes16, w[n]);
  }
  if (blk == first) {
    __syncthreads();  // every old row has been read
    for (int j = first + 2; j <= last; j += 2) {
      const int q = j * kBlk + row;
      if (j < keep || q >= end) continue;
#pragma unroll
      for (int n = 0; n < 2; ++n)
        store16(rings[n] + (q % kRing) * kRowBytes16, load16(src[n] + (int64_t)(q - start) * step[n]));
    }
  }
}

// ---- attention ----------------------------------------------------------------------------------

// Transposing LDS read (ds_read_b64_tr_b16): within each 16-lane group, lane i receives element
// i%4 of the 8-byte chunks read by lanes 4c + i/4 (c = 0..3).
__device__ __forceinline__ u32x2 read_tr16(const uint16_t* p) {
#if __HIP_DEVICE_COMPILE__
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uint32_t)(uintptr_t)p));
#else
  (void)p;
  return u32x2{0, 0};
#endif
}

// max of x over lanes l, l^16, l^32, l^48, in every lane
__device__ __forceinline__ float group4_max(float x) {
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
}

// O^T += V^T P^T over 32 keys, the probabilities as two operands of type E (the rounded value and what
// the rounding left, so that they count with 16 bits or more).
template <typename E>
__device__ __forceinline__ void pv_step(const uint16_t* vt_lane, const float (&p)[8], f32x4 (&o)[4]) {
  u32x4 ph, pl;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ph[j] = Ops<E>::pack(p[2 * j], p[2 * j + 1]);
    pl[j] = Ops<E>::pack(p[2 * j] - Ops<E>::lo(ph[j]), p[2 * j + 1] - Ops<E>::hi(ph[j]));
  }
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    const u32x2 lo = read_tr16(vt_lane + 16 * db);
    const u32x2 hi = read_tr16(vt_lane + 16 * kVPitch + 16 * db);
    const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
    o[db] = Ops<E>::mfma(v, pl, o[db]);
    o[db] = Ops<E>::mfma(v, ph, o[db]);
  }
}

// SQ: query rows a workgroup (1, 8 or 16). HAS_NEW: the call appends.
template <typename T, int SQ, bool HAS_NEW, int kWaves>
__global__ __launch_bounds__(kWaves * 64, 4) void kv8_attn_kernel(Kv8Cache c, Kv8Args a) {
  __shared__ float sm_acc[kWaves][SQ][kHeadDim];
  __shared__ float sm_m[kWaves][SQ];
  __shared__ float sm_l[kWaves][SQ];
  __shared__ __attribute__((aligned(16))) uint16_t sm_v[kWaves][kBlk * kVPitch];
  __shared__ uint32_t sm_red[2][4];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int qi = lane & 15, gq = lane >> 4;  // query slot (and key row) of this lane, 16-lane group

  const int h = (int)(blockIdx.x % (unsigned)c.H);  // heads fastest: neighbours in the cache run together
  const int bq = (int)(blockIdx.x / (unsigned)c.H);
  const int b = bq / a.n_qblocks;
  const int t0 = (bq % a.n_qblocks) * SQ;
  const int split = blockIdx.z;
  const int nq = min(SQ, a.sq - t0);

  const int slot = a.bidx ? a.bidx[b] : b;
  const int len = a.seqlens ? a.seqlens[b] : c.Lk;
  SlotRows rows{b, false};
  if (HAS_NEW && a.bidx)
    rows = slot_rows(a.B, slot, len, [&](int i) { return a.bidx[i]; }, [&](int i) { return a.seqlens[i]; });
  const bool bad = slot < 0 || slot >= c.n_slots || len < 0 || len > c.Lk - (HAS_NEW ? a.sq : 0) || rows.conflict;

  const int key_lim = HAS_NEW ? len + t0 + nq : len;  // keys this query block needs: [0, key_lim)
  const int n_split_b = bad ? 1 : max(1, (key_lim + a.split_len - 1) / a.split_len);
  if (split >= n_split_b) return;
  if (!HAS_NEW && key_lim == 0 && !bad) {  // a row without keys
    for (int i = tid; i < nq * (kHeadDim / 2); i += kWaves * 64)
      *reinterpret_cast<uint32_t*>(a.o + b * a.os[0] + (t0 + i / 32) * a.os[1] + h * a.os[2] + (i % 32) * 4) = 0;
    return;
  }
  const int k_begin = split * a.split_len;  // a multiple of 32
  const int k_end = bad ? k_begin : min(key_lim, k_begin + a.split_len);
  const int k_last = k_end - 1;
  int lim = k_last;  // last key this lane's query may see (slots past the block's rows see none)
  if (HAS_NEW) lim = min(lim, len + t0 + qi);
  if (qi >= nq) lim = -1;

  // Q^T operand halves: query t0 + qi, dims 16 gq + 8 dh .. + 7
  u32x4 qop[2];
  {
    const char* qrow = a.q + b * a.qs[0] + (t0 + min(qi, nq - 1)) * a.qs[1] + h * a.qs[2] + gq * 32;
    qop[0] = load16(qrow);
    qop[1] = load16(qrow + 16);
  }

  const int64_t sh = slot_head(c, bad ? 0 : slot, h);
  const uint8_t* kc = c.kc + sh * c.n_blk * (kBlk * kHeadDim);
  const uint8_t* vc = c.vc + sh * c.n_blk * (kBlk * kHeadDim);
  const float* ks = c.ks + sh * c.n_blk;
  const float* vs = c.vs + sh * c.n_blk;
  char* kr = c.kr + sh * (kRing * kRowBytes16);
  char* vr = c.vr + sh * (kRing * kRowBytes16);
  const char* kn = HAS_NEW ? a.kn + rows.src * a.kns[0] + h * a.kns[2] : nullptr;
  const char* vn = HAS_NEW ? a.vn + rows.src * a.vns[0] + h * a.vns[2] : nullptr;
  const int code_blks = c.kr ? len / kBlk : 0x7fffffff;  // blocks below are read as codes
  auto row16 = [&](int p, const char* ring, const char* nw, int64_t step) __attribute__((always_inline)) {
    return HAS_NEW && p >= len ? nw + (int64_t)(p - len) * step : ring + (p % kRing) * kRowBytes16;
  };

  // Loads of block blk. Codes: kw[kb] is key 16 kb + qi, dims 16 gq ..; vw[i] piece lane + 64 i of the
  // tile's 128 (row piece / 4). 16-bit rows: kw[2 kb + half], vw[i] piece lane + 64 i of 256.
  // Rows past the end re-read the last key.
  u32x4 kw[4], vw[4];
  float kscale = 0.f, vscale = 0.f;
  auto load_block = [&](int blk) __attribute__((always_inline)) {
    const int p0 = blk * kBlk;
    if (blk < code_blks) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kw[i] = load16_stream(kc + (int64_t)min(p0 + 16 * i + qi, k_last) * kHeadDim + 16 * gq);
        const int piece = lane + 64 * i;
        vw[i] = load16_stream(vc + (int64_t)min(p0 + (piece >> 2), k_last) * kHeadDim + (piece & 3) * 16);
      }
      kscale = ks[blk];
      vscale = vs[blk];
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const char* kp = row16(min(p0 + 16 * kb + qi, k_last), kr, kn, HAS_NEW ? a.kns[1] : 0) + gq * 32;
        kw[2 * kb] = load16(kp);
        kw[2 * kb + 1] = load16(kp + 16);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int piece = lane + 64 * i;
        vw[i] = load16(row16(min(p0 + (piece >> 3), k_last), vr, vn, HAS_NEW ? a.vns[1] : 0) + (piece & 7) * 16);
      }
    }
  };

  uint16_t* vt = sm_v[wave];
  const uint16_t* vt_lane = vt + (4 * gq + (qi >> 2)) * kVPitch + 4 * (qi & 3);
  float m, l;
  f32x4 o[4];  // O^T blocks: dims 16 db + 4 gq + i, query qi

  // SAFE: 16-bit values that are not finite count for the queries that see their key, and for no other
  // (a masked key's probability of 0 times NaN is NaN, and an infinity times the two parts of P also).
  bool safe = false;
  for (;;) {
    m = kNegBig;
    l = 0.f;
#pragma unroll
    for (int db = 0; db < 4; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
    int blk = k_begin / kBlk + wave;
    if (blk * kBlk < k_end) load_block(blk);
    for (; blk * kBlk < k_end; blk += kWaves) {
      const int p0 = blk * kBlk;
      const bool codes = blk < code_blks;
      f32x4 s[2];
      float sscale = a.c;
      const float vsc = vscale;
      if (codes) {
        sscale = a.c * kscale;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = Ops<T>::mfma(widen8<T>(kw[kb][0], kw[kb][1], 1.f), qop[0], f32x4{0.f, 0.f, 0.f, 0.f});
          s[kb] = Ops<T>::mfma(widen8<T>(kw[kb][2], kw[kb][3], 1.f), qop[1], s[kb]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int piece = lane + 64 * i;
          uint16_t* dst = &vt[(piece >> 2) * kVPitch + (piece & 3) * 16];
          *reinterpret_cast<u32x4*>(dst) = widen8<Bf16>(vw[i][0], vw[i][1], vsc);
          *reinterpret_cast<u32x4*>(dst + 8) = widen8<Bf16>(vw[i][2], vw[i][3], vsc);
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = Ops<T>::mfma(kw[2 * kb], qop[0], f32x4{0.f, 0.f, 0.f, 0.f});
          s[kb] = Ops<T>::mfma(kw[2 * kb + 1], qop[1], s[kb]);
        }
        if (safe) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if ((vw[i][w] & Ops<T>::kExp) == Ops<T>::kExp) vw[i][w] &= 0xffff0000u;
              if (((vw[i][w] >> 16) & Ops<T>::kExp) == Ops<T>::kExp) vw[i][w] &= 0xffffu;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int piece = lane + 64 * i;
          *reinterpret_cast<u32x4*>(&vt[(piece >> 3) * kVPitch + (piece & 7) * 8]) = vw[i];
        }
      }
      if ((blk + kWaves) * kBlk < k_end) load_block(blk + kWaves);
      // ---- softmax of the lane's 8 scores (log2 units): keys 16 kb + 4 gq + i ----
      float p[8];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p[kb * 4 + i] = p0 + kb * 16 + 4 * gq + i <= lim ? s[kb][i] * sscale : -INFINITY;
      float mb = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
      mb = group4_max(mb);
      if (__any(mb > m + kTau)) {
        const float mn = mb > m + kTau ? mb : m;
        const float alpha = fast_exp2(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < 4; ++db) o[db] *= alpha;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = fast_exp2(p[j] - m);
        l += p[j];
      }
      if (codes) {
        pv_step<Bf16>(vt_lane, p, o);
      } else {
        pv_step<T>(vt_lane, p, o);
        if (safe) {
          for (int j = 0; j < kBlk; ++j) {
            const float pj = __shfl(p[(j >> 4) * 4 + (j & 3)], qi + 16 * ((j & 15) >> 2));
            const char* row = row16(min(p0 + j, k_last), vr, vn, HAS_NEW ? a.vns[1] : 0);
#pragma unroll
            for (int db = 0; db < 4; ++db) {
              const uint2 w = *reinterpret_cast<const uint2*>(row + (16 * db + 4 * gq) * 2);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const uint32_t x = ((i & 2) ? w.y : w.x) >> (16 * (i & 1)) & 0xffffu;
                if ((x & Ops<T>::kExp) == Ops<T>::kExp && p0 + j <= lim) o[db][i] += pj * Ops<T>::lo(x);
              }
            }
          }
        }
      }
    }
    if (safe) break;
    bool nan = false;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) nan = nan || o[db][i] != o[db][i];
    if (!__any(nan && qi < nq)) break;
    safe = true;
  }

  // row sums: the four lane groups hold different keys of the same query
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (qi < nq) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) sm_acc[wave][qi][16 * db + 4 * gq + i] = o[db][i];
    if (gq == 0) {
      sm_m[wave][qi] = m;
      sm_l[wave][qi] = l;
    }
  }
  __syncthreads();
  kv_finish<T, SQ, kWaves>(a, b, t0, nq, a.n_qblocks > 1 ? SQ : nq, h, split, n_split_b, bad, sm_acc, sm_m, sm_l);

  // ---- the append (sq <= 32): by the last query block's last split of the row that gives the new rows ----
  if constexpr (HAS_NEW) {
    if (!a.append || bad || rows.src != b || t0 + nq != a.sq || split != n_split_b - 1) return;
    const int end = len + a.sq, done = len / kBlk;
    for (int i = tid; i < a.sq * 16; i += kWaves * 64) {
      const int t = i >> 4, which = (i >> 3) & 1, ch = i & 7;
      const char* src = (which ? vn + (int64_t)t * a.vns[1] : kn + (int64_t)t * a.kns[1]) + ch * 16;
      store16((which ? vr : kr) + ((len + t) % kRing) * kRowBytes16 + ch * 16, load16(src));
    }
    if (end / kBlk > done) {  // block `done` is complete
      u32x4 w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      if (tid < 256) {
        const int p = done * kBlk + (tid >> 3);
        w[0] = load16(row16(p, kr, kn, a.kns[1]) + (tid & 7) * 16);
        w[1] = load16(row16(p, vr, vn, a.vns[1]) + (tid & 7) * 16);
      }
      const int64_t code = (sh * c.n_blk + done) * (kBlk * kHeadDim);
      quantize_block<T>(w[0], w[1], c.kc + code, c.vc + code, c.ks + sh * c.n_blk + done, c.vs + sh * c.n_blk + done, sm_red);
    }
  }
}

template <typename T, int SQ, int W>
void launch_attn(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * a.n_qblocks * c.H), 1, a.n_splits), block(W * 64);
  if (a.kn) hipLaunchKernelGGL((kv8_attn_kernel<T, SQ, true, W>), grid, block, 0, stream, c, a);
  else hipLaunchKernelGGL((kv8_attn_kernel<T, SQ, false, W>), grid, block, 0, stream, c, a);
}

template <typename T>
void launch_attn_t(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  if (a.sq == 1) launch_attn<T, 1, 4>(c, a, stream);
  else if (a.sq <= 8) launch_attn<T, 8, 4>(c, a, stream);
  else launch_attn<T, 16, 4>(c, a, stream);
}

template <typename T, typename Id>
void launch_write_t(const Kv8Cache& c, const Kv8WriteArgs& a, const Id* slots, hipStream_t stream) {
  // a row of T positions touches at most this many blocks, wherever it starts
  const int blocks = a.starts ? (a.T + kBlk - 2) / kBlk + 1 : (a.start + a.T - 1) / kBlk - a.start / kBlk + 1;
  const dim3 grid((unsigned)blocks, (unsigned)c.H, (unsigned)a.B);
  hipLaunchKernelGGL((kv8_write_kernel<T, Id>), grid, dim3(256), 0, stream, c, a, slots);
}

}  // namespace

// Splits of a row's keys (see launch_kv8_attn's callers for the workspace): rows that are fewer than
// half the CUs and hold 768 keys or more.
void kv8_plan(int64_t B, int64_t sq, int64_t H, int64_t Lk, Kv8Args* a) {
  const int block = sq == 1 ? 1 : sq <= 8 ? 8 : 16;
  a->n_qblocks = (int)((sq + block - 1) / block);
  a->n_splits = 1;
  a->split_len = (int)((Lk + kBlk - 1) / kBlk * kBlk);
  const int64_t units = B * a->n_qblocks * H;
  if (units <= 128 && Lk >= 768) {
    const int64_t want = std::min<int64_t>(std::min<int64_t>((160 + units - 1) / units, (Lk + 191) / 192), kMaxMergeSplits);
    const int64_t len = ((Lk + want - 1) / want + 63) / 64 * 64;
    a->split_len = (int)len;
    a->n_splits = (int)((Lk + len - 1) / len);
  }
}

size_t kv8_workspace_bytes(int64_t B, int64_t sq, int64_t H, int64_t Lk) {
  Kv8Args a{};
  kv8_plan(B, sq, H, Lk, &a);
  return kv_workspace_bytes(B * a.n_qblocks * H, sq < 16 ? sq : 16, a.n_splits);
}

hipError_t launch_kv8_attn(int dtype, const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  if ((int64_t)a.B * a.n_qblocks * c.H > 0x7fffffff) return hipErrorInvalidValue;
  if (dtype == 2) launch_attn_t<Bf16>(c, a, stream);
  else launch_attn_t<F16>(c, a, stream);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !a.kn || a.append) return err;
  Kv8WriteArgs w{};  // a long prompt's append, behind the launch that reads the ring
  w.k = a.kn;
  w.v = a.vn;
  for (int i = 0; i < 3; ++i) {
    w.ks[i] = a.kns[i];
    w.vs[i] = a.vns[i];
  }
  w.starts = a.seqlens;
  w.B = a.B;
  w.T = a.sq;
  return launch_kv8_write(dtype, c, w, a.bidx, nullptr, stream);
}

hipError_t launch_kv8_write(int dtype, const Kv8Cache& c, const Kv8WriteArgs& a, const int32_t* slots32,
                            const int64_t* slots64, hipStream_t stream) {
  if (slots64) {
    if (dtype == 2) launch_write_t<Bf16>(c, a, slots64, stream);
    else launch_write_t<F16>(c, a, slots64, stream);
  } else {
    if (dtype == 2) launch_write_t<Bf16>(c, a, slots32, stream);
    else launch_write_t<F16>(c, a, slots32, stream);
  }
  return hipGetLastError();
}

}  // namespace wdrz
