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
// and the append rides in the attention launch. Longer prompts append in a launch of their own behind it; many of
// them (kv8_prompt_kernel) write the codes, and the ring where no row reads it, beside their attention.
//
// One query: four lanes a key, dot products and sums on the VALU (kv8_row_kernel). More: a wavefront takes a
// block of 32 keys and up to 16 queries a step on the matrix cores (kv8_attn_kernel):
//   S^T (32 keys x 16 queries) = K Q^T with 4 v_mfma_f32_16x16x32, O^T (64 dims x 16 queries) += V^T P^T
// with 8 more, P in two 16-bit parts. Codes become bf16 (fp16 queries: fp16 for K, whose products are
// then exact too) two an instruction; the keys' scale multiplies the scores in fp32, the values' scale
// is the conversion's own, exact in bf16. A lane's 16-byte load is 16 dimensions of one key: the matrix
// product sums over the dimensions in that order, for K and Q alike. V goes through an LDS tile, as
// codes, and comes back transposed. Both read their codes two blocks ahead.
//
// Bound: the stream of codes. 52 streams, one fp16 query over 1500 positions: 36 us for 200 MB (5.6 TB/s
// with the launch). One query on the matrix cores instead took 59: eight exponentials and a pack for two
// a key, the LDS round trip and 128 registers. Small calls: launch, the trip for the row's metadata, one
// for its keys; 1 stream 6.2 us over 1500, append at 200 4.4 us.
#include "kv8_plan.h"
#include "kv_merge.h"
#include "wdrz_common.h"
#include "wdrz_launch.h"

namespace wdrz {
namespace {

constexpr int kBlk = kKv8Block;           // positions a scale covers
constexpr int kRing = 64;                 // ring rows
static_assert(kKv8MaxSplits <= kMaxMergeSplits, "kv_finish joins no more");
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
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, a), __builtin_bit_cast(v2, b), c, false);
  }
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
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, a), __builtin_bit_cast(v2, b), c, false);
  }
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
// RINGS false: codes only.

// Where row b is written: its slot and first position, or false.
template <typename Id>
__device__ __forceinline__ bool write_row(const Kv8Cache& c, const Kv8WriteArgs& a, const Id* slots, int b, int64_t& slot, int& start) {
  slot = slots ? (int64_t)slots[b] : b;
  start = a.starts ? a.starts[b] : a.start;
  if (slot < 0 || slot >= c.n_slots || start < 0 || start > c.Lk - a.T) return false;
  if (!slots) return true;
  const int from = start;
  const SlotRows r = slot_rows(a.B, slot, from, [&](int i) { return (int64_t)slots[i]; },
                               [&](int i) { return a.starts ? a.starts[i] : from; });
  return !r.conflict && r.src == b;
}

// The x-th block that row b touches.
template <typename T, bool RINGS>
__device__ __forceinline__ void write_block(const Kv8Cache& c, const Kv8WriteArgs& a, int64_t slot, int start, int b, int h, int x,
                                            uint32_t (&red)[2][4]) {
  const int end = start + a.T, first = start / kBlk, last = (end - 1) / kBlk;
  const int blk = first + x;
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
  if (!RINGS || !c.kr) return;
  const int keep = end / kBlk - 1;  // blocks from here on stand in the ring
  const bool shared = start % kBlk != 0;  // the first block has old rows in the ring
  if (blk >= keep && p >= start && p < end && (blk == first || !shared || (blk - first) % 2 != 0)) {
#pragma unroll
    for (int n = 0; n < 2; ++n) store16(rings[n] + (p % kRing) * kRowBytes16, w[n]);
  }
  if (shared && blk == first) {
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

template <typename T, typename Id>
__global__ __launch_bounds__(256) void kv8_write_kernel(Kv8Cache c, Kv8WriteArgs a, const Id* slots) {
  __shared__ uint32_t red[2][4];
  int64_t slot;
  int start;
  if (write_row(c, a, slots, blockIdx.z, slot, start))
    write_block<T, true>(c, a, slot, start, blockIdx.z, blockIdx.y, blockIdx.x, red);
}

// The ring rows of appends that start inside a block, whose codes kv8_prompt_kernel has written.
__global__ __launch_bounds__(256) void kv8_ring_kernel(Kv8Cache c, Kv8WriteArgs a, const int32_t* slots) {
  const int h = blockIdx.x, b = blockIdx.y;
  if (a.starts[b] % kBlk == 0) return;
  int64_t slot;
  int start;
  if (!write_row(c, a, slots, b, slot, start)) return;
  const int end = start + a.T, ch = threadIdx.x & 7;
  const int64_t ring = slot_head(c, slot, h) * (kRing * kRowBytes16) + ch * 16;
  for (int p = max(start, (end / kBlk - 1) * kBlk) + (int)(threadIdx.x >> 3); p < end; p += 32) {
    store16(c.kr + ring + (p % kRing) * kRowBytes16, load16(a.k + b * a.ks[0] + h * a.ks[2] + (int64_t)(p - start) * a.ks[1] + ch * 16));
    store16(c.vr + ring + (p % kRing) * kRowBytes16, load16(a.v + b * a.vs[0] + h * a.vs[2] + (int64_t)(p - start) * a.vs[1] + ch * 16));
  }
}

// The append of an attention launch's new rows as a write.
__host__ __device__ inline Kv8WriteArgs append_args(const Kv8Args& a) {
  Kv8WriteArgs w{};
  w.k = a.kn;
  w.v = a.vn;
  for (int i = 0; i < 3; ++i) {
    w.ks[i] = a.kns[i];
    w.vs[i] = a.vns[i];
  }
  w.starts = a.seqlens;
  w.B = a.B;
  w.T = a.sq;
  return w;
}
// Blocks that a row of T positions touches at most, wherever it starts.
__host__ __device__ inline int touched_blocks(int T) { return (T + kBlk - 2) / kBlk + 1; }

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

// The larger of two values. (fmaxf would first quiet each: three instructions.)
__device__ __forceinline__ float max2(float x, float y) {
#if __HIP_DEVICE_COMPILE__
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
  return r;
#else
  return x > y ? x : y;
#endif
}

// max of x over lanes l, l^16, l^32, l^48, in every lane
__device__ __forceinline__ float group4_max(float x) {
  const auto r32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = max2(__uint_as_float(r32[0]), __uint_as_float(r32[1]));
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max2(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
}

// ---- one query -----------------------------------------------------------------------------------
// Four lanes take a key, 16 dimensions each: q.k on v_dot2 (codes widened to the queries' type, exactly),
// P.V in fp32. A step is 32 keys of codes (a block) or 16 keys of 16-bit rows, 16 registers of raw data
// either way, and two steps are in flight while one is computed. The block that is read from the ring
// and the new row comes first, as two steps of the wavefront that has the fewest blocks.

// The append of a call with sq <= 32 new rows, by one workgroup of every (row, head).
template <typename T, int kThreads>
__device__ __forceinline__ void append_rows(const Kv8Cache& c, const Kv8Args& a, int64_t sh, int len, const char* kn,
                                            const char* vn, uint32_t (&red)[2][4]) {
  const int tid = threadIdx.x, end = len + a.sq, done = len / kBlk;
  char* kr = c.kr + sh * (kRing * kRowBytes16);
  char* vr = c.vr + sh * (kRing * kRowBytes16);
  for (int i = tid; i < a.sq * 16; i += kThreads) {
    const int t = i >> 4, which = (i >> 3) & 1, ch = i & 7;
    const char* src = (which ? vn + (int64_t)t * a.vns[1] : kn + (int64_t)t * a.kns[1]) + ch * 16;
    store16((which ? vr : kr) + ((len + t) % kRing) * kRowBytes16 + ch * 16, load16(src));
  }
  if (end / kBlk == done) return;  // block `done` is not complete yet
  u32x4 w[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (tid < 256) {
    const int p = done * kBlk + (tid >> 3), ch = (tid & 7) * 16;
    w[0] = load16((p >= len ? kn + (int64_t)(p - len) * a.kns[1] : kr + (p % kRing) * kRowBytes16) + ch);
    w[1] = load16((p >= len ? vn + (int64_t)(p - len) * a.vns[1] : vr + (p % kRing) * kRowBytes16) + ch);
  }
  const int64_t blk = sh * c.n_blk + done;
  quantize_block<T>(w[0], w[1], c.kc + blk * (kBlk * kHeadDim), c.vc + blk * (kBlk * kHeadDim), c.ks + blk, c.vs + blk, red);
}

template <typename T, bool RING, bool HAS_NEW, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void kv8_row_kernel(Kv8Cache c, Kv8Args a) {
  static_assert(!HAS_NEW || (RING && kWaves >= 4), "appends need a ring and 256 threads");
  __shared__ float sm_acc[kWaves][1][kHeadDim];
  __shared__ float sm_m[kWaves][1];
  __shared__ float sm_l[kWaves][1];
  __shared__ uint32_t sm_red[2][4];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int kg = lane >> 2, r = lane & 3;  // key of a group of 16, quarter of its row

  const int h = (int)(blockIdx.x % (unsigned)c.H);  // heads fastest: neighbours in the cache run together
  const int b = (int)(blockIdx.x / (unsigned)c.H);
  const int split = blockIdx.z;
  const int slot = a.bidx ? a.bidx[b] : b;
  const int len = a.seqlens ? a.seqlens[b] : c.Lk;
  u32x4 q[2];
  {
    const char* qrow = a.q + b * a.qs[0] + h * a.qs[2] + r * 32;
    q[0] = load16(qrow);
    q[1] = load16(qrow + 16);
  }
  SlotRows rows{b, false};
  if (HAS_NEW && a.bidx)
    rows = slot_rows(a.B, slot, len, [&](int i) { return a.bidx[i]; }, [&](int i) { return a.seqlens[i]; });
  const bool bad = slot < 0 || slot >= c.n_slots || len < 0 || len > c.Lk - (HAS_NEW ? 1 : 0) || rows.conflict;
  const int key_lim = HAS_NEW ? len + 1 : len;
  const int n_split_b = bad ? 1 : max(1, (key_lim + a.split_len - 1) / a.split_len);
  if (split >= n_split_b) return;
  if (!HAS_NEW && key_lim == 0 && !bad) {  // a row without keys
    if (tid < kHeadDim / 2) *reinterpret_cast<uint32_t*>(a.o + b * a.os[0] + h * a.os[2] + tid * 4) = 0;
    return;
  }
  const int k_begin = split * a.split_len;
  const int k_end = bad ? k_begin : min(key_lim, k_begin + a.split_len);
  const int k_last = k_end - 1;
  const int64_t sh = slot_head(c, bad ? 0 : slot, h);
  const uint8_t* kc = c.kc + sh * c.n_blk * (kBlk * kHeadDim) + r * 16;
  const uint8_t* vc = c.vc + sh * c.n_blk * (kBlk * kHeadDim) + r * 16;
  const float* ks = c.ks + sh * c.n_blk;
  const float* vs = c.vs + sh * c.n_blk;
  const char* kn = HAS_NEW ? a.kn + rows.src * a.kns[0] + h * a.kns[2] : nullptr;
  const char* vn = HAS_NEW ? a.vn + rows.src * a.vns[0] + h * a.vns[2] : nullptr;
  // blocks of this split: codes [blk0, blk1), then, where the ring begins inside it, one of 16-bit rows
  const Kv8Blocks part = kv8_blocks(RING, len, k_begin, k_end);
  const int blk0 = part.blk0, blk1 = part.blk1;
  const int tail0 = blk1 * kBlk;
  const int tails = RING && (blk1 - blk0) % kWaves == wave ? (k_end - tail0 + 15) / 16 : 0;  // 16-key steps, at most 2
  const int codes = max(0, (blk1 - blk0 - wave + kWaves - 1) / kWaves);
  const int steps = bad ? 0 : tails + codes;

  struct Step {
    u32x4 k[2], v[2];
    float ks, vs;
  };
  auto row16 = [&](int p, const char* ring, const char* nw) __attribute__((always_inline)) {
    return (HAS_NEW && p >= len ? nw : ring + sh * (kRing * kRowBytes16) + (p % kRing) * kRowBytes16) + r * 32;
  };
  auto load_step = [&](int i, Step& s) __attribute__((always_inline)) {
    if (RING && i < tails) {
      const int p = min(tail0 + 16 * i + kg, k_last);
      const char* kp = row16(p, c.kr, kn);
      const char* vp = row16(p, c.vr, vn);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s.k[u] = load16(kp + 16 * u);
        s.v[u] = load16(vp + 16 * u);
      }
    } else {
      const int blk = blk0 + wave + (i - tails) * kWaves;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int64_t at = (int64_t)min(blk * kBlk + 16 * u + kg, k_last) * kHeadDim;
        s.k[u] = load16_stream(kc + at);
        s.v[u] = load16_stream(vc + at);
      }
      s.ks = ks[blk];
      s.vs = vs[blk];
    }
  };
  float m = kNegBig, l = 0.f, acc[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  auto grow = [&](float s) __attribute__((always_inline)) {  // move the reference when a score exceeds it by > kTau
    if (__any(s > m + kTau)) {
      const float mn = s > m + kTau ? s : m;
      const float alpha = fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[e] *= alpha;
    }
  };
  auto quad_sum = [](float x) __attribute__((always_inline)) {
    x += dpp_xor1(x);
    return x + dpp_xor2(x);
  };
  auto compute_step = [&](int i, const Step& s) __attribute__((always_inline)) {
    if (RING && i < tails) {
      const bool seen = tail0 + 16 * i + kg <= k_last;
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) d = Ops<T>::dot2(q[j / 4][j % 4], s.k[j / 4][j % 4], d);
      const float x = seen ? quad_sum(d) * a.c : -INFINITY;
      grow(x);
      const float p = fast_exp2(x - m);
      l += p;
      if (seen) {  // a masked key's value may not be finite: 0 times it would count
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[2 * j] = __builtin_fmaf(p, Ops<T>::lo(s.v[j / 4][j % 4]), acc[2 * j]);
          acc[2 * j + 1] = __builtin_fmaf(p, Ops<T>::hi(s.v[j / 4][j % 4]), acc[2 * j + 1]);
        }
      }
    } else {
      const int p0 = (blk0 + wave + (i - tails) * kWaves) * kBlk + kg;
      const float ksc = a.c * s.ks;
      float x[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const u32x4 k0 = widen8<T>(s.k[u][0], s.k[u][1], 1.f), k1 = widen8<T>(s.k[u][2], s.k[u][3], 1.f);
        float d = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) d = Ops<T>::dot2(q[0][j], k0[j], d);
#pragma unroll
        for (int j = 0; j < 4; ++j) d = Ops<T>::dot2(q[1][j], k1[j], d);
        x[u] = p0 + 16 * u <= k_last ? quad_sum(d) * ksc : -INFINITY;
      }
      grow(fmaxf(x[0], x[1]));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float e = fast_exp2(x[u] - m);
        l += e;
        const float p = e * s.vs;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(s.v[u][j], false);
          const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(s.v[u][j], true);
          acc[4 * j] = __builtin_fmaf(p, lo[0], acc[4 * j]);
          acc[4 * j + 1] = __builtin_fmaf(p, lo[1], acc[4 * j + 1]);
          acc[4 * j + 2] = __builtin_fmaf(p, hi[0], acc[4 * j + 2]);
          acc[4 * j + 3] = __builtin_fmaf(p, hi[1], acc[4 * j + 3]);
        }
      }
    }
  };
  Step A, B;
  if (steps > 0) load_step(0, A);
  if (steps > 1) load_step(1, B);
  for (int i = 0; i < steps; i += 2) {
    compute_step(i, A);
    if (i + 2 < steps) load_step(i + 2, A);
    if (i + 1 < steps) compute_step(i + 1, B);
    if (i + 3 < steps) load_step(i + 3, B);
  }

  // The 16 key groups of the wavefront: a common maximum, then every halving of the lanes keeps half of the
  // 16 sums, until each lane holds one dimension.
  float mx = fmaxf(m, __shfl_xor(m, 4));
  mx = group4_max(fmaxf(mx, __shfl_xor(mx, 8)));
  const float f = fast_exp2(m - mx);
  l *= f;
#pragma unroll
  for (int off = 4; off <= 32; off *= 2) l += __shfl_xor(l, off);
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] *= f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[e]), __float_as_uint(acc[e + 8]), false, false);
    acc[e] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[e]), __float_as_uint(acc[e + 4]), false, false);
    acc[e] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float give = lane & 8 ? acc[e] : acc[e + 2];
    acc[e] = (lane & 8 ? acc[e + 2] : acc[e]) + __shfl_xor(give, 8);
  }
  const float give = lane & 4 ? acc[0] : acc[1];
  const float one = (lane & 4 ? acc[1] : acc[0]) + __shfl_xor(give, 4);
  const int dim = 16 * r + 8 * (lane >> 5) + 4 * ((lane >> 4) & 1) + 2 * ((lane >> 3) & 1) + ((lane >> 2) & 1);
  sm_acc[wave][0][dim] = one;
  if (lane == 0) {
    sm_m[wave][0] = mx;
    sm_l[wave][0] = l;
  }
  __syncthreads();
  kv_finish<T, 1, kWaves>(a, b, 0, 1, 1, h, split, n_split_b, bad, sm_acc, sm_m, sm_l);
  if constexpr (HAS_NEW) {
    if (!bad && rows.src == b && split == n_split_b - 1) append_rows<T, kWaves * 64>(c, a, sh, len, kn, vn, sm_red);
  }
}

// ---- 2 and more queries ----------------------------------------------------------------------------

// Transposing LDS read of bytes (ds_read_b64_tr_b8): within each 16-lane group, lane i receives byte i%8
// of the 8-byte chunks read by lanes 2c + i/8 (c = 0..7), in the order of c.
__device__ __forceinline__ u32x2 read_tr8(const uint8_t* p) {
#if __HIP_DEVICE_COMPILE__
  typedef int i32x2 __attribute__((ext_vector_type(2)));
  typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(uint32_t)(uintptr_t)p));
#else
  (void)p;
  return u32x2{0, 0};
#endif
}

// The largest of a lane's 8 scores, in four instructions.
__device__ __forceinline__ float max8(const float (&x)[8]) {
#if __HIP_DEVICE_COMPILE__
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x[0]), "v"(x[1]), "v"(x[2]));
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(r) : "v"(x[3]), "v"(x[4]));
  asm("v_max3_f32 %0, %0, %1, %2" : "+v"(r) : "v"(x[5]), "v"(x[6]));
  return max2(r, x[7]);
#else
  return x[0];
#endif
}

// The lane's 8 probabilities as two operands of type E: the rounded values and what the rounding left,
// so that they count with 16 bits or more.
template <typename E>
__device__ __forceinline__ void split_p(const float (&p)[8], u32x4& ph, u32x4& pl) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ph[j] = Ops<E>::pack(p[2 * j], p[2 * j + 1]);
    asm("" : "+v"(ph[j]));  // else its halves are rounded a second time
    pl[j] = Ops<E>::pack(p[2 * j] - Ops<E>::lo(ph[j]), p[2 * j + 1] - Ops<E>::hi(ph[j]));
  }
}

constexpr int kV8Pitch = kHeadDim + 16;  // row pitch (bytes) of a tile of codes

// SQ: query rows a workgroup (8 or 16). RING: the cache has one; HAS_NEW: the call appends.
template <typename T, int SQ, bool RING, bool HAS_NEW, int kWaves>
__global__ __launch_bounds__(kWaves * 64, 4) void kv8_attn_kernel(Kv8Cache c, Kv8Args a) {
  static_assert(!HAS_NEW || RING, "appends need a ring");
  __shared__ float sm_acc[kWaves][SQ][kHeadDim];
  __shared__ float sm_m[kWaves][SQ];
  __shared__ float sm_l[kWaves][SQ];
  // one V tile a wavefront: 32 rows of codes, or of 16-bit values
  __shared__ __attribute__((aligned(16))) uint8_t sm_v[kWaves][RING ? kBlk * kVPitch * 2 : kBlk * kV8Pitch];
  __shared__ uint32_t sm_red[2][4];

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int qi = lane & 15, gq = lane >> 4;  // query slot (and key row) of this lane, 16-lane group

  const int h = (int)(blockIdx.x % (unsigned)c.H);
  const int bq = (int)(blockIdx.x / (unsigned)c.H);
  const int b = bq / a.n_qblocks;
  const int t0 = (bq % a.n_qblocks) * SQ;
  const int split = blockIdx.z;
  const int nq = min(SQ, a.sq - t0);

  const int slot = a.bidx ? a.bidx[b] : b;
  const int len = a.seqlens ? a.seqlens[b] : c.Lk;
  // Q^T operand halves: query t0 + qi, dims 16 gq + 8 dh .. + 7
  u32x4 qop[2];
  {
    const char* qrow = a.q + b * a.qs[0] + (t0 + min(qi, nq - 1)) * a.qs[1] + h * a.qs[2] + gq * 32;
    qop[0] = load16(qrow);
    qop[1] = load16(qrow + 16);
  }
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
  // last key this lane's query may see
  const int lim = HAS_NEW ? min(k_last, len + t0 + qi) : k_last;

  const int64_t sh = slot_head(c, bad ? 0 : slot, h);
  const uint8_t* kc = c.kc + sh * c.n_blk * (kBlk * kHeadDim);
  const uint8_t* vc = c.vc + sh * c.n_blk * (kBlk * kHeadDim);
  const float* ks = c.ks + sh * c.n_blk;
  const float* vs = c.vs + sh * c.n_blk;
  const char* kn = HAS_NEW ? a.kn + rows.src * a.kns[0] + h * a.kns[2] : nullptr;
  const char* vn = HAS_NEW ? a.vn + rows.src * a.vns[0] + h * a.vns[2] : nullptr;
  // blocks of this split: codes [blk0, blk1), then 16-bit rows [blk1, blk2), dealt on to the wavefronts in turn
  const Kv8Blocks part = kv8_blocks(RING, len, k_begin, k_end);
  const int blk0 = part.blk0, blk1 = part.blk1, blk2 = part.blk2;

  uint8_t* vt = sm_v[wave];
  float m = kNegBig, l = 0.f;
  f32x4 o[4];  // O^T blocks: dims 16 db + 4 gq + i, query qi
#pragma unroll
  for (int db = 0; db < 4; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  // The running maximum and the probabilities of one block's scores (times `scale`, log2 units): keys
  // 16 kb + 4 gq + i of it; those past `last` do not count.
  auto softmax = [&](const f32x4 (&s)[2], float scale, int last, float (&p)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = s[j >> 2][j & 3];
    if (__any(last < kBlk - 1)) {  // masked behind the scale, which may be 0 (a block nobody wrote): 0 times -inf is NaN
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j] = (j >> 2) * 16 + 4 * gq + (j & 3) > last ? -INFINITY : p[j] * scale;
      scale = 1.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(p[j]));  // keep this rare path a branch
    }
    const float mb = group4_max(max8(p)) * scale;
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
      p[j] = fast_exp2(__builtin_fmaf(p[j], scale, -m));
      l += p[j];
    }
  };

  // ---- blocks of codes: kw[i] is key 16 i + qi, dims 16 gq ..; vw[i] piece lane + 64 i of the tile's 128
  // (row piece / 4). Two blocks in flight while one is computed. Rows past the end re-read the last key.
  struct Codes {
    u32x4 k[2], v[2];
    float ks, vs;
  };
  auto load_codes = [&](int blk, Codes& x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int piece = lane + 64 * i;
      x.k[i] = load16_stream(kc + (int64_t)min(blk * kBlk + 16 * i + qi, k_last) * kHeadDim + 16 * gq);
      x.v[i] = load16_stream(vc + (int64_t)min(blk * kBlk + (piece >> 2), k_last) * kHeadDim + (piece & 3) * 16);
    }
    x.ks = ks[blk];
    x.vs = vs[blk];
  };
  auto compute_codes = [&](int blk, const Codes& x) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int piece = lane + 64 * i;
      *reinterpret_cast<u32x4*>(vt + (piece >> 2) * kV8Pitch + (piece & 3) * 16) = x.v[i];
    }
    f32x4 s[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = Ops<T>::mfma(widen8<T>(x.k[kb][0], x.k[kb][1], 1.f), qop[0], f32x4{0.f, 0.f, 0.f, 0.f});
      s[kb] = Ops<T>::mfma(widen8<T>(x.k[kb][2], x.k[kb][3], 1.f), qop[1], s[kb]);
    }
    float p[8];
    softmax(s, a.c * x.ks, k_last - blk * kBlk, p);
    u32x4 ph, pl;
    split_p<Bf16>(p, ph, pl);
    // V^T operands in the scores' key order: keys 4 gq + (0..3) and 16 + 4 gq + (0..3), dims 16 db + qi
    const int row = (qi >> 1) < 4 ? 4 * gq + (qi >> 1) : 12 + 4 * gq + (qi >> 1);
    const uint8_t* at = vt + row * kV8Pitch + (qi & 1) * 8;
#pragma unroll
    for (int db = 0; db < 4; ++db) {
      const u32x2 w = read_tr8(at + 16 * db);
      const u32x4 v = widen8<Bf16>(w[0], w[1], x.vs);
      o[db] = Ops<Bf16>::mfma(v, pl, o[db]);
      o[db] = Ops<Bf16>::mfma(v, ph, o[db]);
    }
  };
  int blk = blk0 + wave;
  Codes A, B;
  if (blk < blk1) load_codes(blk, A);
  if (blk + kWaves < blk1) load_codes(blk + kWaves, B);

  // ---- blocks of 16-bit rows: the ring's, then the new ones. Values that are not finite stay out of the
  // matrix product, where a masked key's 0 times NaN would be NaN (and an infinity times the two parts of P
  // too), and count for the queries that see their key, one by one.
  if constexpr (RING) {
    auto row16 = [&](int p, const char* ring, const char* nw, int64_t step) __attribute__((always_inline)) {
      return HAS_NEW && p >= len ? nw + (int64_t)(p - len) * step : ring + sh * (kRing * kRowBytes16) + (p % kRing) * kRowBytes16;
    };
    const int64_t kstep = HAS_NEW ? a.kns[1] : 0, vstep = HAS_NEW ? a.vns[1] : 0;
    uint16_t* vt16 = reinterpret_cast<uint16_t*>(vt);
    for (int tb = kv8_first_rows(part, wave, kWaves); tb < blk2; tb += kWaves) {
      const int p0 = tb * kBlk;
      u32x4 kw[4], vw[4];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const char* kp = row16(min(p0 + 16 * kb + qi, k_last), c.kr, kn, kstep) + gq * 32;
        kw[2 * kb] = load16(kp);
        kw[2 * kb + 1] = load16(kp + 16);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int piece = lane + 64 * i;
        vw[i] = load16(row16(min(p0 + (piece >> 3), k_last), c.vr, vn, vstep) + (piece & 7) * 16);
      }
      f32x4 s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        s[kb] = Ops<T>::mfma(kw[2 * kb], qop[0], f32x4{0.f, 0.f, 0.f, 0.f});
        s[kb] = Ops<T>::mfma(kw[2 * kb + 1], qop[1], s[kb]);
      }
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const bool lo = (vw[i][w] & Ops<T>::kExp) == Ops<T>::kExp;
          const bool hi = ((vw[i][w] >> 16) & Ops<T>::kExp) == Ops<T>::kExp;
          odd = odd || lo || hi;
          vw[i][w] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu);
        }
        const int piece = lane + 64 * i;
        *reinterpret_cast<u32x4*>(&vt16[(piece >> 3) * kVPitch + (piece & 7) * 8]) = vw[i];
      }
      float p[8];
      softmax(s, a.c, lim - p0, p);
      u32x4 ph, pl;
      split_p<T>(p, ph, pl);
      const uint16_t* at = vt16 + (4 * gq + (qi >> 2)) * kVPitch + 4 * (qi & 3);
#pragma unroll
      for (int db = 0; db < 4; ++db) {
        const u32x2 v0 = read_tr16(at + 16 * db), v1 = read_tr16(at + 16 * kVPitch + 16 * db);
        const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
        o[db] = Ops<T>::mfma(v, pl, o[db]);
        o[db] = Ops<T>::mfma(v, ph, o[db]);
      }
      if (__any(odd)) {
        for (int j = 0; j < kBlk; ++j) {
          float pj = 0.f;  // the probability of key j, from the lane and register that hold it
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const float x = __shfl(p[r], qi + 16 * ((j & 15) >> 2));
            if (r == (j >> 4) * 4 + (j & 3)) pj = x;
          }
          if (p0 + j > lim) continue;
          const char* row = row16(min(p0 + j, k_last), c.vr, vn, vstep);
#pragma unroll
          for (int db = 0; db < 4; ++db) {
            const uint2 w = *reinterpret_cast<const uint2*>(row + (16 * db + 4 * gq) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t x = ((i & 2) ? w.y : w.x) >> (16 * (i & 1)) & 0xffffu;
              if ((x & Ops<T>::kExp) == Ops<T>::kExp) o[db][i] += pj * Ops<T>::lo(x);
            }
          }
        }
      }
    }
  }
  for (; blk < blk1; blk += 2 * kWaves) {
    compute_codes(blk, A);
    if (blk + 2 * kWaves < blk1) load_codes(blk + 2 * kWaves, A);
    if (blk + kWaves < blk1) compute_codes(blk + kWaves, B);
    if (blk + 3 * kWaves < blk1) load_codes(blk + 3 * kWaves, B);
  }

  // row sums: the four lane groups hold different keys of the same query
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (qi < nq) {
#pragma unroll
    for (int db = 0; db < 4; ++db)
      *reinterpret_cast<f32x4*>(&sm_acc[wave][qi][16 * db + 4 * gq]) = o[db];
    if (gq == 0) {
      sm_m[wave][qi] = m;
      sm_l[wave][qi] = l;
    }
  }
  __syncthreads();
  kv_finish<T, SQ, kWaves>(a, b, t0, nq, a.n_qblocks > 1 ? SQ : nq, h, split, n_split_b, bad, sm_acc, sm_m, sm_l);

  if constexpr (HAS_NEW) {  // the last query block's last split of the row that gives the new rows
    if (a.append && !bad && rows.src == b && t0 + nq == a.sq && split == n_split_b - 1)
      append_rows<T, kWaves * 64>(c, a, sh, len, kn, vn, sm_red);
  }
}

// ---- prompts ---------------------------------------------------------------------------------------
// 64 queries a workgroup, 16 a wavefront. Stages of up to 64 keys are widened to 16 bits once for the
// four wavefronts, into one of two LDS buffers while the other is computed; no partial leaves a wavefront.
// First the stages of codes, then those of 16-bit rows (the ring's and the new ones). The probabilities'
// sums come from the matrix cores too. Bound: issue, 28 matrix products of 16 cycles and about 145 VALU instructions a
// wavefront and stage, which add up: softmax and matrix products of a SIMD's wavefronts hardly overlap (counters of 16
// prompts of 224 over 1500 positions: VALU 60% of the time, MFMA 33%, both at once 11%). These take 67 us, 64 prompts
// 245; in blocks of 16 queries 95. Over themselves, with the append's workgroups behind those of the attention, 26 us;
// with the append in a launch of its own 31 (it takes 10), with each row's next to its attention's 31. 32 queries a
// wavefront and stages of 32 keys were slower. Probabilities of bf16 prompts as one fp16 operand instead of two parts
// took 64 us, 64 prompts 220, but are wrong where many small ones count.
constexpr int kStageKeys = 2 * kBlk;

constexpr int kPromptQueries = kKv8PromptQueries;

template <typename T, bool RING, bool HAS_NEW>
__global__ __launch_bounds__(256, 4) void kv8_prompt_kernel(Kv8Cache c, Kv8Args a) {
  static_assert(!HAS_NEW || RING, "appends need a ring");
  __shared__ __attribute__((aligned(16))) uint16_t sm_k[2][kStageKeys * kVPitch], sm_v[2][kStageKeys * kVPitch];
  __shared__ int sm_odd[2];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int qi = lane & 15, gq = lane >> 4;

  const int h = (int)(blockIdx.x % (unsigned)c.H);
  const int bq = (int)(blockIdx.x / (unsigned)c.H);
  if (HAS_NEW && bq >= a.B * a.n_qblocks) {
    // The append's workgroups. They write codes of blocks from len / 32 on, which nobody reads here. Ring
    // rows are read only where len ends inside a block; those rows' are written by kv8_ring_kernel.
    const int x = bq - a.B * a.n_qblocks, row = x % a.B;
    const Kv8WriteArgs w = append_args(a);
    int64_t to;
    int start;
    if (!write_row(c, w, a.bidx, row, to, start)) return;
    uint32_t(&red)[2][4] = *reinterpret_cast<uint32_t(*)[2][4]>(sm_k);
    if (start % kBlk == 0) write_block<T, true>(c, w, to, start, row, h, x / a.B, red);
    else write_block<T, false>(c, w, to, start, row, h, x / a.B, red);
    return;
  }
  // the last queries of a causal prompt see the most keys: they start first
  const int b = bq / a.n_qblocks, item = a.n_qblocks - 1 - bq % a.n_qblocks;
  // a prompt's blocks of 16 queries, spread evenly over its workgroups: three or four each
  const int n16 = (a.sq + 15) / 16, q0 = item * n16 / a.n_qblocks, q1 = (item + 1) * n16 / a.n_qblocks;
  const int t0 = q0 * 16, nq = min(q1 * 16, a.sq) - t0;
  const int slot = a.bidx ? a.bidx[b] : b;
  const int len = a.seqlens ? a.seqlens[b] : c.Lk;
  // The wavefront without queries is another one from workgroup to workgroup of a CU, so that its SIMDs get alike.
  const int wq = (wave + (int)(blockIdx.x >> 8)) & 3;
  const int w0 = t0 + wq * 16;  // this wavefront's first query
  u32x4 qop[2];  // Q^T halves: query w0 + qi, dims 32 dh + 8 gq ..
  {
    const char* qrow = a.q + b * a.qs[0] + min(w0 + qi, a.sq - 1) * a.qs[1] + h * a.qs[2] + gq * 16;
    qop[0] = load16(qrow);
    qop[1] = load16(qrow + 64);
  }
  SlotRows rows{b, false};
  if (HAS_NEW && a.bidx)
    rows = slot_rows(a.B, slot, len, [&](int i) { return a.bidx[i]; }, [&](int i) { return a.seqlens[i]; });
  const bool bad = slot < 0 || slot >= c.n_slots || len < 0 || len > c.Lk - (HAS_NEW ? a.sq : 0) || rows.conflict;
  const int k_end = bad ? 0 : HAS_NEW ? len + t0 + nq : len, k_last = k_end - 1;
  // the last key that any query of this wavefront sees
  const int w_end = wq >= q1 - q0 ? 0 : HAS_NEW ? min(k_end, len + w0 + 16) : k_end;
  const int64_t sh = slot_head(c, bad ? 0 : slot, h);
  const uint8_t* codes = (tid < 128 ? c.kc : c.vc) + sh * c.n_blk * (kBlk * kHeadDim) + (tid & 3) * 16;
  const float* ks = c.ks + sh * c.n_blk;
  const float* vs = c.vs + sh * c.n_blk;
  const char* kn = HAS_NEW ? a.kn + rows.src * a.kns[0] + h * a.kns[2] : nullptr;
  const char* vn = HAS_NEW ? a.vn + rows.src * a.vns[0] + h * a.vns[2] : nullptr;
  const int64_t kstep = HAS_NEW ? a.kns[1] : 0, vstep = HAS_NEW ? a.vns[1] : 0;
  const Kv8Blocks part = kv8_blocks(RING, len, 0, k_end);
  const int blk1 = part.blk1, blk2 = part.blk2;

  float m = kNegBig;
  f32x4 o[5];  // O^T blocks: dims 16 db + 4 gq + i, query qi; the last one the query's sum of probabilities
#pragma unroll
  for (int db = 0; db < 5; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto row16 = [&](int p, const char* ring, const char* nw, int64_t step) __attribute__((always_inline)) {
    return HAS_NEW && p >= len ? nw + (int64_t)(p - len) * step : ring + sh * (kRing * kRowBytes16) + (p % kRing) * kRowBytes16;
  };
  // One stage: rows of buffer `buf`, positions p0 .. p0 + 63 below `end`; block_scale[half] of the scores of each 32 of them,
  // E the values' type. Both blocks go through each step together: one maximum, one branch, twice the
  // independent work.
  auto compute = [&](int buf, int p0, int end, const float (&block_scale)[2], bool odd, auto etag) __attribute__((always_inline)) {
    typedef decltype(etag) E;
    if (p0 >= w_end) return;  // no query of this wavefront sees the stage
    float p[2][8];
    {
      const uint16_t* kt = &sm_k[buf][qi * kVPitch + 8 * gq];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        f32x4 s = Ops<T>::mfma(*reinterpret_cast<const u32x4*>(kt + 16 * kb * kVPitch), qop[0], f32x4{0.f, 0.f, 0.f, 0.f});
        s = Ops<T>::mfma(*reinterpret_cast<const u32x4*>(kt + 16 * kb * kVPitch + 32), qop[1], s);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[kb >> 1][(kb & 1) * 4 + i] = s[i];
      }
    }
    // the last key of the stage that this query sees
    const int lim = min(HAS_NEW ? min(k_last, len + w0 + qi) : k_last, end - 1) - p0;
    float scale[2] = {block_scale[0], block_scale[1]};
    if (p0 + kStageKeys > min(w_end - (HAS_NEW ? 16 : 0), end)) {  // behind the scale, as in kv8_attn_kernel
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float& x = p[j >> 3][j & 7];
        x = (j >> 2) * 16 + 4 * gq + (j & 3) > lim ? -INFINITY : x * scale[j >> 3];
        asm volatile("" : "+v"(x));  // keep this rare path a branch
      }
      scale[0] = scale[1] = 1.f;
    }
    const float mb = group4_max(max2(max8(p[0]) * scale[0], max8(p[1]) * scale[1]));
    if (__any(mb > m + kTau)) {
      const float mn = mb > m + kTau ? mb : m;
      const float alpha = fast_exp2(m - mn);
      m = mn;
#pragma unroll
      for (int db = 0; db < 5; ++db) o[db] *= alpha;
    }
    constexpr uint32_t kOne = __is_same(E, Bf16) ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < 8; ++j) p[half][j] = fast_exp2(__builtin_fmaf(p[half][j], scale[half], -m));
      u32x4 ph, pl;
      split_p<E>(p[half], ph, pl);
      const uint16_t* at = &sm_v[buf][(half * kBlk + 4 * gq + (qi >> 2)) * kVPitch + 4 * (qi & 3)];
#pragma unroll
      for (int db = 0; db < 5; ++db) {
        u32x4 v = {kOne, kOne, kOne, kOne};
        if (db < 4) {
          const u32x2 v0 = read_tr16(at + 16 * db), v1 = read_tr16(at + 16 * kVPitch + 16 * db);
          v = u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
        o[db] = Ops<E>::mfma(v, pl, o[db]);
        o[db] = Ops<E>::mfma(v, ph, o[db]);
      }
    }
    if (odd) {  // values that are not finite, one by one (see kv8_attn_kernel)
      for (int j = 0; j < kStageKeys; ++j) {
        const char* row = row16(min(p0 + j, k_last), c.vr, vn, vstep);
        float pj = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = __shfl(p[r >> 3][r & 7], qi + 16 * ((j & 15) >> 2));
          if (r == (j >> 4) * 4 + (j & 3)) pj = x;
        }
        if (j > lim) continue;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
          const uint2 w = *reinterpret_cast<const uint2*>(row + (16 * db + 4 * gq) * 2);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t x = ((i & 2) ? w.y : w.x) >> (16 * (i & 1)) & 0xffffu;
            if ((x & Ops<T>::kExp) == Ops<T>::kExp) o[db][i] += pj * Ops<T>::lo(x);
          }
        }
      }
    }
  };

  // ---- codes: threads 0..127 move K, the others V, a 16-byte piece (a quarter row) of each block ----
  // The values become bf16, which holds a code times a scale of any size; so do the two parts of a probability, whose
  // small ones stay what they are (one fp16 operand would drop those under 2^-25: a million of them are 3% of a sum).
  if (blk1 > 0) {
    u32x4 raw[2];
    float kscale[2], vscale[2];
    auto fetch = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int x = min(blk + i, blk1 - 1);
        raw[i] = load16(codes + (int64_t)min(x * kBlk + (tid >> 2 & 31), k_last) * kHeadDim);
        kscale[i] = ks[x];
        vscale[i] = vs[x];
      }
    };
    auto stage = [&](int buf) __attribute__((always_inline)) {
      uint16_t* to = (tid < 128 ? sm_k : sm_v)[buf] + (tid >> 2 & 31) * kVPitch + (tid & 3) * 16;
      auto put = [&](auto etag, float s0, float s1) __attribute__((always_inline)) {
        typedef decltype(etag) E;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          *reinterpret_cast<u32x4*>(to + i * kBlk * kVPitch) = widen8<E>(raw[i][0], raw[i][1], i ? s1 : s0);
          *reinterpret_cast<u32x4*>(to + i * kBlk * kVPitch + 8) = widen8<E>(raw[i][2], raw[i][3], i ? s1 : s0);
        }
      };
      if (tid < 128) put(T{}, 1.f, 1.f);
      else put(Bf16{}, vscale[0], vscale[1]);
    };
    fetch(0);
    stage(0);
    __syncthreads();
    for (int blk = 0, buf = 0; blk < blk1; blk += 2, buf ^= 1) {
      const float scale[2] = {a.c * kscale[0], a.c * kscale[1]};
      fetch(blk + 2);
      compute(buf, blk * kBlk, blk1 * kBlk, scale, false, Bf16{});
      stage(buf ^ 1);  // last read before the barrier that ended the stage before
      __syncthreads();
    }
  }
  // ---- 16-bit rows: a 16-byte piece of K and of V a thread and block ----
  if (RING && blk2 > blk1) {
    u32x4 rk[2], rv[2];
    auto fetch = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int p = min((blk + i) * kBlk + (tid >> 3), k_last);
        rk[i] = load16(row16(p, c.kr, kn, kstep) + (tid & 7) * 16);
        rv[i] = load16(row16(p, c.vr, vn, vstep) + (tid & 7) * 16);
      }
    };
    auto stage = [&](int buf) __attribute__((always_inline)) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = (i * kBlk + (tid >> 3)) * kVPitch + (tid & 7) * 8;
        *reinterpret_cast<u32x4*>(&sm_k[buf][at]) = rk[i];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const bool lo = (rv[i][w] & Ops<T>::kExp) == Ops<T>::kExp, hi = ((rv[i][w] >> 16) & Ops<T>::kExp) == Ops<T>::kExp;
          odd = odd || lo || hi;
          rv[i][w] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu);
        }
        *reinterpret_cast<u32x4*>(&sm_v[buf][at]) = rv[i];
      }
      if (odd) sm_odd[buf] = 1;
    };
    if (tid < 2) sm_odd[tid] = 0;
    __syncthreads();
    fetch(blk1);
    stage(0);
    __syncthreads();
    for (int blk = blk1, buf = 0; blk < blk2; blk += 2, buf ^= 1) {
      fetch(blk + 2);
      const float scale[2] = {a.c, a.c};
      compute(buf, blk * kBlk, blk2 * kBlk, scale, sm_odd[buf] != 0, T{});
      stage(buf ^ 1);
      __syncthreads();
    }
  }
  const int t = w0 + qi;
  if (wq >= q1 - q0 || t >= a.sq) return;
  char* op = a.o + b * a.os[0] + t * a.os[1] + h * a.os[2] + gq * 8;
#pragma unroll
  for (int db = 0; db < 4; ++db) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = bad ? quiet_nan() : k_end == 0 ? 0.f : o[db][i] / o[4][0];
    *reinterpret_cast<u32x2*>(op + db * 32) = u32x2{Ops<T>::pack(v[0], v[1]), Ops<T>::pack(v[2], v[3])};
  }
}

template <typename T, int SQ, int W>
void launch_attn(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * a.n_qblocks * c.H), 1, a.n_splits), block(W * 64);
  if (a.kn) hipLaunchKernelGGL((kv8_attn_kernel<T, SQ, true, true, W>), grid, block, 0, stream, c, a);
  else if (c.kr) hipLaunchKernelGGL((kv8_attn_kernel<T, SQ, true, false, W>), grid, block, 0, stream, c, a);
  else hipLaunchKernelGGL((kv8_attn_kernel<T, SQ, false, false, W>), grid, block, 0, stream, c, a);
}

template <typename T>
void launch_prompt(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * (a.n_qblocks + (a.kn ? touched_blocks(a.sq) : 0)) * c.H)), block(256);
  if (a.kn) hipLaunchKernelGGL((kv8_prompt_kernel<T, true, true>), grid, block, 0, stream, c, a);
  else if (c.kr) hipLaunchKernelGGL((kv8_prompt_kernel<T, true, false>), grid, block, 0, stream, c, a);
  else hipLaunchKernelGGL((kv8_prompt_kernel<T, false, false>), grid, block, 0, stream, c, a);
}

template <typename T, int W>
void launch_row(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  const dim3 grid((unsigned)((int64_t)a.B * c.H), 1, a.n_splits), block(W * 64);
  if (a.kn) hipLaunchKernelGGL((kv8_row_kernel<T, true, true, W>), grid, block, 0, stream, c, a);
  else if (c.kr) hipLaunchKernelGGL((kv8_row_kernel<T, true, false, W>), grid, block, 0, stream, c, a);
  else hipLaunchKernelGGL((kv8_row_kernel<T, false, false, W>), grid, block, 0, stream, c, a);
}

template <typename T>
void launch_row_t(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  if (a.waves == 8) launch_row<T, 8>(c, a, stream);
  else launch_row<T, 4>(c, a, stream);
}

template <typename T>
void launch_attn_t(const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  if (a.sq == 1) launch_row_t<T>(c, a, stream);
  else if (a.block == kPromptQueries) launch_prompt<T>(c, a, stream);
  else if (a.sq <= 8 && a.waves == 8) launch_attn<T, 8, 8>(c, a, stream);
  else if (a.sq <= 8) launch_attn<T, 8, 4>(c, a, stream);
  else if (a.waves == 8) launch_attn<T, 16, 8>(c, a, stream);
  else launch_attn<T, 16, 4>(c, a, stream);
}

template <typename T, typename Id>
void launch_write_t(const Kv8Cache& c, const Kv8WriteArgs& a, const Id* slots, hipStream_t stream) {
  const int blocks = a.starts ? touched_blocks(a.T) : (a.start + a.T - 1) / kBlk - a.start / kBlk + 1;
  const dim3 grid((unsigned)blocks, (unsigned)c.H, (unsigned)a.B);
  hipLaunchKernelGGL((kv8_write_kernel<T, Id>), grid, dim3(256), 0, stream, c, a, slots);
}

}  // namespace

size_t kv8_workspace_bytes(int64_t B, int64_t sq, int64_t H, int64_t Lk) {
  Kv8Args a{};
  kv8_plan(B, sq, H, Lk, &a);
  return kv_workspace_bytes(B * a.n_qblocks * H, sq < 16 ? sq : 16, a.n_splits);
}

hipError_t launch_kv8_attn(int dtype, const Kv8Cache& c, const Kv8Args& a, hipStream_t stream) {
  if ((int64_t)a.B * (a.n_qblocks + touched_blocks(a.sq)) * c.H > 0x7fffffff) return hipErrorInvalidValue;
  if (dtype == 2) launch_attn_t<Bf16>(c, a, stream);
  else launch_attn_t<F16>(c, a, stream);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || !a.kn || a.append) return err;
  // a long prompt's append, or what is left of it, behind the launch that reads the ring
  const Kv8WriteArgs w = append_args(a);
  if (a.block != kPromptQueries) return launch_kv8_write(dtype, c, w, a.bidx, nullptr, stream);
  hipLaunchKernelGGL(kv8_ring_kernel, dim3((unsigned)c.H, (unsigned)a.B), dim3(256), 0, stream, c, w, a.bidx);
  return hipGetLastError();
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
