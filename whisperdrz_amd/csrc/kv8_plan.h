// kv8_plan.h — how a call of the 8-bit cache's attention (kv8.hip) is cut: its queries and keys into workgroups, a
// workgroup's blocks of keys into codes and 16-bit rows and on to its wavefronts. Whole numbers only, for the
// host and the device alike.
#pragma once

#include <algorithm>

#include "wdrz_launch.h"

namespace wdrz {

constexpr int kKv8Block = 32;          // positions a scale covers
constexpr int kKv8PromptQueries = 64;  // queries a workgroup of many prompts
constexpr int kKv8MaxSplits = 32;      // workgroups a row's keys are cut into at most (kv_merge.h joins no more)

// Blocks of the keys [k_begin, k_end) of a row of `len` written positions: codes [blk0, blk1), 16-bit rows of the
// ring or of the call [blk1, blk2). k_begin is a multiple of 32. Behind `len` there are no codes: a part of an
// append's keys that begins there (split rows) has 16-bit rows alone.
struct Kv8Blocks {
  int blk0, blk1, blk2;
};
__host__ __device__ inline Kv8Blocks kv8_blocks(bool ring, int len, int k_begin, int k_end) {
  const int blk0 = k_begin / kKv8Block, blk2 = (k_end + kKv8Block - 1) / kKv8Block;
  const int whole = (len < k_end ? len : k_end) / kKv8Block;
  return Kv8Blocks{blk0, !ring ? blk2 : whole > blk0 ? whole : blk0, blk2};
}
// The first block of 16-bit rows of a wavefront: blocks are dealt in turn from blk0 on, each wavefront's next one
// `waves` further.
__host__ __device__ inline int kv8_first_rows(const Kv8Blocks& b, int wave, int waves) {
  return b.blk1 + (wave + waves - (b.blk1 - b.blk0) % waves) % waves;
}

// One workgroup walks a row unless few long rows leave most of the chip idle: merging splits costs about
// 2 us (publish, count, read back). One query, bf16, cold caches in a graph, us, unsplit / split:
//   1 stream of 20 heads: 500 positions 4.6 / 6.0, 1000 5.3 / 6.3, 1500 6.4 / 6.9, 3000 11.8 / 7.6, 6000
//   19.1 / 8.9, 20000 58.3 / 14.8; 2 streams: 1500 7.8 / 7.2, 3000 12.0 / 8.4; 4: 1500 8.1 / 8.2, 3000
//   12.2 / 9.7, 6000 22.7 / 14.8; 6: 1500 8.4 / 8.7, 6000 24.0 / 19.7; 8: 1500 9.0 / 10.2.
// More splits than fill the CUs once gain nothing (4 streams of 3000: 3 splits 9.7, 4 10.7). Nor do more queries
// over 1500 positions, 1 / 2 / 3 / 4 splits: five queries of 4 streams 8.7 / 8.7 / 8.5 / 9.8, of 8 10.0 / 12.4 /
// 11.3 / 12.1, of 16 15.1 / 17.0 / 17.0 / 18.2, of 52 39 / 43 / 44 / 46; 17 queries of 52 69 / 84 / 89 / 93. One
// stream's five would gain 0.8 us (8.3 / 8.2 / 7.8 / 7.5).
constexpr int64_t kKv8Cus = 256;
constexpr int64_t kKv8SplitMinLk = 2048;
constexpr int64_t kKv8SplitMinKeys = 512;
// Eight wavefronts a workgroup while the launch has no more workgroups than CUs, else four. Us, eight /
// four: cross over 1500, 1 stream 6.4 / 7.7, 8 9.0 / 11.2, 13 (260 workgroups) 14.6 / 13.0, 32 22.6 / 23.2;
// self of 440, 4 streams 6.0 / 6.9, 52 of 447 14.8 / 12.9. Sixteen are slower from 8 streams on. Five
// queries follow the same lines: cross over 1500, 1 stream 7.6 / 9.2, 8 10.1 / 12.3, 16 16.3 / 16.0; 6000
// positions, 1 stream, 1 / 8 splits 23.3 / 9.6.
// 64 queries a workgroup instead of 16 once blocks of 16 would be more than four workgroups a CU. Us, 16 / 64:
// over 1500 positions 4 prompts of 224 (1120 blocks of 16) 28.4 / 31.8, 8 of 224 (2240) 49.8 / 42.4, 16 of 64
// (1280) 37.3 / 32.3, 8 of 40 (480) 16.5 / 23.6; over themselves 4 of 224 20.0 / 13.4, 16 of 224 46.7 / 27.0,
// 16 of 64 17.9 / 9.6. Up to 32 queries blocks of 16 append in the same launch (52 of 17: 68.8 / 74.3).
constexpr int64_t kKv8PromptWgs = 1024;
inline void kv8_plan(int64_t B, int64_t sq, int64_t H, int64_t Lk, Kv8Args* a) {
  const int block = sq == 1 ? 1 : sq <= 8 ? 8 : sq <= kKv8FusedAppend || B * ((sq + 15) / 16) * H <= kKv8PromptWgs ? 16 : kKv8PromptQueries;
  a->block = block;
  a->append = sq <= kKv8FusedAppend;
  a->n_qblocks = (int)((sq + block - 1) / block);
  a->n_splits = 1;
  a->split_len = (int)((Lk + kKv8Block - 1) / kKv8Block * kKv8Block);
  const int64_t units = B * a->n_qblocks * H;
  if (block < kKv8PromptQueries && units <= kKv8Cus / 2 && Lk >= kKv8SplitMinLk) {
    const int64_t want = std::min<int64_t>(std::min<int64_t>(kKv8Cus / units, Lk / kKv8SplitMinKeys), kKv8MaxSplits);
    const int64_t len = ((Lk + want - 1) / want + kKv8Block - 1) / kKv8Block * kKv8Block;
    a->split_len = (int)len;
    a->n_splits = (int)((Lk + len - 1) / len);
  }
  a->waves = units * a->n_splits <= kKv8Cus ? 8 : 4;
}

}  // namespace wdrz
