"""How the 8-bit cache's attention cuts its keys (whisperdrz_amd/csrc/kv8_plan.h, the arithmetic that the kernels
compile): over many sizes every key block of every block of queries is taken exactly once, complete blocks as
codes and the others as 16-bit rows."""
import os
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "whisperdrz_amd" / "csrc"

SOURCE = r"""
#include <cstdio>
#include <vector>
#include "kv8_plan.h"
using namespace wdrz;

static long calls = 0, split_rows = 0, behind = 0;

// One row of `len` positions: append says whether the call's sq rows are appended.
static bool row(int64_t B, int64_t sq, int64_t H, int64_t Lk, int len, bool append, bool ring) {
  Kv8Args a{};
  kv8_plan(B, sq, H, Lk, &a);
  ++calls;
  for (int qb = 0; qb < a.n_qblocks; ++qb) {
    // a prompt's workgroups of 64 queries walk all of their keys and are not split
    const int t0 = qb * a.block, nq = (int)(sq - t0 < a.block ? sq - t0 : a.block);
    const int lim = append ? len + t0 + nq : len;
    const int c0 = ring ? len / 32 : (lim + 31) / 32;
    std::vector<int> seen((lim + 31) / 32, 0);
    const int n_split = lim ? (lim + a.split_len - 1) / a.split_len : 1;
    if (n_split > a.n_splits || n_split > kKv8MaxSplits) return false;
    split_rows += n_split > 1;
    for (int split = 0; split < n_split; ++split) {
      const int begin = split * a.split_len, end = lim < begin + a.split_len ? lim : begin + a.split_len;
      if (begin % 32) return false;
      const Kv8Blocks b = kv8_blocks(ring, len, begin, end);
      behind += ring && begin > len;
      if (b.blk1 < b.blk0 || b.blk2 < b.blk1) return false;
      if (a.block == 1 && b.blk2 - b.blk1 > 1) return false;  // one query: at most one block of 16-bit rows
      for (int wave = 0; wave < a.waves; ++wave) {
        for (int i = b.blk0 + wave; i < b.blk1; i += a.waves) {
          if (i < b.blk0 || i >= c0) return false;
          ++seen[i];
        }
        for (int i = kv8_first_rows(b, wave, a.waves); i < b.blk2; i += a.waves) {
          if (i < b.blk0 || i < c0) return false;
          ++seen[i];
        }
      }
    }
    for (int n : seen)
      if (n != 1) return false;
  }
  return true;
}

int main() {
  const int64_t heads[] = {1, 2, 4, 20}, lens[] = {64, 447, 1500, 2048, 2300, 4096, 6001};
  const int64_t sqs[] = {1, 2, 5, 8, 9, 16, 17, 32, 33, 64, 130, 1100};
  for (int64_t H : heads)
    for (int64_t Lk : lens)
      for (int64_t sq : sqs)
        for (int64_t B : {1, 3, 20}) {
          Kv8Args a{};
          kv8_plan(B, sq, H, Lk, &a);
          for (int64_t at = 0; at <= Lk + a.split_len; at += a.split_len)
            for (int64_t d : {-1101, -64, -63, -33, -32, -31, -17, -5, -4, -2, -1, 0, 1, 31, 32, 40}) {
              const int64_t len = at + d;
              if (len < 0 || len > Lk) continue;
              for (int form = 0; form < 3; ++form) {  // append, read with a ring, read without
                if (form == 0 && len + sq > Lk) continue;
                if (row(B, sq, H, Lk, (int)len, form == 0, form < 2)) continue;
                std::printf("B=%d H=%d Lk=%d sq=%d len=%d form=%d\n", (int)B, (int)H, (int)Lk, (int)sq, (int)len, form);
                return 1;
              }
            }
        }
  std::printf("%ld %ld %ld\n", calls, split_rows, behind);
  return 0;
}
"""


def test_every_block_is_taken_once(tmp_path):
    include = Path(os.environ.get("ROCM_PATH", "/opt/rocm")) / "include"
    if not shutil.which("g++") or not include.is_dir():
        pytest.skip("needs g++ and the HIP headers")
    (tmp_path / "cut.cpp").write_text(SOURCE)
    cmd = ["g++", "-std=c++17", "-O2", "-D__HIP_PLATFORM_AMD__", f"-I{include}", f"-I{CSRC}", "cut.cpp", "-o", "cut"]
    made = subprocess.run(cmd, cwd=tmp_path, capture_output=True, text=True)
    assert made.returncode == 0, made.stderr
    ran = subprocess.run(["./cut"], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout
    calls, split_rows, behind = map(int, ran.stdout.split())
    assert calls > 10000 and split_rows > 1000 and behind > 100  # the sizes reach what they are for
