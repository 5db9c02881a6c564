"""Attention over pages where rows are cut: every rule of the plan, with several tiles of rows, short rows in long tables, and the
most parts that there are; the arrival counters are back at zero after each call."""
import random

import pytest
import torch

import whisperdrz_amd as w
from test_gpu_pages import run_case
from whisperdrz_amd.attention import _COUNTED_WORKSPACES

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def check(cuda, seed, dtype, lens, sq, H, Hk, dim, page, append, max_len, parts):
    rows = min(16, sq * H // Hk)
    units = len(lens) * Hk * -(-sq * H // Hk // 16)
    # the workspace says how many parts a row has at most
    assert w.kvpages_workspace_size(len(lens), sq, H, Hk, dim, max_len) == 4096 * 4 + units * parts * rows * (dim + 2) * 4
    run_case(cuda, seed, dtype, lens, sq, H, Hk, dim, page, append, max_len)
    torch.cuda.synchronize()
    assert _COUNTED_WORKSPACES and not any(b[: 4096 * 4].any() for b in _COUNTED_WORKSPACES.values())


def mostly_short(n, long, seed):
    rng = random.Random(seed)
    lens = [rng.randint(0, 40) for _ in range(n - len(long))] + list(long)
    rng.shuffle(lens)
    return lens


@pytest.mark.parametrize("dtype,append", [(BF16, True), (FP16, False)])
@pytest.mark.parametrize("dim", [64, 128])
def test_more_units_than_cus(cuda, dtype, append, dim):
    """Parts of 4096 keys: in four wavefronts a workgroup, and in two."""
    check(cuda, 1, dtype, mostly_short(130, [8190, 4096, 4097, 5000], 1), 1, 2, 2, dim, 64, append, 8192, 2)
    check(cuda, 2, dtype, mostly_short(200, [16380, 12289, 4095], 2), 1, 4, 2, dim, 256, append, 16384, 4)


def test_the_most_parts(cuda):
    """64 parts of a row of 300000 positions beside short ones."""
    check(cuda, 3, BF16, mostly_short(256, [299999, 100000], 3), 1, 2, 1, 64, 256, True, 300000, 64)


@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
def test_several_tiles_of_rows(cuda, append, dim):
    """36 and 40 rows a key/value head: tiles whose causal limits differ share no part."""
    check(cuda, 4, BF16, [1990, 0, 700], 9, 8, 2, dim, 16, append, 2000, 8)
    check(cuda, 5, FP16, [1500, 511], 40, 2, 2, dim, 32, append, 1600, 7)


def test_several_tiles_of_many_rows(cuda):
    check(cuda, 6, FP16, mostly_short(24, [8183, 4090], 6), 9, 16, 4, 64, 64, True, 8192, 2)


def test_calls_of_other_shapes_share_a_workspace(cuda):
    for i in range(3):
        check(cuda, 7 + i, BF16, [1200, 3, 900], 1, 2, 2, 64, 16, True, 1300, 6)
        check(cuda, 17 + i, BF16, [40000], 2, 8, 2, 128, 64, False, 40000, 32)
        check(cuda, 27 + i, FP16, mostly_short(130, [8000], i), 1, 2, 2, 64, 64, True, 8192, 2)
