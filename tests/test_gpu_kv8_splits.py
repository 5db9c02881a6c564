"""Appends to an 8-bit cache whose keys are split over workgroups, with new rows on both sides of a split's
border: every key counts once. Held to oracle/kv8_oracle.bound, as the other tests of the cache's attention.
"""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as o8

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SCALE = 0.125


def _np(t):
    return t.detach().double().cpu().numpy()


def _append(cuda, dtype, B, sq, H, L, lens, seed):
    """Rows of ``lens`` written positions append ``sq`` more: outputs and the cache's codes against the oracle's."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    g = torch.Generator(device=cuda).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=g, device=cuda).to(dtype)
    c = FlashKVCache8(B, L, H, 64, dtype=dtype, device=cuda)
    top = max(max(lens), 1)
    old_k, old_v = randn(B, top, H, 64), randn(B, top, H, 64)
    for b, n in enumerate(lens):
        if n:
            c.prefill(old_k[b:b + 1, :n], old_v[b:b + 1, :n], 0, torch.tensor([b], device=cuda))
    shape = (B, H, -(-L // 32))
    zeros, ring = np.zeros(shape[:2] + (shape[2] * 32, 64)), np.zeros((B, H, 64, 64))
    ref = o8.Cache(zeros, zeros, np.ones(shape), np.ones(shape), ring, ring, max_seq=L)
    for b, n in enumerate(lens):
        if n:
            ref.append(b, 0, _np(old_k[b, :n]), _np(old_v[b, :n]))
    q, k, v = (randn(B, sq, H, 64) for _ in range(3))
    at = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=at)
    torch.cuda.synchronize()
    for b, n in enumerate(lens):
        kk = np.concatenate([ref.read(0, b, n), _np(k[b]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, b, n), _np(v[b]).transpose(1, 0, 2)], 1)
        want, mag, big = o8.attend(_np(q[b]), kk, vv, [n + t + 1 for t in range(sq)], SCALE)
        over = np.abs(_np(out[b]) - want) - o8.bound(want, mag, big, n + sq, HALF[dtype])
        assert over.max() <= 0, f"row {b} of {n}: {over.max():.3e} over the bound"
        ref.append(b, n, _np(k[b]), _np(v[b]))
        done = (n + sq) // 32 * 32
        assert np.array_equal(_np(c.k_codes[b, :, :done]), ref.codes[0][b, :, :done])
        assert np.array_equal(_np(c.v_codes[b, :, :done]), ref.codes[1][b, :, :done])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length", [480, 507, 508, 510, 511, 512, 513])
@pytest.mark.parametrize("sq", [2, 5, 32])
def test_drafts_over_a_border(cuda, dtype, length, sq):
    """2048 positions of 4 heads are split every 512: lengths just below, at and above the first border."""
    _append(cuda, dtype, 1, sq, 4, 2048, [length], length + sq)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,sq,H,L,lens", [
    (3, 9, 4, 2048, [509, 1023, 1535]),  # every border of three rows
    (1, 64, 20, 2048, [690]),  # four blocks of queries, the append in a launch of its own
    (2, 33, 2, 4096, [511, 2047]),
    (1, 1100, 1, 2048, [0]),  # a prompt longer than a split: whole splits of new rows
    (1, 700, 2, 2300, [31]),
])
def test_prompts_over_borders(cuda, dtype, B, sq, H, L, lens):
    _append(cuda, dtype, B, sq, H, L, lens, sq)
