"""Reads of an 8-bit cache over blocks that nobody has written (codes and scales 0): their keys and values are zeros,
and places behind the length do not count, with one query, with drafts and with many prompts alike."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as o8

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,sq,H", [(3, 1, 4), (3, 5, 4), (3, 20, 4), (17, 64, 16)])
@pytest.mark.parametrize("T,L", [(1450, 1500), (1472, 1500), (5, 33), (40, 100), (33, 130)])
def test_window_shorter_than_the_cache(cuda, dtype, B, sq, H, T, L):
    """A cross cache filled with T of L positions and attended without lengths; the last slot is never filled."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    g = torch.Generator(device=cuda).manual_seed(T + sq)
    c = FlashKVCache8(B, L, H, 64, dtype=dtype, device=cuda, ring=False)
    k, v = (torch.randn(B - 1, T, H, 64, generator=g, device=cuda).to(dtype) for _ in range(2))
    c.set_cross_attention(k, v, torch.arange(B - 1, device=cuda))
    q = torch.randn(B, sq, H, 64, generator=g, device=cuda).to(dtype)
    out = flash_attn_with_kvcache8(q, c)
    torch.cuda.synchronize()
    ref = o8.Cache(_np(c.k_codes), _np(c.v_codes), _np(c.k_scales), _np(c.v_scales), max_seq=L)
    assert torch.isfinite(out).all() and not out[B - 1].any()
    for b in (0, B - 2):
        want, mag, big = o8.attend(_np(q[b]), ref.read(0, b, L), ref.read(1, b, L), [L] * sq, 0.125)
        over = np.abs(_np(out[b]) - want) - o8.bound(want, mag, big, L, HALF[dtype])
        assert over.max() <= 0, f"row {b}: {over.max():.3e} over the bound"


@pytest.mark.parametrize("B,sq,H", [(2, 1, 4), (2, 5, 4), (17, 64, 16)])
def test_scores_scaled_to_nothing(cuda, B, sq, H):
    """A softmax scale that, times a block of zeros' 2^-100, is under every fp32 number: all places alike."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    c = FlashKVCache8(B, 70, H, 64, dtype=torch.bfloat16, device=cuda, ring=False)
    v = torch.ones(B, 70, H, 64, dtype=torch.bfloat16, device=cuda)
    c.set_cross_attention(torch.zeros_like(v), v)
    out = flash_attn_with_kvcache8(v[:, :1].expand(B, sq, H, 64).contiguous(), c, softmax_scale=1e-20)
    assert torch.equal(out, torch.ones_like(out))
