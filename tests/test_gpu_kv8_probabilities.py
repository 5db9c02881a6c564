"""How many bits the probabilities of an 8-bit cache's attention count with, whatever a prompt's company: keys of
small weight are not dropped, and roundings that all point one way stay far below the result's own."""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as o8

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _np(t):
    return t.detach().double().cpu().numpy()


def _codes(cuda, dtype, L, kd0, vd0):
    """A cache of one slot and head whose keys and values are ``kd0`` and ``vd0`` along dimension 0 (e4m3 numbers)."""
    from whisperdrz_amd import FlashKVCache8

    c = FlashKVCache8(1, L, 1, 64, dtype=dtype, device=cuda, ring=False)
    for codes, scales, x in ((c.k_codes, c.k_scales, kd0), (c.v_codes, c.v_scales, vd0)):
        codes[0, 0, :L, 0] = x.to(codes.dtype)
        scales.fill_(1.0)
    return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,sq", [(1, 1), (1, 16), (1, 300), (5, 4096)])
def test_many_keys_of_small_weight(cuda, dtype, B, sq):
    """One key of weight 1 and 2^20 - 1 of 2^-25.5 each: together 2.2% of the sum."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    L = 1 << 20
    k = torch.full((L,), -16.0, device=cuda)
    v = torch.ones(L, device=cuda)
    k[0], v[0] = 0.0, 0.0
    c = _codes(cuda, dtype, L, k, v)
    q = torch.zeros(B, sq, 1, 64, dtype=dtype, device=cuda)
    q[..., 0] = 25.5 / 16
    idx = torch.zeros(B, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, cache_batch_idx=idx, softmax_scale=float(np.log(2.0)))
    torch.cuda.synchronize()
    tail = (L - 1) * 2.0 ** (-16.0 * float(q[0, 0, 0, 0]))
    want = tail / (1 + tail)
    # the result's rounding; 2^-16 for the parts of a probability; 2^-16 for the few roundings of a score of 25.5 and
    # of its exp2; above the line fp32 sums of at most 2^18 equal terms in order, 2^18 2^-24; below it the tail is
    # added to 1, whose fp32 steps are larger than a term: at worst all of it is lost there
    tol = (HALF[dtype] + 2.0 ** -16 + 2.0 ** -16 + 2.0 ** -6 + tail) * want
    got = _np(out)
    assert (np.abs(got[..., 0] - want) <= tol).all(), (got[..., 0].min(), got[..., 0].max(), want)
    assert not got[..., 1:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,sq,H", [(1, 64, 20), (20, 64, 20)])
def test_roundings_that_add_up(cuda, dtype, B, sq, H):
    """56 keys of weight 1 and value 1 beside 72 of weight w and value -1: the result is a small difference of
    large sums, where 2^-12 of w would show. w = exp(-0.125 q) lies near the middle between two fp16 numbers."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    cand = torch.arange(1.75, 2.25, 2.0 ** -6)  # exact in bf16 and fp16
    w = np.exp(-0.125 * cand.double().numpy())
    off = np.abs(w.astype(np.float16).astype(np.float64) - w) / w
    q0 = float(cand[int(off.argmax())])
    assert off.max() > 0.8 * 2.0 ** -12
    c = FlashKVCache8(B, 128, H, 64, dtype=dtype, device=cuda, ring=False)
    one = torch.arange(128, device=cuda) < 56
    c.k_codes[..., 0] = torch.where(one, 0.0, -1.0).to(c.k_codes.dtype)
    c.v_codes[:] = torch.where(one, 1.0, -1.0).to(c.v_codes.dtype)[:, None]
    c.k_scales.fill_(1.0)
    c.v_scales.fill_(1.0)
    q = torch.zeros(B, sq, H, 64, dtype=dtype, device=cuda)
    q[..., 0] = q0
    out = flash_attn_with_kvcache8(q, c)
    torch.cuda.synchronize()
    ref = o8.Cache(_np(c.k_codes[:1]), _np(c.v_codes[:1]), _np(c.k_scales[:1]), _np(c.v_scales[:1]))
    want, mag, big = o8.attend(_np(q[0, :1]), ref.read(0, 0, 128), ref.read(1, 0, 128), [128], 0.125)
    assert (np.abs(want) < 2.0 ** -5).all()
    over = np.abs(_np(out) - want[None]) - o8.bound(want, mag, big, 128, HALF[dtype])[None]
    assert over.max() <= 0, f"{over.max():.3e} over the bound"
