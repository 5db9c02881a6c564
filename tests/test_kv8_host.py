"""The 8-bit cache's and the 4-bit linears' host side: the oracle against torch's e4m3, the weights'
packing, and every refusal that needs no GPU."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import kv8_oracle as o8


def test_oracle_rounding_is_torchs_e4m3():
    x = np.arange(-448 * 512, 448 * 512 + 1) / 512.0
    want = torch.from_numpy(x).float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(o8.e4m3(x), want)


@pytest.mark.parametrize("top,e", [(0.0, -100), (448.0, 0), (449.0, 1), (896.0, 1), (1.0, -8), (1.75, -8), (1.7501, -7),
                                   (2.0 ** -126, -100), (3.3e38, 100)])
def test_oracle_block_scale(top, e):
    x = np.zeros((32, 64))
    x[3, 5], x[4, 6] = top, np.inf
    codes, scale = o8.quantize_block(x)
    assert scale == 2.0 ** e and np.isnan(codes[4, 6]) and np.nanmax(codes) <= 448


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (40, 192, 64), (33, 384, 128)])
def test_pack_round_trip(dtype, N, K, group):
    from whisperdrz_amd import QuantLinear4

    g = torch.Generator().manual_seed(N + K)
    codes = torch.randint(-7, 8, (N, K), generator=g)
    scales = (torch.rand(N, K // group, generator=g) + 0.01).to(dtype)
    lin = QuantLinear4.from_codes(codes, scales)
    want = codes.float() * scales.float().repeat_interleave(group, 1)
    assert torch.equal(lin.dequantize(), want)
    # the layout the header documents, byte by byte
    p = lin.packed.numpy()
    for n in range(N):
        for k in range(0, K, 7):
            c, r = divmod(k, 128)
            s, r = divmod(r, 32)
            gg, i = divmod(r, 8)
            byte = int(p[n // 16, c, 16 * (16 * gg + n % 16) + 4 * s + i % 4])
            nib = byte >> 4 if i >= 4 else byte & 15
            assert (-(nib & 7) if nib & 8 else nib) == int(codes[n, k])
    assert torch.equal(lin.scales[(N - 1) // 16, :, (N - 1) % 16], scales[N - 1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_from_weight_rounds_to_nearest(dtype):
    from whisperdrz_amd import QuantLinear4

    g = torch.Generator().manual_seed(3)
    w = (torch.randn(24, 192, generator=g) * 0.05).to(dtype)
    w[2, 64:128] = 0  # a group of zeros: scale 0, codes 0
    lin = QuantLinear4.from_weight(w, group=64)
    s = (w.float().view(24, 3, 64).abs().amax(-1) / 7).to(dtype).float()[..., None]
    # half a step, and what the scale's own rounding (half an ulp) takes from the 7 steps
    slack = 0.5 * s + 7 * s * torch.finfo(dtype).eps
    assert ((lin.dequantize().view(24, 3, 64) - w.float().view(24, 3, 64)).abs() <= slack).all()
    assert torch.equal(lin.dequantize()[2, 64:128], torch.zeros(64))


def test_from_codes_refusals():
    from whisperdrz_amd import QuantLinear4

    codes, scales = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8, 2, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="-7..7"):
        QuantLinear4.from_codes(codes - 8, scales)
    with pytest.raises(ValueError, match="-7..7"):
        QuantLinear4.from_codes(torch.full((8, 64), 255, dtype=torch.uint8), scales)
    with pytest.raises(TypeError, match="whole"):
        QuantLinear4.from_codes(codes.float(), scales)
    with pytest.raises(TypeError, match="16-bit"):
        QuantLinear4.from_codes(codes, scales.float())
    with pytest.raises(TypeError, match="bias"):
        QuantLinear4.from_codes(codes, scales, torch.zeros(7, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError, match="group 16"):
        QuantLinear4.from_codes(codes, torch.ones(8, 4, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="K / group"):
        QuantLinear4.from_codes(codes, torch.ones(8, 3, dtype=torch.bfloat16))
    with pytest.raises(NotImplementedError, match="divide"):
        QuantLinear4.from_weight(torch.zeros(8, 96, dtype=torch.bfloat16), group=64)
    with pytest.raises(TypeError):
        QuantLinear4.from_weight(torch.zeros(8, 64))


def test_cache_construction():
    from whisperdrz_amd import FlashKVCache8

    c = FlashKVCache8(3, 70, 2, 64, dtype=torch.float16)
    assert c.k_codes.shape == (3, 2, 96, 64) and c.k_codes.dtype == torch.float8_e4m3fn
    assert c.v_scales.shape == (3, 2, 3) and c.k_ring.shape == (3, 2, 64, 64) and c.seq_lens.tolist() == [0, 0, 0]
    x = FlashKVCache8(3, 70, 2, 64, ring=False)
    assert x.k_ring is None and not x.has_ring
    k, v = c.dequantize()
    assert k.shape == (3, 70, 2, 64) and not k.any() and not v.any()
    with pytest.raises(NotImplementedError, match="head_dim"):
        FlashKVCache8(3, 70, 2, 32)
    with pytest.raises(TypeError):
        FlashKVCache8(3, 70, 2, 64, dtype=torch.float32)
    with pytest.raises(ValueError, match="k_codes"):
        FlashKVCache8(3, 70, 2, 64, storage={})
    with pytest.raises(RuntimeError, match="is on cpu"):
        c.prefill(torch.zeros(1, 2, 2, 64, dtype=torch.float16), torch.zeros(1, 2, 2, 64, dtype=torch.float16))
    with pytest.raises(ValueError, match="without a ring"):
        c.set_cross_attention(torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 2, 64))
    with pytest.raises(ValueError, match="with a ring"):
        x.prefill(torch.zeros(1, 2, 2, 64), torch.zeros(1, 2, 2, 64))


def test_cpu_tensors_are_refused():
    from whisperdrz_amd import FlashKVCache8, QuantLinear4, flash_attn_with_kvcache8, linear4, linear4_partials

    c = FlashKVCache8(3, 70, 2, 64, ring=False)
    with pytest.raises(RuntimeError, match="is on cpu"):
        flash_attn_with_kvcache8(torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), c)
    with pytest.raises(TypeError, match="q must be a torch.Tensor"):
        flash_attn_with_kvcache8(None, c)
    lin = QuantLinear4.from_weight(torch.zeros(8, 64, dtype=torch.bfloat16))
    for f in (linear4, linear4_partials):
        with pytest.raises(RuntimeError, match="is on cpu"):
            f(torch.zeros(1, 64, dtype=torch.bfloat16), lin)


# ---- the C entries' own checks: all return before anything is launched ----

P = 0x10000  # a pointer that is never read


def _cache(lib_mod, **kw):
    f = dict(k_codes=P, v_codes=P, k_scales=P, v_scales=P, k_ring=P, v_ring=P, n_slots=4, n_heads=2, max_seq=100)
    f.update(kw)
    return lib_mod.Kv8(**f)


def _st(*s):
    return (ctypes.c_int64 * 4)(*s)


def _attn(cache="default", dtype=2, q=P, qs=(128, 128, 64, 1), k=P, ks=(128, 128, 64, 1), v=P, vs=(128, 128, 64, 1), lens=P,
          idx=P, o=P, os=(128, 128, 64, 1), B=2, sq=1, scale=0.125, ws=None, nbytes=0, **kw):
    from whisperdrz_amd import _lib

    lib = _lib.load()
    c = _cache(_lib, **kw) if cache == "default" else cache
    opt = lambda s: None if s is None else _st(*s)
    return lib.wdrz_attn_kvcache8(dtype, c, q, opt(qs), k, opt(ks), v, opt(vs), lens, idx, o, opt(os), B, sq, scale, ws,
                                  nbytes, None), lib.wdrz_last_error().decode()


@pytest.mark.parametrize("kw,code,word", [
    (dict(cache=None), 1, "cache is NULL"), (dict(dtype=0), 2, "dtype"), (dict(dtype=9), 1, "dtype"),
    (dict(n_slots=0), 1, "sizes"), (dict(n_heads=1 << 20), 2, "too large"), (dict(max_seq=1 << 25), 2, "too large"),
    (dict(k_codes=None), 1, "k_codes"), (dict(v_scales=P + 4), 1, "v_scales"), (dict(k_ring=None), 1, "together"),
    (dict(v_ring=P + 8), 1, "v_ring"), (dict(B=-1), 1, "sizes"), (dict(sq=0), 1, "sizes"), (dict(sq=5000), 2, "too large"),
    (dict(B=70000), 2, "too large"), (dict(scale=0.0), 1, "softmax_scale"), (dict(scale=float("nan")), 1, "softmax_scale"),
    (dict(scale=float("inf")), 1, "softmax_scale"), (dict(k=None), 1, "together"), (dict(lens=None), 1, "cache_seqlens"),
    (dict(k_ring=None, v_ring=None), 1, "ring"), (dict(k=None, v=None, lens=None), 1, "cache_seqlens"),
    (dict(sq=101), 1, "exceeds"), (dict(q=None), 1, "q is NULL"), (dict(q=P + 2), 1, "aligned"),
    (dict(qs=(128, 128, 64, 2)), 1, "stride"), (dict(ks=(128, 4, 64, 1)), 1, "aligned"), (dict(vs=None), 1, "NULL"),
    (dict(os=(3, 128, 64, 1)), 1, "aligned"), (dict(o=None), 1, "out is NULL"),
    (dict(k=None, v=None, k_ring=None, v_ring=None, max_seq=3000, B=1), 4, "workspace"),
    (dict(k=None, v=None, k_ring=None, v_ring=None, max_seq=3000, B=1, ws=P + 16, nbytes=1 << 20), 1, "256-byte"),
])
def test_attention_refusals(kw, code, word):
    rc, msg = _attn(**kw)
    assert rc == code and word in msg, (rc, msg)


def test_attention_of_no_rows():
    assert _attn(B=0, q=None, o=None)[0] == 0


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=0), 2, "dtype"), (dict(B=-1), 1, "sizes"), (dict(start=-1), 1, "sizes"), (dict(B=70000), 2, "too large"),
    (dict(T=98), 1, "exceed"), (dict(T=101), 1, "exceed"), (dict(start=1 << 62), 1, "exceed"),
    (dict(k_ring=None, v_ring=None), 1, "multiples of 32"), (dict(slots=None, B=5), 1, "slots"), (dict(k=None), 1, "k is NULL"),
    (dict(v=P + 8), 1, "aligned"), (dict(st=(128, 100, 64, 1)), 1, "aligned"), (dict(st=(128, 128, 64, 2)), 1, "stride"),
])
def test_write_refusals(kw, code, word):
    from whisperdrz_amd import _lib

    a = dict(dtype=2, k=P, v=P, st=(128, 128, 64, 1), slots=P, B=2, T=5, start=3)
    a.update({n: x for n, x in kw.items() if n in a})
    lib = _lib.load()
    rc = lib.wdrz_kv8_write(a["dtype"], _cache(_lib, **{n: x for n, x in kw.items() if n not in a}), a["k"], _st(*a["st"]),
                            a["v"], _st(*a["st"]), a["slots"], a["B"], a["T"], a["start"], None)
    assert rc == code and word in lib.wdrz_last_error().decode(), lib.wdrz_last_error()


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=0), 2, "dtype"), (dict(M=-1), 1, "sizes"), (dict(N=0), 1, "sizes"), (dict(group=16), 2, "group"),
    (dict(K=96, group=64), 2, "multiple"), (dict(M=1 << 23), 2, "too large"), (dict(x=None), 1, "x is NULL"),
    (dict(w=P + 8), 1, "w_packed"), (dict(s=None), 1, "scales"), (dict(xs=32), 1, "shorter"), (dict(xs=68), 1, "aligned"),
    (dict(y=None), 1, "y is NULL"), (dict(bias=P + 1), 1, "2-byte"), (dict(ys=7), 1, "shorter"), (dict(act=2), 1, "activation"),
])
def test_linear_refusals(kw, code, word):
    from whisperdrz_amd import _lib

    a = dict(dtype=2, x=P, xs=64, w=P, s=P, bias=None, y=P, ys=8, M=2, N=8, K=64, group=32, act=0)
    a.update(kw)
    lib = _lib.load()
    rc = lib.wdrz_linear4(*a.values(), None)
    assert rc == code and word in lib.wdrz_last_error().decode(), lib.wdrz_last_error()
    if "y" in word or "act" in word or "bias" in str(kw) or "ys" in kw:
        return
    del a["bias"], a["ys"], a["act"]
    rc = lib.wdrz_linear4_partials(*a.values(), 2, None)
    assert rc == code, lib.wdrz_last_error()


def test_partials_refuse_other_splits():
    from whisperdrz_amd import _lib

    lib = _lib.load()
    assert lib.wdrz_linear4_partials(2, P, 64, P, P, P, 2, 8, 64, 32, 3, None) == 2
    assert lib.wdrz_linear4_partials(2, None, 64, None, None, None, 0, 8, 64, 32, 2, None) == 0


def test_pool_of_8_bit_caches():
    from whisperdrz_amd.kv_cache import FlashKVCache8, KVSlotPool, cache_bytes_per_slot, plan_slots

    pool = KVSlotPool(2, 5, 2, 64, self_len=40, cross_len=33, dtype=torch.float16, cache_bits=8)
    ptrs = []
    for s, x in zip(pool.self_kv, pool.cross_kv):
        assert isinstance(s, FlashKVCache8) and s.has_ring and not x.has_ring and s.dtype == torch.float16
        assert s.k_codes.shape == (5, 2, 64, 64) and x.v_codes.shape == (5, 2, 64, 64) and s.max_seq_length == 40
        ptrs += [t.data_ptr() for t in (s.k_codes, s.v_codes, s.k_scales, s.v_scales, s.k_ring, s.v_ring, x.k_codes, x.v_scales)]
    base = pool.arena.data_ptr()
    assert len(set(ptrs)) == len(ptrs) and all(base <= p < base + pool.arena.numel() and (p - base) % (2 << 20) == 0 for p in ptrs)
    assert pool.self_kv[1].seq_lens.data_ptr() == pool.self_seq_lens[1].data_ptr()
    per = cache_bytes_per_slot(32, 20, 64, 448, 1500, torch.bfloat16, 8)
    assert per == 32 * 20 * (2 * (448 * 64 + 14 * 4 + 64 * 128) + 2 * (1504 * 64 + 47 * 4))
    plan = plan_slots(272 * 10**9, cache_bits=8)
    assert plan.bytes_per_slot == per and plan.total_bytes <= 272 * 10**9
    assert KVSlotPool.arena_bytes(plan.n_slots + 1, 32, 20, 64, 448, 1500, torch.bfloat16, 8) > 272 * 10**9
    with pytest.raises(ValueError, match="cache_bits"):
        KVSlotPool(1, 1, 1, 64, self_len=8, cross_len=8, cache_bits=4)
