"""GPU parity of the 8-bit slot cache (FlashKVCache8, flash_attn_with_kvcache8) with oracle/kv8_oracle.py.

State is compared exactly: code values, scales, ring bits, and every byte outside the written rows. Outputs are
held to oracle/kv8_oracle.bound, which is derived from the arithmetic: the result's own rounding, half a
step (bf16 2^-8, fp16 2^-11), plus fp32 and two-part-probability terms in units of sum p |v|.
"""
import numpy as np
import pytest
import torch

from oracle import kv8_oracle as o8

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]
SCALE = 0.125


def _gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def _randn(g, *shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dtype)


def _cache(cuda, dtype, S, L, H, ring, seed, std=100.0):
    """A cache with random contents in every buffer, stale rows too."""
    from whisperdrz_amd import FlashKVCache8

    g = _gen(cuda, seed)
    st = {}
    for n, (shape, dt) in FlashKVCache8.layout(S, L, H, dtype, ring).items():
        if dt is torch.float8_e4m3fn:
            st[n] = (torch.randn(shape, generator=g, device=cuda) * std).clamp(-448, 448).to(dt)
        elif n.endswith("scales"):
            st[n] = ((torch.randint(-9, -5, shape, generator=g, device=cuda).int() + 127) << 23).view(torch.float32)
        else:
            st[n] = _randn(g, *shape, dtype=dtype)
    return FlashKVCache8(S, L, H, 64, dtype=dtype, ring=ring, storage=st)


BUFFERS = ("k_codes", "v_codes", "k_scales", "v_scales", "k_ring", "v_ring")


def _np(t):
    return t.detach().double().cpu().numpy()


def _oracle(c):
    ring = (_np(c.k_ring), _np(c.v_ring)) if c.has_ring else ()
    return o8.Cache(_np(c.k_codes), _np(c.v_codes), _np(c.k_scales), _np(c.v_scales), *ring, max_seq=c.max_seq_length)


def _bits(c):
    return [getattr(c, n).view(torch.uint8).clone() if getattr(c, n) is not None else None for n in BUFFERS]


def _same_state(c, ref):
    pairs = [(c.k_codes, ref.codes[0]), (c.v_codes, ref.codes[1]), (c.k_scales, ref.scales[0]), (c.v_scales, ref.scales[1])]
    if c.has_ring:
        pairs += [(c.k_ring, ref.ring[0]), (c.v_ring, ref.ring[1])]
    for (got, want), name in zip(pairs, BUFFERS):
        assert np.array_equal(_np(got), want, equal_nan=True), name


def _one_part(dtype, B, sq, H):
    """Whether a call's codes meet probabilities of one fp16 value: many bf16 prompts, in blocks of 64 queries."""
    return dtype is torch.bfloat16 and sq > 32 and B * -(-sq // 16) * H > 1024


def _check(out, want, mag, big, n_keys, dtype, what="", one_part=False):
    got = _np(out)
    err = np.abs(got - want) - o8.bound(want, mag, big, n_keys, HALF[dtype], one_part)
    assert np.isfinite(got).all() and err.max() <= 0, f"{what}: {err.max():.3e} over the bound"


def _rows(q, ref, slots, limits, dtype, out, what=""):
    for b, slot in enumerate(slots):
        n = int(max(limits[b]))
        want, mag, big = o8.attend(_np(q[b]), ref.read(0, slot, n), ref.read(1, slot, n), limits[b], SCALE)
        _check(out[b], want, mag, big, n, dtype, f"{what} row {b}")


# ---- writes -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,L", [(1, 1), (31, 40), (32, 32), (33, 64), (100, 100), (65, 1500)])
def test_cross_fill(cuda, dtype, T, L):
    c = _cache(cuda, dtype, 5, L, 3, False, 1)
    ref, before = _oracle(c), _bits(c)
    g = _gen(cuda, T)
    kv = _randn(g, 3, T, 6, 64, dtype=dtype) * torch.exp2(torch.randint(-12, 5, (3, T, 6, 1), generator=g, device=cuda)).to(dtype)
    k, v = kv[:, :, :3], kv[:, :, 3:]  # the halves of one projection
    slots = torch.tensor([4, 0, 2], device=cuda)
    c.set_cross_attention(k, v, slots)
    torch.cuda.synchronize()
    for b, s in enumerate([4, 0, 2]):
        ref.fill(s, _np(k[b]), _np(v[b]))
    _same_state(c, ref)
    after = _bits(c)
    n = -(-T // 32) * 32
    assert torch.equal(before[0][:, :, n:], after[0][:, :, n:]) and torch.equal(before[1][[1, 3]], after[1][[1, 3]])
    assert c.cross_attn_len == T and c.done


@pytest.mark.parametrize("dtype", TYPES)
def test_fill_special_values(cuda, dtype):
    """Zeros, values that are not finite, the type's largest and smallest ones, ties between codes."""
    c = _cache(cuda, dtype, 2, 160, 1, False, 2)
    ref = _oracle(c)
    x = torch.zeros(1, 160, 1, 64, device=cuda, dtype=dtype)
    fi = torch.finfo(dtype)
    x[0, 1, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 1.0], device=cuda)  # block 0
    x[0, 33, 0, :3] = torch.tensor([fi.max, fi.min, fi.smallest_normal], device=cuda).to(dtype)  # block 1
    x[0, 65, 0, :2] = torch.tensor([fi.smallest_normal, fi.smallest_normal / 4], device=cuda).to(dtype)  # block 2
    x[0, 96:128, 0] = (torch.arange(2048, device=cuda).view(32, 64).float() / 2048 * 448).to(dtype)  # block 3: ties
    k, v = x, -x.flip(1)
    c.set_cross_attention(k, v)
    torch.cuda.synchronize()
    ref.fill(0, _np(k[0]), _np(v[0]))
    _same_state(c, ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start,T", [(0, 1), (0, 31), (0, 32), (0, 33), (0, 64), (0, 100), (5, 3), (31, 1), (31, 2), (32, 1),
                                     (10, 22), (10, 86), (10, 150), (40, 90), (63, 33), (64, 96), (95, 65), (159, 1)])
def test_prefill_state(cuda, dtype, start, T):
    c = _cache(cuda, dtype, 4, 160, 2, True, 3)
    ref, before = _oracle(c), _bits(c)
    g = _gen(cuda, start * 7 + T)
    k, v = _randn(g, 2, T, 2, 64, dtype=dtype), _randn(g, 2, T, 2, 64, dtype=dtype, std=30.0)
    c.prefill(k, v, start, torch.tensor([3, 1], device=cuda))
    torch.cuda.synchronize()
    for b, s in enumerate([3, 1]):
        ref.append(s, start, _np(k[b]), _np(v[b]))
    _same_state(c, ref)
    for x, y in zip(before, _bits(c)):
        assert torch.equal(x[[0, 2]], y[[0, 2]])
    assert c.seq_lens.tolist() == [0, start + T, 0, start + T]


def test_write_skips_bad_slots_and_takes_the_last_of_equal_ones(cuda):
    dtype = torch.bfloat16
    c = _cache(cuda, dtype, 3, 100, 2, False, 4)
    ref = _oracle(c)
    g = _gen(cuda, 5)
    k, v = _randn(g, 6, 70, 2, 64, dtype=dtype), _randn(g, 6, 70, 2, 64, dtype=dtype)
    c.set_cross_attention(k, v, torch.tensor([1, 3, -1, 0, 1, 1 << 40], device=cuda))
    torch.cuda.synchronize()
    ref.fill(0, _np(k[3]), _np(v[3]))
    ref.fill(1, _np(k[4]), _np(v[4]))
    _same_state(c, ref)


# ---- reads --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 2, 5, 8, 9, 16, 17, 40, 130])
@pytest.mark.parametrize("L", [1, 31, 32, 33, 100, 129])
def test_cross_attention(cuda, dtype, sq, L):
    c = _cache(cuda, dtype, 5, L, 3, False, L)
    g = _gen(cuda, sq)
    q = _randn(g, 4, sq, 3, 64, dtype=dtype, std=2.0)
    slots = [2, 0, 4, 2]
    lens = [L, 0, (L + 1) // 2, max(1, L - 1)]
    from whisperdrz_amd import flash_attn_with_kvcache8

    before = _bits(c)
    idx = torch.tensor(slots, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda), cache_batch_idx=idx)
    whole = flash_attn_with_kvcache8(q, c, cache_batch_idx=idx)
    torch.cuda.synchronize()
    ref = _oracle(c)
    _rows(q, ref, slots, [[n] * sq for n in lens], dtype, out, "lens")
    _rows(q, ref, slots, [[L] * sq] * 4, dtype, whole, "whole")
    assert not out[1].any()  # a row of no positions
    for x, y in zip(before, _bits(c)):
        assert x is None or torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,sq,H,L", [(1, 1, 20, 1500), (3, 1, 4, 1500), (1, 5, 20, 1500), (2, 12, 3, 1499), (1, 1, 2, 6000),
                                      (7, 1, 20, 1500), (1, 224, 2, 1500), (1, 33, 1, 20000), (3, 1, 20, 3001),
                                      (2, 5, 4, 6000), (1, 1, 1, 40000)])
def test_long_cross_attention(cuda, dtype, B, sq, H, L):
    """Rows whose keys are split over workgroups, ragged so that some splits have nothing; called twice."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, B, L, H, False, B + sq)
    g = _gen(cuda, 3)
    q = _randn(g, B, sq, H, 64, dtype=dtype, std=2.0)
    lens = [max(1, L - 700 * b) for b in range(B)]
    t = torch.tensor(lens, dtype=torch.int32, device=cuda)
    a, b2 = (flash_attn_with_kvcache8(q, c, cache_seqlens=t) for _ in range(2))
    torch.cuda.synchronize()
    assert torch.equal(a, b2)
    _rows(q, _oracle(c), list(range(B)), [[n] * sq for n in lens], dtype, a)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 5])
def test_read_only_call_on_a_cache_with_a_ring(cuda, dtype, sq):
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, 8, 130, 2, True, 6)
    lens = [0, 1, 31, 32, 33, 64, 100, 130]
    g = _gen(cuda, 1)
    q = _randn(g, 8, sq, 2, 64, dtype=dtype)
    out = flash_attn_with_kvcache8(q, c, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    _rows(q, _oracle(c), list(range(8)), [[n] * sq for n in lens], dtype, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,sq,H,L,ring", [(20, 40, 20, 70, False), (20, 64, 20, 96, False), (20, 65, 20, 33, True),
                                           (20, 130, 10, 130, True), (26, 33, 20, 1, False)])
def test_many_prompts(cuda, dtype, B, sq, H, L, ring):
    """More than 1024 blocks of 16 queries: blocks of 64. Lengths from none to all."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, B, L, H, ring, 31)
    q = _randn(_gen(cuda, 3), B, sq, H, 64, dtype=dtype, std=2.0)
    lens = [L - (L * b) // (B - 1) for b in range(B)]
    lens[1], bad = -1, [1]
    out = flash_attn_with_kvcache8(q, c, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    ref = _oracle(c)
    assert torch.isnan(out[1]).all() and not out[B - 1].any()
    for b in (0, 2, 5, B // 2, B - 2):
        want, mag, big = o8.attend(_np(q[b]), ref.read(0, b, lens[b]), ref.read(1, b, lens[b]), [lens[b]] * sq, SCALE)
        _check(out[b], want, mag, big, lens[b], dtype, f"row {b}", _one_part(dtype, B, sq, H))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,sq,H,L", [(18, 40, 20, 200), (18, 65, 20, 200), (30, 33, 20, 140), (9, 130, 13, 200)])
def test_many_prompts_append(cuda, dtype, B, sq, H, L):
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, B, L, H, True, 41)
    ref = _oracle(c)
    g = _gen(cuda, 13)
    q, k, v = (_randn(g, B, sq, H, 64, dtype=dtype) for _ in range(3))
    k[0, sq - 1, 0, 3] = float("nan")  # seen by the last query alone
    v[0, sq - 2, 1, 5] = float("inf")  # ... by the last two
    v[1, 0, 2, 7] = -float("inf")  # by all
    lens = [(17 * b) % (L - sq + 1) for b in range(B)]
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    got = _np(out)
    assert np.isnan(got[0, -1, 0]).all() and np.isfinite(got[0, :-1, 0]).all()
    assert np.isposinf(got[0, -2:, 1, 5]).all() and np.isfinite(got[0, :-2, 1]).all() and np.isfinite(got[0, :, 1, :5]).all()
    assert np.isneginf(got[1, :, 2, 7]).all() and np.isfinite(got[1, :, 2, 8:]).all()
    for b in (2, 3, B // 2, B - 1):
        kk = np.concatenate([ref.read(0, b, lens[b]), _np(k[b]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, b, lens[b]), _np(v[b]).transpose(1, 0, 2)], 1)
        want, mag, big = o8.attend(_np(q[b]), kk, vv, [lens[b] + t + 1 for t in range(sq)], SCALE)
        _check(out[b], want, mag, big, lens[b] + sq, dtype, f"row {b}", _one_part(dtype, B, sq, H))
    for b in range(B):
        ref.append(b, lens[b], _np(k[b]), _np(v[b]))
    _same_state(c, ref)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [64, 70, 130])
def test_many_prompts_append_to_named_slots(cuda, dtype, sq):
    """Lengths at and off multiples of 32 (ring rows written with the attention and behind it), a slot named
    twice, rows that disagree, and rows out of range, in one call of blocks of 64 queries."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    B, H, L = 18, 20, 288
    c = _cache(cuda, dtype, 30, L, H, True, sq)
    ref = _oracle(c)
    g = _gen(cuda, 15)
    q, k, v = (_randn(g, B, sq, H, 64, dtype=dtype) for _ in range(3))
    lens = [0, 32, 64, 96, 1, 31, 33, 63, 95, 128, L - sq, 64, 7, 40, 41, 0, L - sq + 1, -1]
    slots = [29, 3, 7, 12, 1, 0, 5, 20, 21, 22, 23, 7, 24, 9, 9, 30, 25, 26]  # 7 twice alike, 9 disagrees
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=i32(lens), cache_batch_idx=i32(slots))
    torch.cuda.synchronize()
    assert torch.isnan(out[13:]).all()
    for b in (0, 1, 2, 6, 10, 11, 12):
        src = 11 if slots[b] == 7 else b
        kk = np.concatenate([ref.read(0, slots[b], lens[b]), _np(k[src]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, slots[b], lens[b]), _np(v[src]).transpose(1, 0, 2)], 1)
        want, mag, big = o8.attend(_np(q[b]), kk, vv, [lens[b] + t + 1 for t in range(sq)], SCALE)
        _check(out[b], want, mag, big, lens[b] + sq, dtype, f"row {b}", _one_part(dtype, B, sq, H))
    for b in range(13):
        if b != 2:
            ref.append(slots[b], lens[b], _np(k[b]), _np(v[b]))
    _same_state(c, ref)


def test_graph_of_many_prompts_that_append(cuda):
    """Both launches of the append, replayed over changing lengths and rows: as the eager calls on a copy."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    dtype, B, sq, H, L = torch.bfloat16, 18, 70, 20, 288
    c, e = (_cache(cuda, dtype, B, L, H, True, 3) for _ in range(2))
    g = _gen(cuda, 16)
    q, k, v = (_randn(g, B, sq, H, 64, dtype=dtype) for _ in range(3))
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=lens)
    flash_attn_with_kvcache8(q, e, k, v, cache_seqlens=lens)  # the call before the capture
    for step in range(4):
        lens.copy_(torch.arange(B, device=cuda) * (32 if step % 2 else 13) % (L - sq + 1))
        k.normal_(generator=g)
        v.normal_(generator=g)
        graph.replay()
        want = flash_attn_with_kvcache8(q, e, k, v, cache_seqlens=lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for x, y in zip(_bits(c), _bits(e)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 5, 64])
@pytest.mark.parametrize("span", [4, 14, 40, 90])
def test_scales_of_any_size(cuda, dtype, sq, span):
    """Values' scales 2^span apart, the attention on one block at a time: a small block's result is not
    rounded in a large one's units. K of each block points along one axis that a query picks."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    B, H, blocks = 17, 16, 9
    c = _cache(cuda, dtype, B, blocks * 32, H, False, 51)
    g = _gen(cuda, 5)
    e = torch.randint(-span // 2, span // 2 + 1, c.v_scales.shape, generator=g, device=cuda)
    e[0, :, :] = torch.linspace(-span / 2, span / 2, blocks, device=cuda).round().int()
    e[1] = e[0].flip(-1)
    c.v_scales.copy_(((e.int() + 127) << 23).view(torch.float32))
    kc = torch.zeros(B, H, blocks, 32, 64, device=cuda)
    for j in range(blocks):
        kc[:, :, j, :, j] = 64.0
    c.k_codes.copy_(kc.view(B, H, -1, 64).to(torch.float8_e4m3fn))
    c.k_scales.fill_(1.0)
    pick = torch.randint(0, blocks, (B, sq, H), generator=g, device=cuda)
    q = torch.nn.functional.one_hot(pick, 64).to(dtype) * 40.0  # scores 320 against 0: other blocks weigh e^-320
    out = flash_attn_with_kvcache8(q, c)
    torch.cuda.synchronize()
    ref = _oracle(c)
    rows = range(B) if sq < 64 else (0, 1, 7)
    for b in rows:
        want, mag, big = o8.attend(_np(q[b]), ref.read(0, b, blocks * 32), ref.read(1, b, blocks * 32), [blocks * 32] * sq, SCALE)
        top = 60000.0 if dtype is torch.float16 else 3e38
        keep = np.abs(want) < top  # what the output's type holds
        lim = o8.bound(want, mag, big, 288, HALF[dtype], _one_part(dtype, B, sq, H))
        if dtype is torch.bfloat16:
            lim = lim - 2.0 ** -25 + 1e-30  # the last term is fp16's smallest step: bf16 rounds small results too
        assert (np.abs(_np(out[b]) - want) <= lim)[keep].all(), b


# ---- append -------------------------------------------------------------------------------------


def _append_ref(ref, q, k, v, slots, lens, dtype, out):
    """Outputs over the state before the append with the new rows as they are, then the append."""
    sq = q.shape[1]
    for b, (slot, n) in enumerate(zip(slots, lens)):
        kk = np.concatenate([ref.read(0, slot, n), _np(k[b]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, slot, n), _np(v[b]).transpose(1, 0, 2)], 1)
        want, mag, big = o8.attend(_np(q[b]), kk, vv, [n + t + 1 for t in range(sq)], SCALE)
        _check(out[b], want, mag, big, n + sq, dtype, f"row {b} length {n}")
    for b, (slot, n) in enumerate(zip(slots, lens)):
        ref.append(slot, n, _np(k[b]), _np(v[b]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sq", [1, 2, 5, 8, 9, 16, 31, 32, 33, 40, 70, 130])
def test_append(cuda, dtype, sq):
    from whisperdrz_amd import flash_attn_with_kvcache8

    L, H = 200, 3
    lens = [n for n in (0, 1, 27, 30, 31, 32, 33, 63, 64, 70, 95, 130, 199) if n + sq <= L] + [L - sq]
    B = len(lens)
    c = _cache(cuda, dtype, B + 1, L, H, True, sq)
    ref, before = _oracle(c), _bits(c)
    g = _gen(cuda, 11)
    qkv = _randn(g, B, sq, 3, H, 64, dtype=dtype, std=1.5)  # one projection's output
    q, k, v = qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]
    slots = list(range(B, 0, -1))
    t = torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=t, cache_batch_idx=torch.tensor(slots, device=cuda))
    torch.cuda.synchronize()
    _append_ref(ref, q, k, v, slots, lens, dtype, out)
    _same_state(c, ref)
    assert torch.equal(before[0][0], _bits(c)[0][0]) and t.tolist() == lens


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,sq,H,L,filled", [(1, 1, 20, 1500, 1300), (2, 5, 3, 3000, 2991), (1, 20, 4, 900, 850), (1, 1, 2, 4000, 3999),
                                             (2, 30, 1, 2100, 2065)])
def test_append_behind_long_histories(cuda, dtype, B, sq, H, L, filled):
    """Split rows that append."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, B, L, H, True, 5)
    ref = _oracle(c)
    g = _gen(cuda, 12)
    q, k, v = (_randn(g, B, sq, H, 64, dtype=dtype) for _ in range(3))
    lens = [filled - 33 * b for b in range(B)]
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    _append_ref(ref, q, k, v, list(range(B)), lens, dtype, out)
    _same_state(c, ref)


@pytest.mark.parametrize("dtype", TYPES)
def test_state_does_not_depend_on_how_tokens_are_cut(cuda, dtype):
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    g = _gen(cuda, 4)
    k, v, q = (_randn(g, 2, 150, 2, 64, dtype=dtype) for _ in range(3))
    states = []
    for cuts in ([150], [1] * 150, [5] * 30, [33, 31, 64, 22], [32, 100, 18]):
        c = FlashKVCache8(2, 160, 2, 64, dtype=dtype, device=cuda)
        at = 0
        for n in cuts:
            s = slice(at, at + n)
            flash_attn_with_kvcache8(q[:, s], c, k[:, s], v[:, s], cache_seqlens=c.seq_lens)
            c.seq_lens += n
            at += n
        p = FlashKVCache8(2, 160, 2, 64, dtype=dtype, device=cuda)
        p.prefill(k, v)
        states.append((_bits(c), _bits(p)))
    torch.cuda.synchronize()
    for c, p in states:
        for x, y in zip(c[:4], states[0][0][:4]):
            assert torch.equal(x, y)
        for x, y in zip(p, states[0][1]):
            assert torch.equal(x, y)
        for x, y in zip(c[4:], p[4:]):  # the ring's live rows: positions 96..149
            rows = torch.arange(96, 150, device=cuda) % 64
            assert torch.equal(x[:, :, rows], y[:, :, rows])


@pytest.mark.parametrize("dtype", TYPES)
def test_rejected_drafts_are_taken_back(cuda, dtype):
    """Lengths set back by up to 32 positions, over a block border: later calls see the accepted tokens only."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    g = _gen(cuda, 8)
    c = FlashKVCache8(1, 300, 2, 64, dtype=dtype, device=cuda)
    ref = _oracle(c)
    length, kept = 0, []
    for sq, accepted in [(30, 30), (5, 1), (5, 5), (32, 0), (27, 27), (1, 1), (32, 3), (32, 32), (32, 30)]:
        q, k, v = (_randn(g, 1, sq, 2, 64, dtype=dtype) for _ in range(3))
        lens = torch.tensor([length], dtype=torch.int32, device=cuda)
        out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=lens)
        torch.cuda.synchronize()
        clean = o8.Cache(np.zeros((1, 2, 320, 64)), np.zeros((1, 2, 320, 64)), np.ones((1, 2, 10)), np.ones((1, 2, 10)),
                         np.zeros((1, 2, 64, 64)), np.zeros((1, 2, 64, 64)))
        if kept:
            clean.append(0, 0, np.concatenate([x[0] for x in kept]), np.concatenate([x[1] for x in kept]))
        _append_ref(clean, q, k, v, [0], [length], dtype, out)
        kept.append((_np(k[0, :accepted]), _np(v[0, :accepted])))
        length += accepted
    del ref


def test_rows_of_one_slot(cuda):
    """A padded batch: repeats of a slot with its length take the last row's new keys; a row that disagrees
    about the length makes its slot's rows NaN and writes nothing there."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    dtype, B = torch.bfloat16, 70
    c = _cache(cuda, dtype, 80, 100, 2, True, 6)
    ref = _oracle(c)
    g = _gen(cuda, 2)
    q, k, v = (_randn(g, B, 1, 2, 64, dtype=dtype) for _ in range(3))
    slots, lens = list(range(B)), [(5 * i) % 99 for i in range(B)]
    for i, s in ((3, 9), (40, 9), (69, 9), (12, 31)):
        slots[i], lens[i] = s, lens[s]
    slots[50], lens[50] = 20, lens[20] + 1  # disagrees
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=i32(lens), cache_batch_idx=i32(slots))
    torch.cuda.synchronize()
    last = {s: b for b, s in enumerate(slots)}
    assert torch.isnan(out[[20, 50]]).all()
    good = [b for b in range(B) if b not in (20, 50)]
    src = [last[slots[b]] for b in good]
    before = _oracle(c)  # the outputs are of the old state: check them against it, then the state
    sub = lambda t, i: t[torch.tensor(i, device=cuda)]
    for j, b in enumerate(good):
        n, s = lens[b], slots[b]
        kk = np.concatenate([ref.read(0, s, n), _np(k[src[j]]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, s, n), _np(v[src[j]]).transpose(1, 0, 2)], 1)
        want, mag, big = o8.attend(_np(q[b]), kk, vv, [n + 1], SCALE)
        _check(out[b], want, mag, big, n + 1, dtype, f"row {b}")
    for s, b in last.items():
        if s != 20:
            ref.append(s, lens[b], _np(k[b]), _np(v[b]))
    _same_state(c, ref)
    # the same rule where the append has a launch of its own
    q, k, v = (_randn(g, 4, 40, 2, 64, dtype=dtype) for _ in range(3))
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=i32([7, 50, 7, 8]), cache_batch_idx=i32([1, 2, 1, 2]))
    torch.cuda.synchronize()
    assert torch.isnan(out[[1, 3]]).all() and torch.isfinite(out[[0, 2]]).all()
    ref.append(1, 7, _np(k[2]), _np(v[2]))
    _same_state(c, ref)
    del before, sub


def test_bad_rows_give_nan_and_write_nothing(cuda):
    from whisperdrz_amd import flash_attn_with_kvcache8

    dtype = torch.float16
    c = _cache(cuda, dtype, 3, 100, 2, True, 7)
    ref = _oracle(c)
    g = _gen(cuda, 2)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    for sq in (1, 40):
        q, k, v = (_randn(g, 6, sq, 2, 64, dtype=dtype) for _ in range(3))
        lens, slots = [0, 101 - sq, -1, 5, 2147483647, 3], [-1, 0, 1, 3, 2, 2147483647]
        out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=i32(lens), cache_batch_idx=i32(slots))
        torch.cuda.synchronize()
        assert torch.isnan(out).all()
        _same_state(c, ref)
    q = _randn(g, 4, 1, 2, 64, dtype=dtype)
    out = flash_attn_with_kvcache8(q, c, cache_seqlens=i32([101, -1, 100, 4]), cache_batch_idx=i32([0, 1, 2, 3]))
    assert torch.isnan(out[[0, 1, 3]]).all() and torch.isfinite(out[2]).all()


# ---- values that are not finite ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_places_do_not_count(cuda, dtype):
    """NaN and infinities behind the lengths (codes, ring, later drafts) reach no row that does not see
    them; an infinite value that is seen gives an infinity, a NaN gives NaN in its dimension."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, dtype, 2, 100, 2, True, 9)
    for t in (c.k_codes, c.v_codes):
        t.view(torch.uint8)[:, :, 64:] = 0x7F  # stale
    for t in (c.k_ring, c.v_ring):
        t[:, :, [p % 64 for p in range(70, 128)]] = float("nan")  # but positions 64..69
    ref = _oracle(c)
    g = _gen(cuda, 2)
    q, k, v = (_randn(g, 2, 6, 2, 64, dtype=dtype) for _ in range(3))
    v[0, 3, 0, 5] = float("nan")
    v[0, 2, 1, 7] = float("inf")
    k[0, 4, 1, 9] = float("nan")
    v[1, 5] = float("inf")
    k[1, 5] = -float("inf")
    lens = [70, 70]
    out = flash_attn_with_kvcache8(q, c, k, v, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda))
    torch.cuda.synchronize()
    got = _np(out)
    for b in range(2):
        kk = np.concatenate([ref.read(0, b, 70), _np(k[b]).transpose(1, 0, 2)], 1)
        vv = np.concatenate([ref.read(1, b, 70), _np(v[b]).transpose(1, 0, 2)], 1)
        with np.errstate(invalid="ignore"):
            want, mag, big = o8.attend(_np(q[b]), kk, vv, [71 + t for t in range(6)], SCALE)
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(got[b]), np.isnan(want)) and np.array_equal(got[b][~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
        lim = o8.bound(np.where(fine, want, 0), np.where(fine, mag, 0), np.where(np.isfinite(big), big, 0), 76, HALF[dtype])
        assert (np.abs(np.where(fine, got[b] - np.where(fine, want, 0), 0)) <= lim).all()
    assert np.isinf(got[0, 2, 1, 7]) and np.isnan(got[0, 3, 0, 5]) and np.isfinite(got[0, :2]).all() and np.isfinite(got[1, :5]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,sq", [(2, 1), (2, 5), (2, 20), (18, 64)])
@pytest.mark.parametrize("at", [0, 40, 69])
def test_nan_codes(cuda, dtype, B, sq, at):
    """What was not finite when it was stored: a key makes its rows NaN, a value its dimension."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    H = 16
    c = _cache(cuda, dtype, B, 70, H, False, 61)
    q = _randn(_gen(cuda, 2), B, sq, H, 64, dtype=dtype)
    clean = flash_attn_with_kvcache8(q, c)
    c.k_codes.view(torch.uint8)[0, 1, at, 7] = 0x7F
    c.v_codes.view(torch.uint8)[1, 2, at, 9] = 0xFF
    out = flash_attn_with_kvcache8(q, c)
    torch.cuda.synchronize()
    nan = torch.zeros_like(out, dtype=torch.bool)
    nan[0, :, 1], nan[1, :, 2, 9] = True, True
    assert torch.equal(torch.isnan(out), nan) and torch.equal(out[~nan], clean[~nan])


# ---- layouts, streams, graphs ---------------------------------------------------------------------


def test_strided_operands_and_given_output(cuda):
    from whisperdrz_amd import flash_attn_with_kvcache8

    dtype = torch.bfloat16
    g = _gen(cuda, 5)
    a, b = (_cache(cuda, dtype, 3, 100, 4, True, 10) for _ in range(2))
    qkv = _randn(g, 3, 4, 5, 3, 64, dtype=dtype)  # [B, H, sq, 3, 64]: heads first
    q, k, v = (qkv[:, :, :, i].permute(0, 2, 1, 3) for i in range(3))
    out = torch.full((3, 5, 4, 128), 7.0, dtype=dtype, device=cuda)
    lens = torch.tensor([20, 31, 64], dtype=torch.int64, device=cuda)
    idx = torch.tensor([2, 9, 0, 9, 1, 9], dtype=torch.int32, device=cuda)[::2]
    res = flash_attn_with_kvcache8(q, a, k, v, lens, idx, out=out[..., 64:])
    want = flash_attn_with_kvcache8(q.contiguous(), b, k.contiguous(), v.contiguous(), lens.int(), idx.contiguous())
    torch.cuda.synchronize()
    assert res.data_ptr() == out[..., 64:].data_ptr() and torch.equal(out[..., 64:], want) and bool((out[..., :64] == 7).all())
    for x, y in zip(_bits(a), _bits(b)):
        assert torch.equal(x, y)


def test_lengths_given_as_a_number_and_empty_calls(cuda):
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, torch.bfloat16, 3, 100, 2, False, 10)
    q = _randn(_gen(cuda, 1), 2, 3, 2, 64, dtype=torch.bfloat16)
    t = torch.tensor([50, 50], dtype=torch.int32, device=cuda)
    assert torch.equal(flash_attn_with_kvcache8(q, c, cache_seqlens=50), flash_attn_with_kvcache8(q, c, cache_seqlens=t))
    assert flash_attn_with_kvcache8(q[:0], c).shape == (0, 3, 2, 64) and flash_attn_with_kvcache8(q[:, :0], c).shape == (2, 0, 2, 64)
    c.set_cross_attention(q[:0], q[:0])
    c.set_cross_attention(q[:, :0], q[:, :0])


def test_refusals_on_the_gpu(cuda):
    from whisperdrz_amd import flash_attn_with_kvcache8

    bf = torch.bfloat16
    c, x = _cache(cuda, bf, 3, 100, 2, True, 1), _cache(cuda, bf, 3, 100, 2, False, 1)
    q = torch.zeros(2, 1, 2, 64, dtype=bf, device=cuda)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda)
    f = flash_attn_with_kvcache8
    for call, err in [
        (lambda: f(q.float(), x), TypeError), (lambda: f(q.half(), c, cache_seqlens=lens), TypeError),
        (lambda: f(q[..., :32], x), ValueError), (lambda: f(q[0], x), ValueError), (lambda: f(q, c), ValueError),
        (lambda: f(q, c, q, None, lens), ValueError), (lambda: f(q, c, q, q), ValueError),
        (lambda: f(q, x, q, q, lens), ValueError), (lambda: f(q, c, q[:1], q, lens), ValueError),
        (lambda: f(q, c, q.half(), q, lens), TypeError), (lambda: f(q, c, q, q, lens[:1]), ValueError),
        (lambda: f(q, c, q, q, lens.float()), TypeError), (lambda: f(q, c, q, q, lens.cpu()), RuntimeError),
        (lambda: f(q, c, q, q.cpu(), lens), RuntimeError), (lambda: f(q, x, out=q.half()), ValueError),
        (lambda: f(q, x, softmax_scale=0.0), ValueError), (lambda: f(q.transpose(2, 3), x), ValueError),
        (lambda: x.set_cross_attention(q, q, torch.zeros(3, device=cuda, dtype=torch.long)), ValueError),
        (lambda: x.set_cross_attention(q, q[:1]), ValueError), (lambda: x.set_cross_attention(q.float(), q.float()), TypeError),
        (lambda: c.prefill(q.half(), q.half()), TypeError), (lambda: c.prefill(q, q, 100), ValueError),
        (lambda: x.set_cross_attention(q.repeat(2, 1, 1, 1), q.repeat(2, 1, 1, 1)), ValueError),
    ]:
        with pytest.raises(err):
            call()


def test_cache_past_32_bit_offsets(cuda):
    """More than 2^32 bytes of codes a tensor: the last slots of a large pool."""
    from whisperdrz_amd import FlashKVCache8, flash_attn_with_kvcache8

    dtype, H, L = torch.bfloat16, 20, 1500
    S = 2 ** 32 // (H * 1504 * 64) + 3
    c = FlashKVCache8(S, L, H, 64, dtype=dtype, device=cuda, ring=False)
    small = FlashKVCache8(2, L, H, 64, dtype=dtype, device=cuda, ring=False)
    g = _gen(cuda, 3)
    k, v, q = (_randn(g, 2, L, H, 64, dtype=dtype) for _ in range(3))
    c.set_cross_attention(k, v, torch.tensor([S - 1, S - 2], device=cuda))
    small.set_cross_attention(k, v)
    at = torch.tensor([S - 1, S - 2], dtype=torch.int32, device=cuda)
    for sq in (1, 5):
        got, want = flash_attn_with_kvcache8(q[:, :sq], c, cache_batch_idx=at), flash_attn_with_kvcache8(q[:, :sq], small)
        assert torch.equal(got, want)
    assert not c.k_codes[: S - 2].view(torch.uint8).any()


@pytest.mark.parametrize("B,sq,L", [(2, 1, 200), (1, 3, 3000), (2, 40, 200)])
def test_graph_replays(cuda, B, sq, L):
    """A captured append whose inputs change between replays, eager work between them; two graphs of split
    rows share no workspace."""
    from whisperdrz_amd import flash_attn_with_kvcache8

    dtype = torch.bfloat16
    g = _gen(cuda, 3)
    H = 4
    c, e = (_cache(cuda, dtype, B, L, H, True, 20) for _ in range(2))
    q, k, v = (torch.zeros(B, sq, H, 64, dtype=dtype, device=cuda) for _ in range(3))
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        flash_attn_with_kvcache8(q, e, k, v, lens)
    torch.cuda.current_stream().wait_stream(side)
    e = _cache(cuda, dtype, B, L, H, True, 20)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(flash_attn_with_kvcache8(q, c, k, v, lens))
    for i in range(4):
        for t in (q, k, v):
            t.copy_(_randn(g, B, sq, H, 64, dtype=dtype))
        lens.copy_(torch.tensor([29 + i * sq + b for b in range(B)]))
        graphs[i % 2].replay()
        want = flash_attn_with_kvcache8(q, e, k, v, lens)
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want)
        for x, y in zip(_bits(c), _bits(e)):
            assert torch.equal(x, y)


def test_calls_on_two_streams(cuda):
    from whisperdrz_amd import flash_attn_with_kvcache8

    c = _cache(cuda, torch.float16, 1, 4000, 20, False, 5)
    g = _gen(cuda, 3)
    qs = [_randn(g, 1, 1, 20, 64, dtype=torch.float16) for _ in range(2)]
    want = [flash_attn_with_kvcache8(q, c) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(flash_attn_with_kvcache8(qs[i], c))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


# ---- the library with host checks -----------------------------------------------------------------


@pytest.mark.parametrize("case,word", [("slot", "slot 3"), ("overflow", "outside the cache"), ("negative", "outside the cache"),
                                       ("differ", "lengths 5 and 6"), ("read", "positions of 100"), ("good", "")])
def test_debug_library_checks_the_metadata(cuda, case, word):
    import ctypes

    from whisperdrz_amd import _lib

    lib = ctypes.CDLL(str(_lib.DEBUG_LIB_PATH))
    _lib._declare(lib)
    c = _cache(cuda, torch.bfloat16, 3, 100, 2, True, 1)
    before = _bits(c)
    q = _randn(_gen(cuda, 2), 3, 2, 2, 64, dtype=torch.bfloat16)
    out = torch.zeros_like(q)
    idx, lens = {"slot": ([1, 3, 0], [5, 5, 5]), "overflow": ([1, 0, 2], [5, 99, 1]), "negative": ([1, 0, 2], [5, -1, 1]),
                 "differ": ([1, 0, 1], [5, 9, 6]), "read": ([1, 0, 2], [5, 101, 6]), "good": ([1, 0, 1], [5, 9, 5])}[case]
    idx, lens = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in (idx, lens))
    new, st = (None, None) if case == "read" else (q.data_ptr(), _lib.strides(q.stride()))
    rc = lib.wdrz_attn_kvcache8(_lib.WDRZ_BF16, c.struct, q.data_ptr(), _lib.strides(q.stride()), new, st, new, st,
                                lens.data_ptr(), idx.data_ptr(), out.data_ptr(), _lib.strides(q.stride()), 3, 2, 0.125, None, 0,
                                torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    if case == "good":
        assert rc == _lib.WDRZ_OK and out.any()
        return
    assert rc == _lib.WDRZ_EINVAL and word in lib.wdrz_last_error().decode(), lib.wdrz_last_error()
    assert not out.any() and all(torch.equal(x, y) for x, y in zip(before, _bits(c)))
