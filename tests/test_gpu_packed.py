"""packed_attention on the GPU against the 64-bit restatement.

Tolerance: half a step of the output type of the value, and the probabilities' relative error times the largest value
they weigh: 2 d for scores off by d = (D + 4) 2^-24 scale max(sum |q| |k|), 2^-20 of the exponential, and the half
step of their one 16-bit operand."""
import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import attention

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def sums(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int64).cumsum(0).to(torch.int32)


def assert_rows(got, want, big, vmax, dtype, dim):
    u, d = torch.finfo(dtype).eps / 2, (dim + 4) * 2.0**-24 * dim**-0.5 * big
    tol = u * want.abs() + (2 * d + 2.0**-20 + u) * vmax + 1e-7
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"


def check(cuda, dtype, lens, H, Hk, dim, causal=True, klens=None, extra=0, seed=0):
    print(f"packed {dtype} lens={lens[:8]} keys={klens and klens[:8]} H={H}/{Hk} D={dim} causal={causal}", flush=True)
    g = torch.Generator().manual_seed(seed + sum(lens))
    T = sum(lens) + extra
    if klens is None:
        x = torch.randn(T, H + 2 * Hk, dim, generator=g).to(dtype).to(cuda)
        q, k, v = x[:, :H], x[:, H : H + Hk], x[:, H + Hk :]
    else:
        q = torch.randn(T, H, dim, generator=g).to(dtype).to(cuda)
        x = torch.randn(sum(klens) + 3, 2 * Hk, dim, generator=g).to(dtype).to(cuda)
        k, v = x[:, :Hk], x[:, Hk:]
    out = torch.full((T, H, dim), 7.0, dtype=dtype, device=cuda)
    cu = sums(lens).to(cuda)
    got = w.packed_attention(q, k, v, cu, None if klens is None else sums(klens).to(cuda), causal, out=out)
    assert got is out and bool((out[sum(lens) :] == 7.0).all())
    a = b = 0
    for n, nk in zip(lens, klens or lens):
        limit = [t + 1 + nk - n for t in range(n)] if causal else [nk] * n
        if n > 40:  # the restatement takes every query by itself: some of a long sequence, both ends and block edges
            pick = sorted({t for t in (0, 1, 31, 32, 63, 64, 127, 128, 255, 256, n // 2, n - 2, n - 1) if t < n})
        else:
            pick = list(range(n))
        want, big = attention(q[a : a + n].cpu()[pick], k[b : b + nk].cpu(), v[b : b + nk].cpu(), [limit[t] for t in pick], dim**-0.5)
        assert_rows(got[a : a + n][pick], want, big, float(v.float().abs().max()), dtype, dim)
        a, b = a + n, b + nk
    return q, k, v, got


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,Hk,dim", [(1, 1, 64), (4, 4, 64), (6, 2, 64), (8, 1, 128), (3, 3, 128), (20, 20, 64)])
def test_short_sequences(cuda, dtype, H, Hk, dim):
    check(cuda, dtype, [1, 0, 13, 2, 33, 0, 1], H, Hk, dim, extra=5)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[63, 64, 65], [31, 32, 127, 128, 129], [255, 256, 257], [700], [1, 513, 1], [2000, 3, 40]])
def test_lengths_around_the_blocks(cuda, dim, lens):
    check(cuda, BF16, lens, 2, 1, dim)
    check(cuda, FP16, lens, 2, 2, dim, causal=False, extra=70)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_their_own(cuda, dim, causal):
    """More keys than queries, fewer (queries that see nothing), and none."""
    lens, klens = [5, 40, 17, 3, 130, 64], [70, 7, 17, 0, 300, 33]
    q, k, v, got = check(cuda, BF16, lens, 4, 2, dim, causal, klens)
    if causal:
        assert not got[5 : 5 + 33].any() and not got[62:65].any()  # 33 of 40 queries, and all of the fourth
    check(cuda, FP16, [1, 224, 9], 3, 3, dim, causal, [1500, 700, 64])


def test_many_sequences(cuda):
    """More than one wavefront of sums: the work items are found over all of them."""
    lens = [(i * 7) % 23 for i in range(300)]
    check(cuda, BF16, lens, 2, 2, 64)
    check(cuda, FP16, [1] * 130 + [90] + [0] * 70, 1, 1, 128)


@pytest.mark.parametrize("dim", [64, 128])
def test_scores_that_grow_move_the_reference(cuda, dim):
    n = 300
    g = torch.Generator().manual_seed(1)
    q = torch.randn(n, 1, dim, generator=g)
    k = q[:1] * (torch.arange(n) // 16 % 11)[:, None, None] * 0.4 + 0.1 * torch.randn(n, 1, dim, generator=g)
    v = torch.randn(n, 1, dim, generator=g)
    q = (q * 0.2 + q[:1]).to(FP16)
    k, v = k.to(FP16), v.to(FP16)
    got = w.packed_attention(q.to(cuda), k.to(cuda), v.to(cuda), sums([n]).to(cuda))
    want, big = attention(q, k, v, [t + 1 for t in range(n)], dim**-0.5)
    assert_rows(got, want, big, float(v.float().abs().max()), FP16, dim)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_what_nobody_sees_does_not_count(cuda, dim, odd):
    """Later tokens of a sequence, other sequences and rows behind the last may hold anything."""
    lens = [40, 70, 150]
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(260 + 9, 2, dim, generator=g).to(BF16) for _ in range(3))
    k[60], v[60] = odd, odd  # position 20 of the second sequence
    k[149:], v[149:] = odd, odd  # from position 39 of the third on
    got = w.packed_attention(q.to(cuda), k.to(cuda), v.to(cuda), sums(lens).to(cuda)).cpu()
    a = 0
    for n, clean in zip(lens, (40, 20, 39)):
        want, big = attention(q[a : a + clean], k[a : a + clean], v[a : a + clean], [t + 1 for t in range(clean)], dim**-0.5)
        assert_rows(got[a : a + clean], want, big, float(v[a : a + clean].float().abs().max()), BF16, dim)
        assert got[a + clean : a + n].isnan().all()
        a += n


def test_sums_out_of_order_stay_in_bounds(cuda):
    q = torch.randn(50, 2, 64, device=cuda).to(BF16)
    for cu in ([0, 60], [-5, 10, 8, 90, 3], [50, 0], [70, 80], [-9, -3]):
        out = w.packed_attention(q, q, q, torch.tensor(cu, dtype=torch.int32, device=cuda), out=torch.zeros_like(q))
        assert out.isfinite().all()


def test_nothing_to_do_and_refusals(cuda):
    x = torch.randn(6, 4, 64, device=cuda).to(BF16)
    cu = sums([2, 4]).to(cuda)
    assert w.packed_attention(x[:0], x[:0], x[:0], sums([0, 0]).to(cuda)).shape == (0, 4, 64)
    assert w.packed_attention(x, x, x, sums([]).to(cuda)).shape == x.shape
    assert not w.packed_attention(x, x[:0], x[:0], cu, sums([0, 0]).to(cuda), causal=False).any()
    for args, err in (((x.float(),) * 3 + (cu,), TypeError), ((x, x.half(), x, cu), TypeError), ((x, x[:, :3], x[:, :3], cu), ValueError),
                      ((x, x[:4], x[:4], cu), ValueError), ((x, x, x, cu, cu[:2]), ValueError), ((x[0], x, x, cu), ValueError),
                      ((x, x, x, cu.float()), TypeError), ((x, x, x, cu[None]), ValueError), ((x[..., :32],) * 3 + (cu,), NotImplementedError)):
        with pytest.raises(err):
            w.packed_attention(*args)
    with pytest.raises(ValueError):
        w.packed_attention(x, x, x, cu, out=x[:4])
    assert torch.equal(w.packed_attention(x, x, x, cu.long()), w.packed_attention(x, x, x, cu))


def test_captured_calls_follow_their_sums(cuda):
    q, k, v = (torch.randn(200, 2, 64, device=cuda).to(BF16) for _ in range(3))
    cu = sums([50, 100]).to(cuda)
    w.packed_attention(q, k, v, cu)
    g, out = torch.cuda.CUDAGraph(), torch.zeros_like(q)
    with torch.cuda.graph(g):
        w.packed_attention(q, k, v, cu, out=out)
    for lens in ([50, 100], [1, 199], [120, 0], [50, 100]):
        cu.copy_(sums(lens))
        out.zero_()
        g.replay()
        assert torch.equal(out, w.packed_attention(q, k, v, cu, out=torch.zeros_like(q)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("H,Hk", [(1, 1), (4, 4), (6, 3), (8, 1)])
def test_few_queries_over_many_keys(cuda, causal, H, Hk):
    """Two wavefronts share a query block: sequences of which one half of a tile's keys is empty, that begin or end inside a tile, and
    queries that see no key at all."""
    check(cuda, BF16, [1, 40, 3, 70, 0, 33], H, Hk, 64, causal, klens=[20, 700, 0, 33, 900, 1100])
    check(cuda, FP16, [5], H, Hk, 64, causal, klens=[289])


def test_few_queries_of_many_sequences(cuda):
    check(cuda, BF16, [1] * 40 + [0, 2] * 15, 1, 1, 64, False, klens=[300, 250] * 35)


@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_what_nobody_sees_does_not_count_in_halves(cuda, odd):
    """As above with one sequence long enough for two wavefronts: either may hold the value, in its first step or later."""
    for at in (0, 31, 32, 63, 64, 250, 300):
        g = torch.Generator().manual_seed(at)
        q, k, v = (torch.randn(310, 2, 64, generator=g).to(BF16) for _ in range(3))
        k[at], v[at] = odd, odd
        got = w.packed_attention(q.to(cuda), k.to(cuda), v.to(cuda), sums([305]).to(cuda)).cpu()
        pick = [t for t in (0, 1, 15, 16, 31, 32, 60, 249, 299) if t < at]
        if pick:
            clean = pick[-1] + 1
            want, big = attention(q[pick], k[:clean], v[:clean], [t + 1 for t in pick], 64**-0.5)
            assert_rows(got[pick], want, big, float(v[:clean].float().abs().max()), BF16, 64)
        assert got[at:305].isnan().all()
