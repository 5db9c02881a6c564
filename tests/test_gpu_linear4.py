"""GPU parity of the 4-bit linears (linear4, linear4_partials) with the 64-bit product of the values that
codes and scales stand for.

Bound of one result: half a step of its type; the fp32 sum of K products and of the groups' scaled
sums, (K + 64) 2^-24 sum |x w|, through the GELU with a factor of its largest slope, 1.13, and erff's and
the bias's few fp32 roundings, 2^-20 of the pre-activation.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = [torch.bfloat16, torch.float16]


def _layer(cuda, dtype, N, K, group, seed, bias=True):
    from whisperdrz_amd import QuantLinear4

    g = torch.Generator(device=cuda).manual_seed(seed)
    codes = torch.randint(-7, 8, (N, K), generator=g, device=cuda)
    scales = ((torch.rand(N, K // group, generator=g, device=cuda) + 0.5) / (4 * K ** 0.5)).to(dtype)
    b = torch.randn(N, generator=g, device=cuda).to(dtype) if bias else None
    return QuantLinear4.from_codes(codes, scales, b), codes.double() * scales.double().repeat_interleave(group, 1), g


def _check(y, x, w, bias, gelu, dtype):
    pre = x.double() @ w.T
    mag = x.double().abs() @ w.abs().T
    if bias is not None:
        pre, mag = pre + bias.double(), mag + bias.double().abs()
    want = torch.nn.functional.gelu(pre) if gelu else pre
    tol = HALF[dtype] * want.abs() + 1.13 * (w.shape[1] + 64) * 2.0 ** -24 * mag + 2.0 ** -20 * pre.abs() + 2.0 ** -25
    over = ((y.double() - want).abs() - tol).max().item()
    assert torch.isfinite(y).all() and over <= 0, f"{over:.3e} over the bound"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 33, 64, 65, 130])
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (8, 128, 128), (17, 160, 32), (40, 1280, 64), (100, 704, 64), (130, 512, 128)])
def test_linear4(cuda, dtype, M, N, K, group):
    from whisperdrz_amd import linear4

    lin, w, g = _layer(cuda, dtype, N, K, group, M + N + K)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    for gelu in (False, True):
        _check(linear4(x, lin, gelu), x, w, lin.bias, gelu, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group", [(1, 5120, 1280, 32), (52, 3840, 1280, 64), (4, 1280, 5120, 128), (500, 1280, 1280, 32),
                                         (1000, 1000, 5120, 64), (3, 51866, 1280, 128), (257, 2048, 512, 128),
                                         # tiles of 64 x 128 and of 128 x 160, whole and with all three ends inside a tile
                                         (2048, 1280, 1280, 128), (2047, 1100, 1312, 32), (2040, 1111, 1344, 64),
                                         (3584, 1280, 5120, 128), (3500, 1234, 2080, 32), (3333, 1249, 2112, 64)])
def test_linear4_at_the_decoders_sizes(cuda, dtype, M, N, K, group):
    from whisperdrz_amd import linear4

    lin, w, g = _layer(cuda, dtype, N, K, group, M, bias=M != 4)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    _check(linear4(x, lin, M == 1), x, w, lin.bias, M == 1, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("N,K,group", [(7169, 160, 32), (7300, 1280, 64), (16393, 288, 32), (20001, 1280, 128), (32769, 1376, 32), (51865, 640, 64)])
def test_many_features_and_few_rows(cuda, dtype, M, N, K, group):
    """One, two and four feature tiles a workgroup, the last ones part of a group or past the features."""
    from whisperdrz_amd import linear4

    lin, w, g = _layer(cuda, dtype, N, K, group, M + N)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    _check(linear4(x, lin), x, w, lin.bias, False, dtype)
    if M > 1:
        assert torch.equal(linear4(x, lin)[:1], linear4(x[:1], lin))  # a row's result is its own


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K,group,n_split", [(1, 1280, 1280, 64, 2), (5, 1280, 5120, 32, 4), (64, 1000, 640, 128, 4),
                                                 (17, 40, 96, 32, 4), (70, 33, 256, 64, 2), (600, 1280, 5120, 64, 4),
                                                 (900, 1240, 1376, 32, 2), (3584, 1280, 5120, 128, 2), (100, 2000, 160, 32, 4)])
def test_linear4_partials(cuda, dtype, M, N, K, group, n_split):
    from whisperdrz_amd import linear4_partials

    lin, w, g = _layer(cuda, dtype, N, K, group, M + K)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    part = linear4_partials(x, lin, n_split)
    assert part.shape == (n_split, M, N) and part.dtype == torch.float32
    mag = x.double().abs() @ w.abs().T
    assert ((part.double().sum(0) - x.double() @ w.T).abs() <= (K + 64) * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_every_weight_value(cuda, dtype):
    """One-hot rows read back every code exactly, each place of a tile."""
    from whisperdrz_amd import QuantLinear4, linear4

    codes = torch.arange(48 * 160, device=cuda).view(48, 160) % 15 - 7
    scales = torch.ones(48, 5, device=cuda, dtype=dtype)
    lin = QuantLinear4.from_codes(codes, scales)
    assert torch.equal(linear4(torch.eye(160, device=cuda, dtype=dtype), lin).float().T, codes.float())


def test_strided_rows_and_shapes(cuda):
    from whisperdrz_amd import linear4, linear4_partials

    dtype = torch.bfloat16
    lin, w, g = _layer(cuda, dtype, 40, 256, 64, 3)
    big = torch.randn(6, 2, 320, generator=g, device=cuda).to(dtype)
    x = big[:, 1, 16:272]
    y = linear4(x, lin)
    _check(y, x, w, lin.bias, False, dtype)
    assert torch.equal(lin(x), y)
    assert torch.equal(linear4(x.contiguous().view(2, 3, 256), lin).view(6, 40), y)
    assert linear4(x[:0], lin).shape == (0, 40) and linear4_partials(x[:0], lin, 2).shape == (2, 0, 40)
    assert torch.equal(linear4(x[2], lin), y[2])  # one row without a batch
    for bad, err in [(x.float(), TypeError), (x.half(), TypeError), (x[:, :128], ValueError), (x.cpu(), RuntimeError),
                     (big[:, 0, 1:257], ValueError), (big.transpose(0, 1)[:, :, :256], ValueError)]:  # rows without one stride
        with pytest.raises(err):
            linear4(bad, lin)
    with pytest.raises(NotImplementedError, match="n_split 3"):
        linear4_partials(x, lin, 3)


def test_rows_far_apart(cuda):
    """Rows more than 2^22 elements apart: beyond the tiles' 31-bit offsets."""
    from whisperdrz_amd import linear4

    dtype = torch.bfloat16
    lin, w, g = _layer(cuda, dtype, 512, 256, 64, 3)
    big = torch.empty(600, (1 << 22) + 8, dtype=dtype, device=cuda)
    x = big[:, 64:320]
    x.copy_(torch.randn(600, 256, generator=g, device=cuda))
    _check(linear4(x, lin), x, w, lin.bias, False, dtype)


@pytest.mark.parametrize("M,K", [(200, 256), (700, 288), (3000, 1312), (3000, 160)])
def test_infinities_in_tiles(cuda, M, K):
    """An infinity in the last inputs of a K that ends inside a chunk counts once, in its row."""
    from whisperdrz_amd import linear4

    dtype = torch.bfloat16
    lin, w, g = _layer(cuda, dtype, 1280, K, 32, 9)
    x = torch.randn(M, K, generator=g, device=cuda).to(dtype)
    y = linear4(x, lin)
    x[M // 2, K - 1] = float("inf")
    x[M - 1, K - 8] = float("nan")
    z = linear4(x, lin)
    want = x[M // 2].double() @ w.T + lin.bias.double()
    rest = [i for i in range(M) if i not in (M // 2, M - 1)]
    assert torch.equal(y[rest], z[rest]) and torch.isnan(z[M - 1]).all()
    assert torch.equal(torch.isnan(z[M // 2]), torch.isnan(want)) and torch.equal(torch.isinf(z[M // 2]), torch.isinf(want))


@pytest.mark.parametrize("M", [1, 20, 200])
def test_what_is_not_finite_stays_in_its_row(cuda, M):
    from whisperdrz_amd import linear4

    dtype = torch.float16
    lin, w, g = _layer(cuda, dtype, 64, 256, 64, 9)
    x = torch.randn(M, 256, generator=g, device=cuda).to(dtype)
    y = linear4(x, lin)
    x[M - 1, 7] = float("inf")
    z = linear4(x, lin)
    want = (x[M - 1].double() @ w.T) + lin.bias.double()
    assert torch.equal(y[: M - 1], z[: M - 1])
    assert torch.equal(torch.isnan(z[M - 1]), torch.isnan(want))
    assert torch.equal(z[M - 1][~torch.isnan(want)].double(), want[~torch.isnan(want)])


def test_partials_into_the_residual(cuda):
    """linear4_partials with add_layernorm_partials_, as the decode step uses them."""
    from whisperdrz_amd import add_layernorm_partials_, linear4_partials

    dtype = torch.bfloat16
    lin, w, g = _layer(cuda, dtype, 1280, 1280, 64, 4)
    ln = torch.nn.LayerNorm(1280).to(cuda, dtype)
    h, x = (torch.randn(7, 1280, generator=g, device=cuda).to(dtype) for _ in range(2))
    delta = (h.double() @ w.T + lin.bias.double())
    got = x.clone()
    y = add_layernorm_partials_(got, linear4_partials(h, lin, 2), lin, ln)
    # two roundings of half a step: the Linear's output's and the sum's
    assert ((got.double() - (x.double() + delta)).abs() <= 2.0 ** -8 * (delta.abs() + got.double().abs()) * 1.01 + 1e-4).all()
    assert torch.equal(y, torch.nn.functional.layer_norm(got.float(), (1280,), ln.weight.float(), ln.bias.float(), ln.eps).to(dtype)) or \
        (y.float() - torch.nn.functional.layer_norm(got.float(), (1280,))).abs().max() < 2.0 ** -5


def test_graph_replays(cuda):
    from whisperdrz_amd import linear4

    dtype = torch.bfloat16
    lin, w, g = _layer(cuda, dtype, 512, 512, 32, 4)
    x = torch.zeros(20, 512, device=cuda, dtype=dtype)
    linear4(x, lin)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = linear4(x, lin)
    for _ in range(3):
        x.copy_(torch.randn(20, 512, generator=g, device=cuda))
        gr.replay()
        assert torch.equal(y, linear4(x, lin))
