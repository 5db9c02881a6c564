"""linear4_partials with add_layernorm_partials_, as the decode step uses them: the residual and the LayerNorm, with
weights and a bias of its own, against 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,K,n_split", [(1, 1280, 2), (7, 1280, 2), (52, 5120, 4)])
def test_partials_into_the_residual_and_its_norm(cuda, dtype, rows, K, n_split):
    from whisperdrz_amd import QuantLinear4, add_layernorm_partials_, linear4_partials

    n = 1280
    g = torch.Generator(device=cuda).manual_seed(rows)
    randn = lambda *shape: torch.randn(shape, generator=g, device=cuda)
    lin = QuantLinear4.from_weight((randn(n, K) / K ** 0.5).to(dtype), randn(n).to(dtype), 64)
    ln = torch.nn.LayerNorm(n).to(cuda, dtype)
    with torch.no_grad():
        ln.weight.copy_(1 + 0.3 * randn(n))
        ln.bias.copy_(randn(n))
    h, x = randn(rows, K).to(dtype), randn(rows, n).to(dtype)
    w = lin.dequantize().double()
    delta = h.double() @ w.T + lin.bias.double()
    sums = (K + 64) * 2.0 ** -24 * (h.double().abs() @ w.abs().T + lin.bias.double().abs())  # fp32 sums
    got = x.clone()
    with torch.no_grad():
        y = add_layernorm_partials_(got, linear4_partials(h, lin, n_split), lin, ln)
    # two roundings of half a step: the Linear's output and the sum
    want = x.double() + delta
    assert ((got.double() - want).abs() <= HALF[dtype] * (1.01 * delta.abs() + 1.01 * want.abs()) + 2 * sums + 2.0 ** -24).all()
    # the norm of the residual as it stands: its own rounding, and fp32 statistics over n values, (n + 64) 2^-24 at
    # most of the row's largest normalised magnitude, times the weight
    r = got.double()
    mean, var = r.mean(1, keepdim=True), r.var(1, unbiased=False, keepdim=True)
    z = (r - mean) / (var + ln.eps).sqrt()
    norm = z * ln.weight.double() + ln.bias.double()
    slack = (n + 64) * 2.0 ** -24 * z.abs().amax(1, keepdim=True) * ln.weight.double().abs() + 2.0 ** -20 * ln.bias.double().abs()
    assert ((y.double() - norm).abs() <= HALF[dtype] * norm.abs() + slack + 2.0 ** -24).all()
