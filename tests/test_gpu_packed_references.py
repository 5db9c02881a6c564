"""The softmax reference of packed attention where a query's first keys have scores of -inf: they weigh nothing, and the
reference comes from the first that do, however low their scores are."""
import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("none,n", [(32, 40), (40, 300), (100, 700), (64, 64 + 33)])
def test_first_keys_without_weight(cuda, dtype, dim, causal, none, n):
    """Scores are exact products of powers of two plus small ones: d = (D + 4) 2^-24 times their largest sum, 2 d of the weights,
    half a step of a probability and 2^-20 of the exponential, of the largest value; half a step of the result."""
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(n, 2, dim, generator=g).to(dtype) for _ in range(3))
    q[:, :, 0], k[:, :, 0] = 32.0, -64.0  # scores around -2048 scale: 2^-150 of a reference of 0 and below
    k[:none, :, 0] = -float("inf")
    scale = 0.125
    cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    got = w.packed_attention(q.to(cuda), k.to(cuda), v.to(cuda), cu, causal=causal, scale=scale).cpu()
    pick = [t for t in (none, none + 1, none + 31, n // 2, n - 1) if none <= t < n] if causal else [0, 1, n // 2, n - 1]
    limit = [t + 1 if causal else n for t in pick]
    want, _ = attention(q[pick], k, v, limit, scale)
    assert want.isfinite().all()
    d = (dim + 4) * 2.0**-24 * scale * float((q.float().abs().amax((0, 1)) * k[none:].float().abs().amax((0, 1))).sum())
    u = torch.finfo(dtype).eps / 2
    tol = u * want.abs() + (2 * d + 2.0**-20 + u) * float(v.float().abs().max()) + 1e-7
    err = (got[pick].double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
