"""Infinite values that queries see, in attention over pages: a key's weight is above 0 however small, so its infinite value
is the result, of both signs NaN, and NaN is NaN. The other dims and rows keep their results."""
import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import attention

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,group,dim,sq,append,max_len", [
    (2, 1, 64, 1, True, 300), (2, 4, 128, 1, False, 300), (1, 2, 64, 5, True, 300), (3, 3, 128, 7, False, 300), (2, 1, 64, 1, True, 3000),
    (1, 4, 128, 5, True, 3000)])
def test_infinite_values_that_are_seen(cuda, dtype, heads, group, dim, sq, append, max_len):
    """Tolerance of the finite results as in the other tests of pages: half a step of the output, 2 d + 2^-16 of the largest value,
    d = (D + 4) 2^-24 scale max(sum |q| |k|)."""
    lens = [290, 40, max_len - sq, 200]
    g = torch.Generator().manual_seed(dim + sq)
    t = w.PageTables(4, sum(-(-(n + sq) // 16) for n in lens), 16, max_len, device=cuda)
    cache = w.FlashKVPages(t, heads, dim, dtype)
    k, v = (torch.randn(sum(lens), heads, dim, generator=g).to(dtype) for _ in range(2))
    first = [sum(lens[:i]) for i in range(4)]
    v[first[0] + 3, 0, 5] = INF  # in a block that every query sees whole
    v[first[0] + 70, 0, 9], v[first[0] + 71, 0, 9] = INF, -INF
    v[first[0] + 100, 0, 20] = NAN
    v[first[1] + 39, 0, dim - 1] = -INF  # in the block that ends the cached rows
    v[first[2] + lens[2] // 2, 0, 33] = INF
    v[first[2] + lens[2] - 1, 0, 40] = -INF
    ids = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)
    cache.write(k.to(cuda), v.to(cuda), t.plan(ids(lens), sum(lens)).slots)
    q = torch.randn(4, sq, heads * group, dim, generator=g).to(dtype)
    new = tuple(torch.randn(4, sq, heads, dim, generator=g).to(dtype) for _ in range(2)) if append else (None, None)
    if append:
        t.plan(sq)
    got = w.flash_attn_with_kvpages(q.to(cuda), cache, *(None if x is None else x.to(cuda) for x in new), cache_seqlens=ids(lens)).cpu()
    for b, n in enumerate(lens):
        K, V = k[first[b] : first[b] + n], v[first[b] : first[b] + n]
        limit = [n] * sq
        if append:
            K, V, limit = torch.cat([K, new[0][b]]), torch.cat([V, new[1][b]]), [n + i + 1 for i in range(sq)]
        want, big = attention(q[b], K, V, limit, dim**-0.5)
        assert b == 3 or not want[:, :group].isfinite().all()
        fine = want.isfinite()
        assert torch.equal(got[b].double()[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0))
        assert torch.equal(got[b].isnan(), want.isnan())
        d = (dim + 4) * 2.0**-24 * dim**-0.5 * big
        vmax = float(V.float()[V.isfinite()].abs().max())
        tol = torch.finfo(dtype).eps / 2 * want.abs() + (2 * d + 2.0**-16) * vmax + 1e-7
        assert bool(((got[b].double() - want).abs() <= tol)[fine].all())


@pytest.mark.parametrize("sq,max_len", [(1, 200), (1, 3000), (4, 200)])
def test_infinite_values_of_the_call_itself(cuda, sq, max_len):
    """An infinite value among the appended rows: its own query and those behind it have it, those before it do not."""
    n, dim = max_len - sq, 64
    g = torch.Generator().manual_seed(sq)
    t = w.PageTables(1, -(-max_len // 16), 16, max_len, device=cuda)
    cache = w.FlashKVPages(t, 2, dim, torch.bfloat16)
    k, v = (torch.randn(n, 2, dim, generator=g).bfloat16() for _ in range(2))
    cache.write(k.to(cuda), v.to(cuda), t.plan(n).slots)
    q, kn, vn = (torch.randn(1, sq, 2, dim, generator=g).bfloat16() for _ in range(3))
    vn[0, sq // 2, 0, 7], vn[0, sq - 1, 1, 0] = -INF, INF
    start = t.plan(sq).starts
    got = w.flash_attn_with_kvpages(q.to(cuda), cache, kn.to(cuda), vn.to(cuda), cache_seqlens=start).cpu()[0].double()
    want, big = attention(q[0], torch.cat([k, kn[0]]), torch.cat([v, vn[0]]), [n + i + 1 for i in range(sq)], dim**-0.5)
    fine = want.isfinite()
    assert int((~fine).sum()) == sq - sq // 2 + 1 and torch.equal(got[~fine], want[~fine])
    tol = 2.0**-8 * want.abs() + (2 * (dim + 4) * 2.0**-24 * dim**-0.5 * big + 2.0**-16) * float(v.float().abs().max() + 4) + 1e-7
    assert bool(((got - want).abs() <= tol)[fine].all())
