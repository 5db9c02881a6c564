"""token_logprobs on the GPU against the 64-bit restatement.

Tolerance: the exponentials are off by 2^-21 relative (2 steps of 2^-23 of the hardware's, one rounding each of the
difference and of its product with log2 e where it counts, |d| up to 4), fp32 sums of up to 64 terms by 64 * 2^-24, and the
results are rounded to fp32: 2^-17 of the part that the sum makes (ln Z and the entropy) and 2^-24 of the value."""
import math

import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import logprobs

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(cuda, x, tokens, top, blocked=None):
    got = w.token_logprobs(x.to(cuda), tokens.to(cuda), top, None if blocked is None else blocked.to(cuda))
    lp, entropy, values, ids = logprobs(x.reshape(-1, x.shape[-1]), tokens.reshape(-1), top, blocked)
    assert got.top_ids.shape == (*tokens.shape, top) and got.logprobs.shape == tokens.shape
    assert torch.equal(got.top_ids.cpu().view(ids.shape), ids)
    for name, a, b in (("logprobs", got.logprobs, lp), ("entropy", got.entropy, entropy), ("top", got.top_logprobs, values)):
        a, b = a.cpu().double().reshape(b.shape), b
        fine = torch.isfinite(b)
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()]), name
        tol = 2.0**-17 * b.abs().clamp(max=1.0) + 2.0**-23 * b.abs() + 2.0**-40
        assert bool(((a - b).abs() <= tol)[fine].all()), (name, float(((a - b).abs() / tol)[fine].max()))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,V,top", [(1, 1, 1), (3, 2, 5), (2, 7, 7), (5, 8, 3), (4, 9, 32), (1, 1000, 5), (3, 8193, 20), (70, 500, 1),
                                        (2, 51866, 5), (65, 9000, 4), (1, 66000, 32), (2, 150001, 8), (3, 40000, 0)])
def test_rows_and_vocabularies(cuda, dtype, rows, V, top):
    g = torch.Generator().manual_seed(V + rows)
    x = (2.5 * torch.randn(rows, V, generator=g)).to(dtype)
    tokens = torch.randint(0, V, (rows,), generator=g)
    check(cuda, x, tokens, top)
    if V > 8:
        blocked = torch.rand(rows, V + 3, generator=g) < 0.3  # wider than the rows
        check(cuda, x, tokens, top, blocked)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_logits_go_to_the_lowest_index(cuda, dtype):
    x = torch.zeros(4, 20000)
    x[1] = -3.0
    x[2, 5000:] = 2.0
    x[3, ::7] = 1.5
    x[0, 3] = -0.0
    got = check(cuda, x.to(dtype), torch.tensor([0, 19999, 4999, 7]), 20)
    assert got.top_ids[0].tolist() == list(range(20)) and got.top_ids[2].tolist() == list(range(5000, 5020))


def test_alternatives_that_one_thread_holds(cuda):
    """The largest logits next to each other, far apart in a thread's share, and falling or rising along the row."""
    V = 60000
    x = torch.zeros(5, V)
    x[0, 800:832] = torch.arange(32).float() + 1
    x[1, 16::8192] = torch.arange(len(range(16, V, 8192))).float() + 1
    x[2] = torch.arange(V).float() * 1e-3
    x[3] = -torch.arange(V).float() * 1e-3
    x[4, -3:] = 5.0
    check(cuda, x, torch.tensor([831, 16, V - 1, 0, V - 1]), 32)
    check(cuda, x[:, 1:].half(), torch.tensor([831, 16, V - 2, 0, V - 2]), 32)  # rows that begin at any element


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_little_or_nothing_left(cuda, dtype):
    V, inf, nan = 12000, float("inf"), float("nan")
    low = float(torch.finfo(dtype).min)
    x = torch.randn(9, V, generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0] = -inf
    x[1] = -inf
    x[1, 77] = 2.0
    x[2, 5] = nan
    x[3, 11999] = inf
    x[4] = low  # a mask of the type's lowest value, over all of the row
    x[5] = low
    x[5, 9] = 1.0
    x[6] = -low
    x[6, 100:] = low
    x[8, 3] = nan
    blocked = torch.zeros(9, V, dtype=torch.bool)
    blocked[7] = True
    blocked[8, 3] = True  # its NaN does not count
    tokens = torch.tensor([5, 77, 5, 7, 8, 9, 50, 3, 4])
    got = check(cuda, x, tokens, 3, blocked)
    assert got.entropy[0] == 0 and got.logprobs[0] == -inf and got.top_ids[0].tolist() == [-1] * 3
    assert got.logprobs[1] == 0 and got.top_ids[1].tolist() == [77, -1, -1] and got.top_ids[2].tolist() == [-1] * 3
    assert got.logprobs[7] == -inf and abs(float(got.entropy[4]) - math.log(V)) < 1e-4


def test_tokens_out_of_range_and_blocked(cuda):
    x = torch.randn(5, 300, generator=torch.Generator().manual_seed(2))
    blocked = torch.zeros(5, 300, dtype=torch.bool)
    blocked[3, 7] = True
    got = check(cuda, x, torch.tensor([-1, 300, 2**40, 7, 299]), 2, blocked)
    assert got.logprobs[:3].isnan().all() and got.logprobs[3] == -float("inf") and got.entropy.isfinite().all()


def test_small_log_sums_keep_their_digits(cuda):
    """One token far above the others: log p is about -1e-5, and as exact relative to itself."""
    x = torch.zeros(2, 5000)
    x[:, 17] = 20.0
    x[1, 4000] = 19.0
    check(cuda, x, torch.tensor([17, 17]), 2)
    got = w.token_logprobs(x.to(cuda), torch.tensor([17, 17], device=cuda))
    want = -math.log1p(4999 * math.exp(-20.0))
    assert abs(float(got.logprobs[0]) - want) <= 2.0**-17 * abs(want)


def test_shapes_strides_and_refusals(cuda):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 3, 100, generator=g).to(torch.bfloat16)
    tokens = torch.randint(0, 100, (2, 3), generator=g)
    a = check(cuda, x, tokens, 2)
    wide = torch.zeros(6, 140, dtype=torch.bfloat16, device=cuda)
    wide[:, 21:121] = x.view(6, 100).to(cuda)
    b = w.token_logprobs(wide[:, 21:121], tokens.view(6).to(cuda), 2)
    c = w.token_logprobs(x.to(cuda).transpose(0, 1), tokens.to(cuda).transpose(0, 1), 2)
    d = w.token_logprobs(x.to(cuda).permute(2, 0, 1).contiguous().permute(1, 2, 0), tokens.to(cuda), 2)
    for i in range(4):
        assert torch.equal(a[i].reshape(b[i].shape), b[i]) and torch.equal(a[i].transpose(0, 1), c[i]) and torch.equal(a[i], d[i])
    one = w.token_logprobs(x[0, 0].to(cuda), tokens[0, 0].to(cuda), 2)
    assert one.logprobs.shape == () and torch.equal(one.top_ids, a.top_ids[0, 0])
    assert w.token_logprobs(x[:0].to(cuda), tokens[:0].to(cuda), 2).top_ids.shape == (0, 3, 2)
    x, tokens = x.to(cuda), tokens.to(cuda)
    mask = torch.zeros(6, 100, dtype=torch.bool, device=cuda)
    for args, kw, err in (((x, tokens.int()), {}, ValueError), ((x, tokens[0]), {}, ValueError), ((x.long(), tokens), {}, TypeError),
                          ((x, tokens, 33), {}, NotImplementedError), ((x, tokens, -1), {}, NotImplementedError),
                          ((x[..., :0], tokens), {}, ValueError), ((x, tokens, 1), dict(blocked=mask[:5]), ValueError),
                          ((x, tokens, 1), dict(blocked=mask[:, :99]), ValueError), ((x, tokens, 1), dict(blocked=mask.int()), ValueError)):
        with pytest.raises(err):
            w.token_logprobs(*args, **kw)


def test_many_split_rows_run_in_launches(cuda):
    """More rows of a large vocabulary than there are counters; every row as it is alone."""
    x = torch.randn(4100, 70001, device=cuda, dtype=torch.bfloat16)
    tokens = torch.arange(4100, device=cuda)
    got = w.token_logprobs(x, tokens, 2)
    for r in (0, 1, 4095, 4096, 4099):
        check(cuda, x[r : r + 1].cpu(), tokens[r : r + 1].cpu(), 2)
        alone = w.token_logprobs(x[r : r + 1], tokens[r : r + 1], 2)
        assert torch.equal(got.top_ids[r], alone.top_ids[0]) and torch.allclose(got.logprobs[r], alone.logprobs[0], rtol=0, atol=1e-5)


def test_graphs_and_streams(cuda):
    xs = [torch.randn(3, 51866, device=cuda) for _ in range(3)]
    tokens = torch.tensor([1, 2, 3], device=cuda)
    want = [w.token_logprobs(x, tokens, 4) for x in xs]
    graphs, outs = [], []
    for x in xs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(w.token_logprobs(x, tokens, 4))
        graphs.append(g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(6):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
            eager = w.token_logprobs(xs[2], tokens, 4)
        torch.cuda.synchronize()
        for got, exp in zip((*outs, eager), want):
            assert all(torch.equal(a, b) for a, b in zip(got, exp))
