"""The paged cache, packed attention and token log probabilities where numbers get large: byte offsets beyond 32 bits, sums
of pages beyond 31, probabilities far below a row's largest, keys and rows that share memory."""
import math

import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import Tables, attention, logprobs
from whisperdrz_amd.decoder import TextDecoderStack

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def ids(cuda, x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=cuda)


def test_sums_of_pages_beyond_31_bits(cuda):
    """2048 requests of 2^20 pages each, none of which can be served; one of a single page behind them neither: the pages
    before it do not suffice. Alone it is."""
    n = 2049
    t = w.PageTables(n, 100, 16, 1 << 24, device=cuda)
    new = torch.full((n,), 1 << 24, dtype=torch.int32, device=cuda)
    new[-1] = 1
    plan = t.plan(new, 10)
    assert bool((plan.starts == -1).all()) and bool((t.seq_lens == 0).all()) and int(t.n_free) == 100
    assert plan.cu_seqlens.tolist() == [0] + [10] * n and plan.slots.tolist() == [-1] * 10
    assert t.plan(ids(cuda, [1]), 1, ids(cuda, [n - 1])).slots.tolist() == [0] and int(t.n_free) == 99


@pytest.mark.parametrize("heads,dim", [(8, 64), (4, 128)])
def test_pages_beyond_32_bit_offsets(cuda, heads, dim):
    """The last pages of 2^19 of 16 KB: elements from 2^32 on. Written by slots and by steps, read by both."""
    n = (1 << 19) + 64
    t = w.PageTables(3, n, 16, 600, device=cuda)
    t.free_pages.copy_(torch.arange(n, dtype=torch.int32))  # the last page goes first
    cache = w.FlashKVPages(t, heads, dim, BF16)
    assert cache.k_pages.numel() > 1 << 32
    g = torch.Generator().manual_seed(dim)
    lens = [50, 0, 579]
    q, k, v = (torch.randn(sum(lens), heads, dim, generator=g).to(BF16).to(cuda) for _ in range(3))
    plan = t.plan(ids(cuda, lens), sum(lens), ids(cuda, [0, 1, 2]))
    assert int(plan.slots.min()) >= (1 << 19) * 16
    cache.write(k, v, plan.slots)
    packed = w.packed_attention(q, k, v, plan.cu_seqlens)
    q1, k1, v1 = (torch.randn(3, 1, heads, dim, generator=g).to(BF16).to(cuda) for _ in range(3))
    step = t.plan(1, 3, ids(cuda, [0, 1, 2]))
    got = w.flash_attn_with_kvpages(q1, cache, k1, v1, cache_seqlens=step.starts, cache_batch_idx=ids(cuda, [0, 1, 2]))
    a = 0
    for b, m in enumerate(lens):
        K, V = torch.cat([k[a : a + m], k1[b]]).cpu(), torch.cat([v[a : a + m], v1[b]]).cpu()
        want, big = attention(q1[b].cpu(), K, V, [m + 1], dim**-0.5)
        d = (dim + 4) * 2.0**-24 * dim**-0.5 * big
        tol = 2.0**-8 * want.abs() + (2 * d + 2.0**-16) * float(V.float().abs().max()) + 1e-7
        assert bool(((got[b].double().cpu() - want).abs() <= tol).all())
        if m:  # the last token's prompt form sees the same keys
            want, big = attention(q[a + m - 1 : a + m].cpu(), K[:m], V[:m], [m], dim**-0.5)
            tol = 2.0**-8 * want.abs() + (2 * d + 2.0**-20 + 2.0**-8) * float(V.float().abs().max()) + 1e-7
            assert bool(((packed[a + m - 1 : a + m].double().cpu() - want).abs() <= tol).all())
        a += m


def test_rows_far_apart(cuda):
    """Strides that take offsets beyond 32 bits: rows of queries, keys and logits."""
    g = torch.Generator().manual_seed(1)
    T, far = 300, 1 << 23  # 2^23 elements a row: 4.7 GiB
    big = torch.zeros(T * far, dtype=BF16, device=cuda)
    x = big.as_strided((T, 3, 64), (far, 64, 1))
    x.copy_(torch.randn(T, 3, 64, generator=g))
    cu = ids(cuda, [0, 40, T])
    got = w.packed_attention(x[:, :1], x[:, 1:2], x[:, 2:], cu)
    y = x.contiguous()
    assert torch.equal(got, w.packed_attention(y[:, :1], y[:, 1:2], y[:, 2:], cu))
    out = big.as_strided((T, 1, 64), (far, 64, 1), 1024)
    w.packed_attention(y[:, :1], y[:, 1:2], y[:, 2:], cu, out=out)
    assert torch.equal(out, got)
    rows = big.as_strided((2, 1000), ((T - 1) * far, 1))
    rows.copy_(torch.randn(2, 1000, generator=g))
    tokens = ids(cuda, [3, 999], torch.int64)
    for a, b in zip(w.token_logprobs(rows, tokens, 4), w.token_logprobs(rows.contiguous(), tokens, 4)):
        assert torch.equal(a, b)


def test_keys_that_share_a_row(cuda):
    """Expanded keys and values (a row stride of 0): every key weighs the same, the result is the one row's value."""
    g = torch.Generator().manual_seed(2)
    for dim in (64, 128):
        q = torch.randn(130, 4, dim, generator=g).to(BF16).to(cuda)
        k, v = (torch.randn(1, 2, dim, generator=g).to(BF16).to(cuda).expand(130, 2, dim) for _ in range(2))
        got = w.packed_attention(q, k, v, ids(cuda, [0, 1, 70, 130]))
        want = v.repeat_interleave(2, 1).double()
        # weights of 1 / n in 16 bits, which sum to n (1 + e) / n with e the one rounding that all of them share
        assert bool(((got.double() - want).abs() <= 2 * 2.0**-8 * want.abs()).all())


@pytest.mark.parametrize("order", ["first", "last"])
@pytest.mark.parametrize("op", ["packed", "pages"])
def test_many_small_probabilities_beside_a_large_one(cuda, op, order):
    """One key with probability 1 and value 0, thousands at 1.5 x 2^-24, which is between two fp16 numbers, with values of 1:
    the result is their sum. Values are not negative, so the error is relative: half a step of the result and half a
    step of the probability in fp16 (2^-11 each), 2^-20 of the exponential, scores off by (D + 4) 2^-24 x 24 and so
    twice that; results are above 2^-14, where fp16 has all digits."""
    n, dim = 8192, 64
    q = torch.ones(1, 1, dim, dtype=FP16)
    k = torch.full((n, 1, dim), (math.log2(1.5) - 24) * math.log(2) / dim).to(FP16)
    v = torch.ones(n, 1, dim, dtype=FP16)
    at = 0 if order == "first" else n - 1
    k[at], v[at] = 0, 0
    want, _ = attention(q, k, v, [n], 1.0)
    assert float(want.min()) > 2.0**-14
    q, k, v = q.to(cuda), k.to(cuda), v.to(cuda)
    if op == "packed":
        got = w.packed_attention(q, k, v, ids(cuda, [0, 1]), ids(cuda, [0, n]), scale=1.0)
    else:
        t = w.PageTables(1, n // 16, 16, n, device=cuda)
        cache = w.FlashKVPages(t, 1, dim, FP16)
        cache.write(k, v, t.plan(n).slots)
        got = w.flash_attn_with_kvpages(q[None], cache, cache_seqlens=t.seq_lens, softmax_scale=1.0)[0]
    err = ((got.double().cpu() - want).abs() / want).max()
    assert float(err) <= 2 * 2.0**-11 + 2.0**-20 + 2 * (dim + 4) * 24 * 2.0**-24, float(err)


def test_a_pool_longer_than_the_decoder_is_refused(cuda):
    stack = TextDecoderStack(100, 32, 128, 2, 1).to(cuda).to(BF16)
    pool = w.KVPagePool(1, 2, 8, 2, 64, 64, 10, BF16, cuda)
    with pytest.raises(ValueError, match="positions"):
        stack.prefill_packed(ids(cuda, [1, 2], torch.int64), ids(cuda, [1, 1]), torch.zeros(2, 10, 128, device=cuda, dtype=BF16), pool,
                             ids(cuda, [0, 1], torch.int64))


def test_captured_workspaces_are_cleared_by_replays(cuda):
    """Split rows and split logits in one graph, replayed over other inputs with eager calls between: every replay equals the
    eager result."""
    g = torch.Generator().manual_seed(3)
    t = w.PageTables(2, 400, 16, 3000, device=cuda)
    cache = w.FlashKVPages(t, 2, 64, BF16)
    x = torch.randn(5800, 2, 64, generator=g).to(BF16).to(cuda)
    cache.write(x, x, t.plan(2900).slots)
    q, logits = torch.zeros(2, 1, 2, 64, dtype=BF16, device=cuda), torch.zeros(2, 20000, device=cuda)
    tokens = ids(cuda, [5, 19999], torch.int64)
    run = lambda: (w.flash_attn_with_kvpages(q, cache, cache_seqlens=t.seq_lens), *w.token_logprobs(logits, tokens, 3))
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g))
        logits.copy_(torch.randn(logits.shape, generator=g))
        want = [o.clone() for o in run()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i
    want = logprobs(logits.cpu(), tokens.cpu(), 3)
    assert torch.equal(outs[4].cpu(), want[3])


@pytest.mark.parametrize("lens", [[33000, 0, 17, 33000], [40] * 300 + [9000] + [3] * 1500, [5000] * 20])
def test_requests_of_many_pages(cuda, lens):
    """Long and short requests in one call, taken and given back in part and whole, with a request in between that finds no
    pages; equal to the restatement that moves a page at a time."""
    n, most = len(lens), max(lens)
    pages = sum(-(-x // 16) for x in lens) - 2
    t, ref = w.PageTables(n, pages, 16, most, device=cuda), Tables(n, pages, 16, most)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(n)).tolist()
    streams = ids(cuda, order)
    for new, back in ((lens, [x // 3 for x in lens]), ([x - x // 3 for x in lens], [0] * n)):
        got, want = t.plan(ids(cuda, new), sum(new), streams), ref.plan(order, new, sum(new))
        for a, b in zip(got, want):
            assert a.tolist() == list(b)
        t.truncate(ids(cuda, back), streams)
        ref.truncate(order, back)
        assert t.free_pages[: int(t.n_free)].tolist() == ref.free and t.seq_lens.tolist() == ref.lens
        for row, held in zip(t.tables.tolist(), ref.rows):
            assert row[: len(held)] == held and set(row[len(held):]) <= {-1}
