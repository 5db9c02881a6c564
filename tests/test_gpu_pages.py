"""flash_attn_with_kvpages on the GPU against the 64-bit restatement.

Tolerance: half a step of the output type of the value; the probabilities' relative error times the largest value
they weigh. That error is 2 d + 2^-16: a score is off by at most d = (D + 4) 2^-24 scale max(sum |q| |k|) (fp32 sums of
exact products, a product with the scale, a difference), in the sum over the keys and in the weight, and the
probabilities are two 16-bit parts with 2^-17 or less behind, 2^-21 of the exponential beside them."""
import random

import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import attention

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def make(cuda, seed, dtype, B, heads, dim, page, max_len, lens, sq, spare=2):
    """A cache in use: rows of streams in any order, pages in any order, stale values everywhere else."""
    g = torch.Generator().manual_seed(seed)
    n = B + 2
    streams = torch.randperm(n, generator=g)[:B]
    held = [-(-(x + sq) // page) for x in lens]
    n_pages = sum(held) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    tables = w.PageTables(n, n_pages, page, max_len, device=cuda)
    at = 0
    host = torch.full(tables.tables.shape, -1, dtype=torch.int32)
    for s, h in zip(streams.tolist(), held):
        host[s, :h] = torch.tensor(order[at : at + h], dtype=torch.int32)
        at += h
    tables.tables.copy_(host)
    cache = w.FlashKVPages(tables, heads, dim, dtype)
    for x in (cache.k_pages, cache.v_pages):
        x.copy_(torch.randn(x.shape, generator=g).to(dtype))
    return cache, streams, g


def rows_of(cache, pages, stream, n):
    """Positions 0 .. n - 1 of a stream: [n, heads, dim]."""
    page = cache.page_tables.page_size
    at = cache.page_tables.tables[stream].cpu()[: -(-n // page)].long()
    return pages.cpu()[at].transpose(1, 2).reshape(-1, cache.n_heads, cache.head_dim)[:n]


def want_rows(cache, streams, lens, q, k=None, v=None):
    out, big = [], 0.0
    for b, (s, n) in enumerate(zip(streams.tolist(), lens)):
        K, V = (rows_of(cache, p, s, n) for p in (cache.k_pages, cache.v_pages))
        limit = [n] * q.shape[1]
        if k is not None:
            K, V = torch.cat([K, k[b].cpu()]), torch.cat([V, v[b].cpu()])
            limit = [n + t + 1 for t in range(q.shape[1])]
        o, m = attention(q[b].cpu(), K, V, limit, q.shape[-1] ** -0.5)
        out.append(o)
        big = max(big, m)
    return torch.stack(out), big


def assert_near(got, want, big, vmax, dtype, dim):
    d = (dim + 4) * 2.0**-24 * dim**-0.5 * big
    tol = torch.finfo(dtype).eps / 2 * want.abs() + (2 * d + 2.0**-16) * vmax + 1e-7
    err = (got.double().cpu() - want).abs()
    assert torch.isfinite(got).all() and bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of the tolerance"


def run_case(cuda, seed, dtype, lens, sq, H, Hk, dim, page, append, max_len=None):
    B = len(lens)
    print(f"pages seed={seed} {dtype} lens={lens[:8]} sq={sq} H={H}/{Hk} D={dim} page={page} append={append}", flush=True)
    max_len = max_len or max(max(lens) + sq, 1)
    cache, streams, g = make(cuda, seed, dtype, B, Hk, dim, page, max_len, lens, sq if append else 0)
    qkv = torch.randn(B, sq, H + 2 * Hk, dim, generator=g).to(dtype).to(cuda)
    q, k, v = qkv[:, :, :H], qkv[:, :, H : H + Hk], qkv[:, :, H + Hk :]
    before = [x.clone() for x in (cache.k_pages, cache.v_pages)]
    new = (k, v) if append else (None, None)
    want, big = want_rows(cache, streams, lens, q, *new)
    got = w.flash_attn_with_kvpages(q, cache, *new, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda),
                                    cache_batch_idx=streams.to(cuda))
    vmax = max(float(cache.v_pages.abs().max()), float(v.abs().max()))
    assert_near(got, want, big, vmax, dtype, dim)
    if append:  # the rows stand in their pages, and nothing else has changed
        for b, (s, n) in enumerate(zip(streams.tolist(), lens)):
            for t in range(sq):
                p = cache.page_tables.tables[s, (n + t) // page].item()
                before[0][p, :, (n + t) % page], before[1][p, :, (n + t) % page] = k[b, t], v[b, t]
    assert torch.equal(before[0], cache.k_pages) and torch.equal(before[1], cache.v_pages)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,Hk,dim", [(1, 1, 64), (4, 4, 64), (6, 2, 64), (8, 1, 128), (4, 2, 128), (40, 2, 64)])
@pytest.mark.parametrize("sq,append", [(1, True), (1, False), (5, True), (3, False)])
def test_heads_and_tokens(cuda, dtype, H, Hk, dim, sq, append):
    run_case(cuda, H + sq, dtype, [0, 1, 15, 16, 31, 33, 100], sq, H, Hk, dim, 16, append)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("sq", [1, 4])
def test_page_sizes_and_their_edges(cuda, page, sq):
    run_case(cuda, page, BF16, [page - 1, page, page + 1, 2 * page - sq, 3 * page + 7], sq, 2, 2, 64, page, True)
    run_case(cuda, page, FP16, [page - 1, page, page + 1, 2 * page, 0], sq, 4, 2, 128, page, False)


@pytest.mark.parametrize("sq,H,Hk", [(1, 64, 1), (17, 2, 2), (40, 4, 1), (9, 16, 4), (33, 3, 3)])
def test_rows_over_several_tiles(cuda, sq, H, Hk):
    run_case(cuda, sq, BF16, [0, 5, 50, 200], sq, H, Hk, 64, 16, True)
    run_case(cuda, sq, FP16, [0, 64], sq, H, Hk, 128, 32, False)


@pytest.mark.parametrize("max_len,lens", [(1025, [1024, 3, 511, 512]), (5000, [4999, 1, 0, 513, 2048]), (40000, [33000]), (40000, [700, 20000])])
@pytest.mark.parametrize("H,Hk,dim", [(2, 2, 64), (8, 2, 128)])
def test_long_rows_are_split_and_joined(cuda, max_len, lens, H, Hk, dim):
    assert w.kvpages_workspace_size(len(lens), 1, H, Hk, dim, max_len) > 0
    run_case(cuda, max_len, BF16, lens, 1, H, Hk, dim, 64, True, max_len + 8)
    run_case(cuda, max_len, FP16, lens, 3, H, Hk, dim, 16, False, max_len)


def test_many_rows(cuda):
    rng = random.Random(3)
    run_case(cuda, 3, BF16, [rng.randint(0, 60) for _ in range(150)], 1, 2, 2, 64, 16, True)


def test_scores_far_apart_move_the_reference(cuda):
    """Keys that grow along the row: the softmax reference moves block by block, in one workgroup and over splits."""
    for max_len in (300, 3000):
        cache, streams, g = make(cuda, 1, FP16, 2, 2, 64, 16, max_len, [290, max_len - 2], 0)
        q = torch.randn(2, 1, 2, 64, generator=g).to(FP16).to(cuda)
        at = cache.page_tables.tables[streams[1]].long()
        for j in range(-(-(max_len - 2) // 16)):
            cache.k_pages[at[j]] = (q[1, 0][:, None] * (j % 19) * 0.5).expand(2, 16, 64)
        lens = [290, max_len - 2]
        want, big = want_rows(cache, streams, lens, q)
        got = w.flash_attn_with_kvpages(q, cache, cache_seqlens=torch.tensor(lens, device=cuda), cache_batch_idx=streams.to(cuda))
        assert_near(got, want, big, float(cache.v_pages.abs().max()), FP16, 64)


@pytest.mark.parametrize("sq", [1, 5])
@pytest.mark.parametrize("odd", [float("nan"), float("inf")])
def test_what_nobody_sees_does_not_count(cuda, sq, odd):
    """Stale rows of pages, the rows of other streams and a draft's later tokens may hold anything."""
    lens, H = [20, 0, 45], 2
    cache, streams, g = make(cuda, 2, BF16, 3, H, 64, 16, 64, lens, sq)
    keep = torch.zeros(cache.k_pages.shape[0], 1, 16, 1, dtype=torch.bool)
    for s, n in zip(streams.tolist(), lens):
        for p in range(n):
            keep[cache.page_tables.tables[s, p // 16].item(), 0, p % 16] = True
    for x in (cache.k_pages, cache.v_pages):
        x.masked_fill_(~keep.to(cuda), odd)
    q, k, v = (torch.randn(3, sq, H, 64, generator=g).to(BF16).to(cuda) for _ in range(3))
    if sq > 1:
        k[0, 3], v[0, 3] = odd, odd  # row 0's queries 3 and 4 see it, its first three do not
    want, big = want_rows(cache, streams, lens, q[:, :3], k[:, :3], v[:, :3])
    got = w.flash_attn_with_kvpages(q, cache, k, v, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=cuda), cache_batch_idx=streams.to(cuda))
    assert_near(got[:, :3], want, big, 8.0, BF16, 64)
    if sq > 1:
        assert got[0, 3:].isnan().all() and got[1:].isfinite().all()


def test_streams_lengths_and_pages_out_of_range(cuda):
    """NaN rows that write nothing; the other rows are served."""
    lens = [20, 30, 10, 40, 5, 6, 60]
    cache, streams, g = make(cuda, 4, FP16, 7, 2, 64, 16, 64, lens, 1)
    q, k, v = (torch.randn(7, 1, 2, 64, generator=g).to(FP16).to(cuda) for _ in range(3))
    names, at = streams.to(torch.int32), torch.tensor(lens, dtype=torch.int32)
    names[0] = -1
    at[1] = -1
    names[2] = 9
    at[3] = 64  # no room for another
    names[5] = names[4]  # two rows append to one stream
    want, big = want_rows(cache, streams[6:], lens[6:], q[6:], k[6:], v[6:])
    before = cache.k_pages.clone()
    got = w.flash_attn_with_kvpages(q, cache, k, v, cache_seqlens=at.to(cuda), cache_batch_idx=names.to(cuda))
    assert got[:6].isnan().all()
    assert_near(got[6:], want, big, 8.0, FP16, 64)
    page = cache.page_tables.tables[streams[6], 60 // 16].item()
    before[page, :, 60 % 16] = k[6, 0]
    assert torch.equal(before, cache.k_pages)
    cache.page_tables.tables[streams[6], 1] = cache.page_tables.n_pages  # no page
    got = w.flash_attn_with_kvpages(q[6:], cache, k[6:], v[6:], cache_seqlens=at[6:].to(cuda), cache_batch_idx=names[6:].to(cuda))
    assert got.isnan().all()
    # without an append the same stream may be read by several rows
    same = torch.full((3,), int(streams[0]), dtype=torch.int32, device=cuda)
    got = w.flash_attn_with_kvpages(q[:1].expand(3, -1, -1, -1), cache, cache_seqlens=torch.tensor([20, 20, 20], device=cuda), cache_batch_idx=same)
    assert got.isfinite().all() and torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_outputs_workspaces_and_identity(cuda):
    lens = [1500, 1200]
    cache, streams, g = make(cuda, 6, BF16, 2, 2, 64, 16, 1600, lens, 1)
    q, k, v = (torch.randn(2, 1, 2, 64, generator=g).to(BF16).to(cuda) for _ in range(3))
    at = torch.tensor(lens, dtype=torch.int32, device=cuda)
    call = lambda **kw: w.flash_attn_with_kvpages(q, cache, k, v, cache_seqlens=at, cache_batch_idx=streams.to(cuda), **kw)
    want = call()
    out = torch.empty(2, 1, 4, 64, dtype=BF16, device=cuda)[:, :, ::2]
    ws = torch.zeros(w.kvpages_workspace_size(2, 1, 2, 2, 64, 1600), dtype=torch.uint8, device=cuda)
    for _ in range(3):  # the counters are back at zero
        assert torch.equal(call(out=out, workspace=ws), want) and torch.equal(out, want)
    with pytest.raises(ValueError):
        call(workspace=ws[:-4])
    n = int(cache.page_tables.n_streams)
    everyone = torch.zeros(n, dtype=torch.int32, device=cuda)
    everyone[streams.to(cuda)] = at
    every = w.flash_attn_with_kvpages(torch.zeros(n, 1, 2, 64, dtype=BF16, device=cuda).index_copy(0, streams.to(cuda), q), cache, cache_seqlens=everyone)
    row = w.flash_attn_with_kvpages(q, cache, cache_seqlens=at, cache_batch_idx=streams.to(cuda))
    assert torch.equal(every[streams.to(cuda)], row)
    assert torch.equal(every[[i for i in range(n) if i not in streams.tolist()]], torch.zeros(2, 1, 2, 64, dtype=BF16, device=cuda))
    assert w.flash_attn_with_kvpages(q[:0], cache, cache_seqlens=at[:0]).shape == (0, 1, 2, 64)
    for kw, err in ((dict(k=k), ValueError), (dict(cache_seqlens=None), ValueError), (dict(q=q[0]), ValueError), (dict(q=q.half()), TypeError),
                    (dict(q=torch.cat([q, q[:, :, :1]], 2)), ValueError), (dict(k=k[:1], v=v[:1]), ValueError),
                    (dict(cache_seqlens=at[:1]), ValueError), (dict(out=out[:, :, :1]), ValueError)):
        a = dict(q=q, k=None, v=None, cache_seqlens=at, cache_batch_idx=None)
        a.update(kw)
        out_kw = {"out": a.pop("out")} if "out" in a else {}
        with pytest.raises(err):
            w.flash_attn_with_kvpages(a["q"], cache, a["k"], a["v"], cache_seqlens=a["cache_seqlens"], **out_kw)


def test_streams_and_graphs_share_nothing(cuda):
    """Two graphs of split calls captured on one stream, replayed beside each other and beside eager calls."""
    lens = [3000, 2800]
    cache, streams, g = make(cuda, 8, BF16, 2, 2, 128, 32, 3100, lens, 0)
    at, names = torch.tensor(lens, dtype=torch.int32, device=cuda), streams.to(torch.int32).to(cuda)
    qs = [torch.randn(2, 1, 4, 128, generator=g).to(BF16).to(cuda) for _ in range(3)]
    call = lambda q: w.flash_attn_with_kvpages(q, cache, cache_seqlens=at, cache_batch_idx=names)
    want = [call(q) for q in qs]
    graphs, outs = [], []
    for q in qs[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(q))
        graphs.append(gr)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(6):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
            eager = call(qs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
