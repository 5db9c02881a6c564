"""PageTables.plan / truncate and FlashKVPages.write on the GPU against the restatement that serves one request and
one page at a time. Whole numbers: everything is equal."""
import random

import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import Tables

pytestmark = pytest.mark.gpu


def ids(cuda, x):
    return torch.tensor(x, dtype=torch.int32, device=cuda)


def assert_state(t, ref):
    held = [len(r) for r in ref.rows]
    assert t.page_counts.tolist() == held and t.seq_lens.tolist() == ref.lens
    assert t.free_pages[: int(t.n_free)].tolist() == ref.free
    want = torch.full(t.tables.shape, -1, dtype=torch.int32)
    for s, r in enumerate(ref.rows):
        want[s, : len(r)] = torch.tensor(r, dtype=torch.int32)
    assert torch.equal(t.tables.cpu(), want)


def assert_plan(plan, want):
    for name, got, exp in zip(plan._fields, plan, want):
        assert got.tolist() == list(exp), name


@pytest.mark.parametrize("seed,n_streams,page,max_len,n_pages", [
    (0, 1, 16, 16, 1), (1, 5, 16, 100, 20), (2, 40, 32, 448, 200), (3, 300, 16, 448, 4000), (4, 2500, 64, 200, 3000), (5, 7, 256, 3000, 60)])
def test_histories_of_plans_and_truncations(cuda, seed, n_streams, page, max_len, n_pages):
    rng = random.Random(seed)
    t, ref = w.PageTables(n_streams, n_pages, page, max_len, device=cuda), Tables(n_streams, n_pages, page, max_len)
    for step in range(8):
        B = rng.choice([n_streams, rng.randint(1, n_streams)])
        named = rng.sample(range(n_streams), B)
        if step % 3 == 2:  # some are no stream, some named twice
            named = [rng.choice([s, s, -1, n_streams, rng.choice(named)]) for s in named]
        new = [rng.choice([0, 1, 1, rng.randint(0, max(1, max_len // 3)), max_len + 5 if step % 4 == 3 else 2]) for _ in range(B)]
        total = max(0, sum(new) + rng.choice([0, 3, -2]))
        assert_plan(t.plan(ids(cuda, new), total, ids(cuda, named)), ref.plan(named, new, total))
        assert_state(t, ref)
        back = [rng.choice([0, n // 2, n, n + 1, -1]) for n in (ref.lens[s] if 0 <= s < n_streams else 0 for s in named)]
        t.truncate(ids(cuda, back), ids(cuda, named))
        ref.truncate(named, back)
        assert_state(t, ref)


@pytest.mark.parametrize("new", [0, 1, 17])
def test_every_stream_the_same(cuda, new):
    t, ref = w.PageTables(6, 12, 16, 48, device=cuda), Tables(6, 12, 16, 48)
    for _ in range(4):  # at 17 the pages run out for the last streams, then for all
        assert_plan(t.plan(new), ref.plan(range(6), [new] * 6, 6 * new))
        assert_state(t, ref)
    t.truncate(1)
    ref.truncate(range(6), [1] * 6)
    assert_state(t, ref)
    t.truncate(0)
    assert t.seq_lens.sum() == 0 and int(t.n_free) == 12 and sorted(t.free_pages.tolist()) == list(range(12))
    t.reset()
    assert t.free_pages.tolist() == list(range(11, -1, -1))


def test_a_plan_that_is_taken_back_leaves_the_state(cuda):
    t = w.PageTables(9, 64, 16, 100, device=cuda)
    t.plan(ids(cuda, [40, 3, 17]), 60, ids(cuda, [4, 8, 0]))
    before = [x.clone() for x in (t.tables, t.page_counts, t.seq_lens, t.free_pages, t.n_free)]
    lens = t.seq_lens.clone()
    order = ids(cuda, [8, 0, 5, 4])
    t.plan(ids(cuda, [20, 30, 16, 50]), 116, order)
    t.truncate(lens[order.long()], order)
    assert all(torch.equal(a, b) for a, b in zip(before, (t.tables, t.page_counts, t.seq_lens, t.free_pages, t.n_free)))


def test_no_requests_and_no_tokens(cuda):
    t = w.PageTables(4, 8, 16, 64, device=cuda)
    none = torch.zeros(0, dtype=torch.int32, device=cuda)
    plan = t.plan(none, 5, none)
    assert plan.cu_seqlens.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and plan.positions.tolist() == [0] * 5
    plan = t.plan(ids(cuda, [0, 0]), 0)
    assert plan.cu_seqlens.tolist() == [0, 0, 0] and plan.starts.tolist() == [0, 0] and plan.slots.numel() == 0
    t.truncate(none, none)


def test_large_numbers_stay_whole(cuda):
    """Counts whose sum leaves 32 bits, and one that reaches the longest stream."""
    big = 2**31 - 1
    t = w.PageTables(4, 8, 16, 64, device=cuda)
    plan = t.plan(ids(cuda, [big, big, 64, big]), 10)
    assert plan.cu_seqlens.tolist() == [0, 10, 10, 10, 10] and plan.starts.tolist() == [-1, -1, 0, -1] and int(t.n_free) == 4


def test_as_many_streams_as_there_may_be(cuda):
    n = w.PageTables.MAX_STREAMS
    t = w.PageTables(n, 3 * n, 16, 64, device=cuda)
    order = torch.randperm(n, device=cuda).to(torch.int32)
    new = (torch.arange(n, device=cuda) % 40).to(torch.int32)
    plan = t.plan(new, int(new.sum()), order)
    assert torch.equal(plan.starts, torch.zeros_like(new)) and torch.equal(t.seq_lens[order.long()], new)
    held = (new + 15) // 16
    assert torch.equal(t.page_counts[order.long()], held) and int(t.n_free) == 3 * n - int(held.sum())
    assert plan.slots.unique().numel() == plan.slots.numel() and bool((plan.slots >= 0).all())
    t.truncate(0, order)
    assert torch.equal(t.free_pages, torch.arange(3 * n - 1, -1, -1, dtype=torch.int32, device=cuda))


def test_ids_of_other_types_and_strides(cuda):
    t, ref = w.PageTables(8, 30, 16, 64, device=cuda), Tables(8, 30, 16, 64)
    streams = torch.tensor([5, 0, 3, 0, 1, 0], device=cuda)[::2]
    new = torch.tensor([3, 20, 33], dtype=torch.int64, device=cuda)
    assert_plan(t.plan(new, 56, streams), ref.plan([5, 3, 1], [3, 20, 33], 56))
    assert_state(t, ref)
    with pytest.raises(TypeError):
        t.plan(new.float(), 56, streams)
    with pytest.raises(ValueError):
        t.plan(new, None, streams)
    with pytest.raises(ValueError):
        t.plan(new[:2], 23, streams)
    with pytest.raises(ValueError):
        t.plan(torch.ones(9, dtype=torch.int32, device=cuda), 9)


def test_captured_plans_advance_the_state(cuda):
    t, ref = w.PageTables(5, 20, 16, 64, device=cuda), Tables(5, 20, 16, 64)
    order, new = ids(cuda, [3, 1, 4]), ids(cuda, [7, 9, 2])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        t.plan(new, 18, order)
        t.truncate(0, order)
    side.synchronize()
    t.reset()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan = t.plan(new, 18, order)
    for i in range(5):
        if i == 3:
            new.copy_(ids(cuda, [20, 0, 16]))
        g.replay()
        assert_plan(plan, ref.plan([3, 1, 4], new.tolist(), 18))
        assert_state(t, ref)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,heads,dim,page", [(1, 1, 64, 16), (7, 3, 128, 64), (300, 20, 64, 32), (2000, 2, 128, 256)])
def test_writes(cuda, dtype, T, heads, dim, page):
    g = torch.Generator(device=cuda).manual_seed(T)
    n_pages = -(-T // page) + 3
    cache = w.FlashKVPages(w.PageTables(2, n_pages, page, 4096, device=cuda), heads, dim, dtype)
    x = torch.randn(T, 3 * heads, dim, generator=g, device=cuda).to(dtype)
    k, v = x[:, heads : 2 * heads], x[:, 2 * heads :]
    slots = torch.randperm(n_pages * page, generator=g, device=cuda)[:T]
    slots[:: 5] = torch.where(torch.arange(slots[::5].numel(), device=cuda) % 2 == 0, -1, n_pages * page)  # no slots
    cache.k_pages.normal_(generator=g), cache.v_pages.normal_(generator=g)
    want = [cache.k_pages.clone(), cache.v_pages.clone()]
    ok = (slots >= 0) & (slots < n_pages * page)
    for y, src in zip(want, (k, v)):
        y[slots[ok] // page, :, slots[ok] % page] = src[ok]
    cache.write(k, v, slots)
    assert torch.equal(cache.k_pages, want[0]) and torch.equal(cache.v_pages, want[1])
    cache.write(k[:0], v[:0], slots[:0])
    for bad, err in (((k[:, :, :32], v[:, :, :32], slots), ValueError), ((k.float(), v.float(), slots), TypeError),
                     ((k, v, slots.int()), ValueError), ((k, v, slots[:-1]), ValueError), ((k[0], v[0], slots), ValueError)):
        with pytest.raises(err):
            cache.write(*bad)
