"""Refusals of the paged cache, the packed attention and the token log probabilities that need no GPU: bad sizes,
strides, pointers and types come back as codes with a message before any launch, and as exceptions from Python."""
import ctypes

import pytest
import torch

import whisperdrz_amd as w
from whisperdrz_amd import _lib

FAKE = 0x10000  # a 16-byte aligned address that nothing reads: every call here is refused first
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def tables(**over):
    a = dict(tables=FAKE, page_counts=FAKE, seq_lens=FAKE, free_pages=FAKE, n_free=FAKE, n_streams=8, n_pages=100,
             page_size=16, max_pages=28, max_seq=448)
    a.update(over)
    return _lib.PageTables(*a.values())


def pages(**over):
    a = dict(k_pages=FAKE, v_pages=FAKE, n_pages=100, n_heads=4, page_size=16, head_dim=64)
    a.update(over)
    return _lib.KvPages(*a.values())


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def check(lib, rc, code, msg):
    text = lib.wdrz_last_error().decode()
    assert rc == code and msg in text, (rc, text)


BAD_TABLES = [
    (dict(tables=None), INVALID, "NULL"), (dict(n_free=None), INVALID, "NULL"), (dict(page_size=24), UNSUPPORTED, "page_size"),
    (dict(page_size=8), UNSUPPORTED, "page_size"), (dict(page_size=512), UNSUPPORTED, "page_size"),
    (dict(n_streams=0), INVALID, "sizes"), (dict(n_pages=0), INVALID, "sizes"), (dict(max_seq=449), INVALID, "sizes"),
    (dict(n_streams=12289), UNSUPPORTED, "too large"), (dict(n_pages=(1 << 26) + 1), UNSUPPORTED, "too large"),
]


@pytest.mark.parametrize("over,code,msg", BAD_TABLES)
def test_tables_are_checked_by_plan_and_truncate(lib, over, code, msg):
    t = tables(**over)
    check(lib, lib.wdrz_page_plan(t, FAKE, 0, FAKE, FAKE, FAKE, FAKE, FAKE, 4, 10, None), code, msg)
    check(lib, lib.wdrz_page_truncate(t, FAKE, 0, FAKE, 4, None), code, msg)


@pytest.mark.parametrize("over,code,msg", [
    (dict(B=-1), INVALID, "sizes"), (dict(B=65536), UNSUPPORTED, "too large"), (dict(total=-1), INVALID, "total"),
    (dict(total=(1 << 28) + 1), UNSUPPORTED, "too large"), (dict(cu=None), INVALID, "NULL"), (dict(slots=None), INVALID, "NULL"),
    (dict(lens=None, all=449), INVALID, "outside"), (dict(lens=None, all=-1), INVALID, "outside"),
    (dict(streams=None, B=9), INVALID, "exceed"), (dict(pages=None), INVALID, "NULL"),
])
def test_plan_requests_are_checked(lib, over, code, msg):
    a = dict(pages=tables(), lens=FAKE, all=0, streams=FAKE, cu=FAKE, starts=FAKE, slots=FAKE, positions=FAKE, B=4, total=10)
    a.update(over)
    check(lib, lib.wdrz_page_plan(*a.values(), None), code, msg)


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=0), UNSUPPORTED, "dtype"), (dict(dtype=9), INVALID, "dtype"), (dict(cache=pages(head_dim=96)), UNSUPPORTED, "head_dim"),
    (dict(cache=pages(page_size=48)), UNSUPPORTED, "page_size"), (dict(cache=pages(k_pages=FAKE + 8)), INVALID, "aligned"),
    (dict(cache=pages(n_heads=0)), INVALID, "sizes"), (dict(ks=strides(256, 60, 1)), INVALID, "aligned"),
    (dict(vs=strides(256, 64, 2)), INVALID, "head_dim stride"), (dict(slots=None), INVALID, "NULL"), (dict(T=-1), INVALID, "sizes"),
    (dict(k=None), INVALID, "k is NULL"),
])
def test_writes_are_checked(lib, over, code, msg):
    a = dict(dtype=2, cache=pages(), k=FAKE, ks=strides(256, 64, 1), v=FAKE, vs=strides(256, 64, 1), slots=FAKE, T=5)
    a.update(over)
    check(lib, lib.wdrz_page_write(*a.values(), None), code, msg)


Q4 = strides(256, 256, 64, 1)


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=0), UNSUPPORTED, "dtype"), (dict(cache=pages(page_size=32)), INVALID, "pages of"), (dict(cache=pages(n_pages=99)), INVALID, "pages of"),
    (dict(pages=tables(page_size=20)), UNSUPPORTED, "page_size"), (dict(H=6), INVALID, "multiple"), (dict(H=0), INVALID, "sizes"),
    (dict(sq=0), INVALID, "sizes"), (dict(sq=65537), UNSUPPORTED, "too large"), (dict(scale=0.0), INVALID, "softmax_scale"),
    (dict(scale=float("nan")), INVALID, "softmax_scale"), (dict(v=None), INVALID, "together"), (dict(lens=None), INVALID, "cache_seqlens"),
    (dict(streams=None, B=9), INVALID, "exceed"), (dict(q=FAKE + 4), INVALID, "aligned"), (dict(qs=strides(256, 256, 64, 2)), INVALID, "stride"),
    (dict(os=strides(256, 250, 64, 1)), INVALID, "aligned"), (dict(ks=strides(255, 256, 64, 1)), INVALID, "aligned"),
    (dict(pages=tables(max_pages=4096, max_seq=65536)), WORKSPACE, "workspace"),
    (dict(pages=tables(max_pages=4096, max_seq=65536), ws=FAKE + 16, nbytes=1 << 30), INVALID, "256-byte"),
])
def test_attention_over_pages_is_checked(lib, over, code, msg):
    a = dict(dtype=2, cache=pages(), pages=tables(), q=FAKE, qs=Q4, k=FAKE, ks=Q4, v=FAKE, vs=Q4, lens=FAKE, streams=FAKE, o=FAKE, os=Q4,
             B=2, sq=1, H=4, scale=0.125, ws=None, nbytes=0)
    a.update(over)
    check(lib, lib.wdrz_attn_kvpages(*a.values(), None), code, msg)


def test_the_workspace_covers_the_plan(lib):
    for B in (1, 2, 4, 33, 500):
        for sq, H, Hk, D in ((1, 20, 20, 64), (5, 20, 20, 64), (1, 32, 8, 128), (40, 8, 1, 128)):
            last = 0
            for L in (1, 448, 1024, 1025, 4096, 32768, 1 << 20):
                n = lib.wdrz_attn_kvpages_workspace_size(B, sq, H, Hk, D, L)
                assert n == 0 or n > 16384 and n % 4 == 0
                assert L > 512 or n == 0  # such rows are not split
                last = max(last, n)
            assert last < 1 << 31
    assert lib.wdrz_attn_kvpages_workspace_size(0, 1, 4, 4, 64, 100) == 0
    assert lib.wdrz_attn_kvpages_workspace_size(1, 1, 4, 3, 64, 100) == 0


R3 = strides(256, 64, 1)


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=0), UNSUPPORTED, "dtype"), (dict(D=32), UNSUPPORTED, "head_dim"), (dict(T=-1), INVALID, "sizes"), (dict(Hk=3), INVALID, "multiple"),
    (dict(Hk=0), INVALID, "sizes"), (dict(cu=None), INVALID, "cu_seqlens"), (dict(cu_k=None, Tk=9), INVALID, "keys"), (dict(B=65536), UNSUPPORTED, "large"),
    (dict(T=(1 << 24) + 1, Tk=(1 << 24) + 1), UNSUPPORTED, "large"), (dict(scale=-1.0), INVALID, "scale"), (dict(q=None), INVALID, "q is NULL"),
    (dict(k=FAKE + 2), INVALID, "aligned"), (dict(vs=strides(250, 64, 1)), INVALID, "aligned"), (dict(os=strides(256, 64, 3)), INVALID, "stride"),
])
def test_packed_attention_is_checked(lib, over, code, msg):
    a = dict(dtype=1, q=FAKE, qs=R3, k=FAKE, ks=R3, v=FAKE, vs=R3, o=FAKE, os=R3, cu=FAKE, cu_k=FAKE, B=2, T=8, Tk=8, H=4, Hk=4, D=64,
             scale=0.125, causal=1)
    a.update(over)
    check(lib, lib.wdrz_attn_packed(*a.values(), None), code, msg)


@pytest.mark.parametrize("over,code,msg", [
    (dict(dtype=3), INVALID, "dtype"), (dict(V=0), INVALID, "sizes"), (dict(V=(1 << 20) + 1), UNSUPPORTED, "large"), (dict(rows=-1), INVALID, "sizes"),
    (dict(top=33), UNSUPPORTED, "top"), (dict(top=-1), UNSUPPORTED, "top"), (dict(tokens=None), INVALID, "NULL"), (dict(ids=None), INVALID, "NULL"),
    (dict(logits=FAKE + 1), INVALID, "aligned"), (dict(stride=-1), INVALID, "strides"), (dict(V=1 << 20), WORKSPACE, "workspace"),
    (dict(V=1 << 20, ws=FAKE + 16, nbytes=1 << 30), INVALID, "256-byte"),
])
def test_token_logprobs_are_checked(lib, over, code, msg):
    a = dict(dtype=0, logits=FAKE, stride=1000, blocked=None, b_stride=0, tokens=FAKE, lp=FAKE, entropy=FAKE, top_lp=FAKE, ids=FAKE, rows=3,
             V=1000, top=5, ws=None, nbytes=0)
    a.update(over)
    check(lib, lib.wdrz_token_logprobs(*a.values(), None), code, msg)


def test_nothing_to_do_is_no_error(lib):
    assert lib.wdrz_page_truncate(tables(), FAKE, 0, FAKE, 0, None) == 0
    assert lib.wdrz_page_write(2, pages(), None, None, None, None, None, 0, None) == 0
    assert lib.wdrz_attn_packed(2, None, None, None, None, None, None, None, None, FAKE, None, 0, 0, 0, 4, 4, 64, 0.125, 1, None) == 0
    assert lib.wdrz_token_logprobs(2, None, 0, None, 0, None, None, None, None, None, 0, 10, 0, None, 0, None) == 0


@pytest.mark.parametrize("kw,err", [(dict(page_size=24), NotImplementedError), (dict(n_streams=0), ValueError), (dict(n_streams=12289), ValueError),
                                    (dict(n_pages=0), ValueError), (dict(max_seq_length=0), ValueError)])
def test_page_tables_are_refused(kw, err):
    with pytest.raises(err):
        w.PageTables(**{**dict(n_streams=4, n_pages=10, page_size=16, max_seq_length=100), **kw})


def test_new_tables_and_their_storage():
    t = w.PageTables(3, 10, 16, 100)
    assert t.tables.shape == (3, 7) and int(t.tables.max()) == -1 and int(t.n_free) == 10
    assert t.free_pages.tolist() == list(range(9, -1, -1)) and not t.seq_lens.any() and not t.page_counts.any()
    st = {n: torch.zeros(s, dtype=torch.int32) for n, s in w.PageTables.layout(3, 10, 16, 100).items()}
    assert w.PageTables(3, 10, 16, 100, storage=st).tables is st["tables"]
    for bad in (dict(tables=torch.zeros(3, 8, dtype=torch.int32)), dict(seq_lens=torch.zeros(3, dtype=torch.int64)), dict(n_free=None),
                dict(tables=torch.zeros(7, 3, dtype=torch.int32).T)):
        with pytest.raises(ValueError):
            w.PageTables(3, 10, 16, 100, storage={**st, **bad})


def test_calls_on_the_cpu_are_refused():
    t = w.PageTables(3, 10, 16, 100)
    ids = lambda *x: torch.tensor(x, dtype=torch.int32)
    for call in (lambda: t.plan(1), lambda: t.plan(ids(1, 2, 3), 6), lambda: t.truncate(0), lambda: t.truncate(ids(1), ids(0))):
        with pytest.raises(RuntimeError):
            call()
    c = w.FlashKVPages(t, 2, 64)
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: c.write(x, x, torch.arange(4)), lambda: w.flash_attn_with_kvpages(x[:, None], c, cache_seqlens=ids(0, 0, 0, 0)),
                 lambda: w.packed_attention(x, x, x, ids(0, 4)), lambda: w.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError):
            call()


def test_requests_of_bad_shapes_are_refused():
    t = w.PageTables(3, 10, 16, 100)
    for lens, streams, err in ((1.5, None, TypeError), (4, torch.zeros(2, 2, dtype=torch.int32), ValueError), (None, None, TypeError)):
        with pytest.raises(err):
            t.plan(lens, 4, streams)
        with pytest.raises(err):
            t.truncate(lens, streams)


@pytest.mark.parametrize("kw,err", [(dict(head_dim=96), NotImplementedError), (dict(dtype=torch.float32), TypeError),
                                    (dict(storage={}), ValueError),
                                    (dict(storage={n: torch.zeros(10, 2, 32, 64, dtype=torch.bfloat16) for n in ("k_pages", "v_pages")}), ValueError)])
def test_pages_of_other_kinds_are_refused(kw, err):
    with pytest.raises(err):
        w.FlashKVPages(w.PageTables(3, 10, 16, 100), 2, **kw)


def test_a_pool_and_its_bytes():
    pool = w.KVPagePool(2, 3, 12, n_heads=4, self_len=100, cross_len=50, page_size=32)
    assert [c.k_pages.shape for c in pool.self_kv] == [(12, 4, 32, 64)] * 2 and pool.cross_kv[1].k_cache.shape == (3, 50, 4, 64)
    held = sum(t.numel() * 2 for c in pool.self_kv for t in (c.k_pages, c.v_pages))
    assert held == 12 * w.KVPagePool.page_bytes(2, 4, 64, 32, torch.bfloat16)
    assert w.KVPagePool.page_bytes(32, 20, 64, 16, torch.bfloat16) == 2621440


def test_launches_of_too_many_threads_are_refused(lib):
    """2^32 threads and more along the grid's first axis: refused before the launch, not by it."""
    q4 = strides(1 << 20, 1 << 20, 64, 1)
    assert lib.wdrz_page_write(2, pages(n_heads=65535), FAKE, R3, FAKE, R3, FAKE, 1 << 14, None) == UNSUPPORTED
    assert lib.wdrz_attn_packed(2, FAKE, R3, FAKE, R3, FAKE, R3, FAKE, R3, FAKE, FAKE, 1, 1 << 24, 8, 128, 128, 64, 0.125, 1, None) == UNSUPPORTED
    assert lib.wdrz_attn_packed(2, FAKE, R3, FAKE, R3, FAKE, R3, FAKE, R3, FAKE, FAKE, 65535, 65535, 8, 131, 131, 128, 0.125, 1, None) == UNSUPPORTED
    assert lib.wdrz_attn_kvpages(2, pages(n_heads=1024), tables(), FAKE, q4, None, None, None, None, FAKE, FAKE, FAKE, q4, 65535, 16, 1024, 0.125, None, 0, None) == UNSUPPORTED
    assert lib.wdrz_token_logprobs(0, FAKE, 10, None, 0, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 24, 10, 0, None, 0, None) == UNSUPPORTED
    assert b"too large" in lib.wdrz_last_error()
