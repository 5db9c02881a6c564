"""The debug library (WDRZ_DEBUG) reads the metadata of the paged cache's and the packed calls and refuses what is out of range
or named twice, before anything is launched; what is valid gives the release library's results."""
import ctypes

import pytest
import torch

import whisperdrz_amd as w

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def dbg(cuda):
    from whisperdrz_amd import _lib

    lib = ctypes.CDLL(str(_lib.DEBUG_LIB_PATH))
    _lib._declare(lib)
    return lib


def ids(cuda, x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=cuda)


def strides(t):
    return (ctypes.c_int64 * t.dim())(*t.stride())


def stream():
    return torch.cuda.current_stream().cuda_stream


def refused(lib, rc, *words):
    from whisperdrz_amd import _lib

    msg = lib.wdrz_last_error().decode()
    assert rc == _lib.WDRZ_EINVAL and "debug check" in msg and all(x in msg for x in words), msg


@pytest.fixture
def cache(cuda):
    t = w.PageTables(3, 12, 16, 64, device=cuda)
    c = w.FlashKVPages(t, 2, 64, BF16)
    x = torch.randn(60, 2, 64, device=cuda).to(BF16)
    c.write(x, x, t.plan(20).slots)
    return c


def attend(lib, c, lens, streams, new=True, out=None):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(len(lens), 1, 2, 64, generator=g).to(BF16).to(c.device) for _ in range(3))
    out = torch.zeros_like(q) if out is None else out
    at, by = ids(c.device, lens), ids(c.device, streams)
    rc = lib.wdrz_attn_kvpages(2, c.struct, c.page_tables.struct, q.data_ptr(), strides(q), k.data_ptr() if new else None, strides(k),
                               v.data_ptr() if new else None, strides(v), at.data_ptr(), by.data_ptr(), out.data_ptr(), strides(out),
                               len(lens), 1, 2, 0.125, None, 0, stream())
    torch.cuda.synchronize()
    return rc, out


@pytest.mark.parametrize("lens,streams,words", [
    ([20, 20], [0, 3], ["row 1", "stream 3"]), ([20, 20], [-1, 1], ["row 0", "stream -1"]), ([-1, 20], [0, 1], ["row 0", "covers"]),
    ([20, 64], [0, 1], ["row 1", "covers"]), ([20, 20], [2, 2], ["rows 0 and 1", "stream 2"]), ([20, 40], [0, 1], ["page 2 of its table is -1"])])
def test_rows_that_are_refused(cuda, dbg, cache, lens, streams, words):
    before = cache.k_pages.clone()
    refused(dbg, attend(dbg, cache, lens, streams)[0], *words)
    assert torch.equal(cache.k_pages, before)


def test_slots_and_sums_that_are_refused(cuda, dbg, cache):
    x = torch.randn(3, 2, 64, device=cuda).to(BF16)
    st = (ctypes.c_int64 * 3)(*x.stride())
    write = lambda s: dbg.wdrz_page_write(2, cache.struct, x.data_ptr(), st, x.data_ptr(), st, s.data_ptr(), 3, stream())
    before = cache.k_pages.clone()
    refused(dbg, write(ids(cuda, [0, 192, -1], torch.int64)), "slot 192")
    refused(dbg, write(ids(cuda, [7, -1, 7], torch.int64)), "slot 7", "twice")
    assert torch.equal(cache.k_pages, before)
    out = torch.zeros_like(x)
    packed = lambda cu, cu_k: dbg.wdrz_attn_packed(2, x.data_ptr(), st, x.data_ptr(), st, x.data_ptr(), st, out.data_ptr(), st, cu.data_ptr(),
                                                   cu_k.data_ptr(), 2, 3, 3, 2, 2, 64, 0.125, 1, stream())
    good = ids(cuda, [0, 1, 3])
    for bad in ([0, 2, 1], [0, 2, 4], [-1, 1, 2]):
        refused(dbg, packed(ids(cuda, bad), good), "cu_seqlens[")
        refused(dbg, packed(good, ids(cuda, bad)), "cu_seqlens_k[")
    assert not out.any()
    assert packed(good, good) == 0
    assert torch.equal(out, w.packed_attention(x, x, x, good, scale=0.125))
    assert write(ids(cuda, [100, -1, 7], torch.int64)) == 0


def test_valid_rows_equal_the_release(cuda, dbg, cache):
    from whisperdrz_amd import _lib

    keep = cache.k_pages.clone(), cache.v_pages.clone()
    for lens, streams, new in (([20, 5], [2, 0], True), ([20, 0, 20], [1, 1, 0], False)):
        results = []
        for lib in (dbg, _lib.load()):
            cache.k_pages.copy_(keep[0]), cache.v_pages.copy_(keep[1])
            rc, out = attend(lib, cache, lens, streams, new)
            assert rc == 0
            results.append((out, cache.k_pages.clone(), cache.v_pages.clone()))
        assert all(torch.equal(a, b) for a, b in zip(*results))
