"""The debug library refuses a plan whose requests have more tokens than it gives places for."""
import ctypes

import pytest
import torch

import whisperdrz_amd as w

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new,total,ok", [([3, 4], 7, True), ([3, -9, 4], 7, True), ([3, 5], 7, False), ([2**31 - 1, 2**31 - 1], 7, False)])
def test_counts_beyond_the_total(cuda, new, total, ok):
    from whisperdrz_amd import _lib

    lib = ctypes.CDLL(str(_lib.DEBUG_LIB_PATH))
    _lib._declare(lib)
    t = w.PageTables(4, 10, 16, 64, device=cuda)
    lens = torch.tensor(new, dtype=torch.int32, device=cuda)
    cu, starts = torch.zeros(len(new) + 1, dtype=torch.int32, device=cuda), torch.zeros_like(lens)
    slots, positions = (torch.zeros(total, dtype=torch.int64, device=cuda) for _ in range(2))
    call = lambda lens, each: lib.wdrz_page_plan(t.struct, lens, each, None, cu.data_ptr(), starts.data_ptr(), slots.data_ptr(),
                                                 positions.data_ptr(), len(new), total, torch.cuda.current_stream().cuda_stream)
    rc = call(lens.data_ptr(), 0)
    msg = lib.wdrz_last_error().decode()
    torch.cuda.synchronize()
    assert rc == (_lib.WDRZ_OK if ok else _lib.WDRZ_EINVAL), msg
    if not ok:
        assert "debug check" in msg and "total" in msg and not t.seq_lens.any() and int(t.n_free) == 10
    assert call(None, 4) == _lib.WDRZ_EINVAL and "total" in lib.wdrz_last_error().decode()
