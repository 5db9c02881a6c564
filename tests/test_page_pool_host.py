"""What a KVPagePool and a plan refuse on the host."""
import pytest
import torch

import whisperdrz_amd as w


@pytest.mark.parametrize("dim", [128, 96, 32])
def test_a_pool_of_other_heads_is_refused(dim):
    """Its cross caches are attended with heads of 64; pages alone take 128."""
    with pytest.raises(NotImplementedError, match="head_dim"):
        w.KVPagePool(1, 2, 8, n_heads=2, head_dim=dim, self_len=64, cross_len=10)
    if dim == 128:
        assert w.FlashKVPages(w.PageTables(2, 8, 16, 64), 2, dim).k_pages.shape == (8, 2, 16, 128)


@pytest.mark.parametrize("new,total,streams", [(3, 8, None), (1, 0, torch.tensor([0, 2], dtype=torch.int32)), (2, -1, None)])
def test_a_plan_of_too_few_tokens_is_refused(new, total, streams):
    t = w.PageTables(3, 10, 16, 100)
    with pytest.raises(ValueError, match="total"):
        t.plan(new, total, streams)
