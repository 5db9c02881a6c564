"""A plan's requests are served in order while pages last."""
import pytest
import torch

import whisperdrz_amd as w

pytestmark = pytest.mark.gpu


def test_nobody_overtakes_a_request_that_finds_too_few_pages(cuda):
    """Three pages for needs of 1, 5, 1 and 0: the first is served, the second not, the third waits behind it; the fourth needs none."""
    t = w.PageTables(4, 3, 16, 96, device=cuda)
    t.plan(torch.tensor([0, 0, 0, 3], dtype=torch.int32, device=cuda), 3)
    t.truncate(torch.tensor([0, 0, 0, 2], dtype=torch.int32, device=cuda))
    plan = t.plan(torch.tensor([16, 80, 16, 14], dtype=torch.int32, device=cuda), 126)
    assert plan.starts.tolist() == [0, -1, -1, 2] and t.seq_lens.tolist() == [16, 0, 0, 16] and int(t.n_free) == 1
    plan = t.plan(torch.tensor([0, 0, 16, 0], dtype=torch.int32, device=cuda), 16)
    assert plan.starts.tolist() == [16, 0, 0, 16] and int(t.n_free) == 0
