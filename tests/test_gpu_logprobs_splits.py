"""Token log probabilities where rows begin to be split: 512 rows are the most that are, each over two workgroups."""
import pytest
import torch

import whisperdrz_amd as w
from oracle.paged_oracle import logprobs
from whisperdrz_amd.attention import _COUNTED_WORKSPACES
from whisperdrz_amd.decode_ops import _logprobs_workspace_size

pytestmark = pytest.mark.gpu

V, TOP = 70001, 4


@pytest.fixture(scope="module")
def data(cuda):
    """Rows with a likely token each, and what they are in 64 bits; ties among the alternatives in some."""
    g = torch.Generator().manual_seed(11)
    x = (2.0 * torch.randn(513, V, generator=g)).to(torch.bfloat16)
    tokens = torch.randint(0, V, (513,), generator=g)
    x[torch.arange(513), tokens] = 12.0
    x[::7, V - 1], x[::7, 5] = 13.0, 13.0
    d = x.double()
    lp = torch.log_softmax(d, -1)
    entropy = torch.special.entr(lp.exp()).sum(-1)
    order = torch.sort(d, dim=-1, descending=True, stable=True).indices[:, :TOP]
    return x.to(cuda), tokens.to(cuda), lp.gather(1, tokens[:, None])[:, 0], entropy, lp.gather(1, order), order


def test_workspaces_end_where_rows_are_not_split(cuda):
    size = 8 * 35  # two sums, the largest key and 32 others
    for rows, parts in ((1, 32), (32, 32), (33, 31), (340, 3), (341, 3), (342, 2), (511, 2), (512, 2), (513, 1), (4100, 1)):
        assert _logprobs_workspace_size(rows, V, TOP) == (0 if parts == 1 else 4096 * 4 + rows * parts * size), rows


@pytest.mark.parametrize("counts", [(340, 513, 341), (342, 1, 512), (511, 33, 512, 32, 513)])
def test_rows_at_the_edges_of_splitting(cuda, data, counts):
    """One workspace for calls of changing row counts. Tolerance: sums in fp32 of at most 2^10 terms a thread and fp64 above, a
    logarithm and a difference in fp64, one rounding: 2^-17 of a log probability or entropy."""
    x, tokens, lp, entropy, values, ids = data
    for rows in counts:
        got = w.token_logprobs(x[:rows], tokens[:rows], TOP)
        assert torch.equal(got.top_ids.cpu(), ids[:rows]), rows
        for a, b in ((got.logprobs, lp), (got.entropy, entropy), (got.top_logprobs, values)):
            assert torch.allclose(a.cpu().double(), b[:rows], rtol=2**-17, atol=2.0**-40), rows
        torch.cuda.synchronize()
        assert not any(b[: 4096 * 4].any() for b in _COUNTED_WORKSPACES.values())
    some = [0, counts[0] // 2, counts[0] - 1]
    want = logprobs(x[some].cpu(), tokens[some].cpu(), TOP)
    assert torch.equal(want[3], ids[some])
