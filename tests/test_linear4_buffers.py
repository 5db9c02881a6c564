"""A 4-bit layer's buffers are held to its sizes: the kernels read all that the features and groups stand for."""
import pytest
import torch

from whisperdrz_amd import QuantLinear4, linear4, linear4_partials

BF = torch.bfloat16


def _parts(N=40, K=192, group=64, bias=True):
    tiles = -(-N // 16)
    return [K, N, group, torch.zeros(tiles, -(-K // 128), 1024, dtype=torch.uint8), torch.ones(tiles, K // group, 16, dtype=BF),
            torch.zeros(N, dtype=BF) if bias else None]


def test_whole_buffers_are_taken():
    for bias in (True, False):
        lin = QuantLinear4(*_parts(bias=bias))
        assert lin.dequantize().shape == (40, 192) and (lin.bias is None) != bias


@pytest.mark.parametrize("at,value,err", [
    (3, torch.zeros(1, 2, 1024, dtype=torch.uint8), ValueError),  # fewer tiles than features
    (3, torch.zeros(3, 1, 1024, dtype=torch.uint8), ValueError),  # fewer chunks than inputs
    (3, torch.zeros(3, 2, 512, dtype=torch.uint8), ValueError),
    (3, torch.zeros(3, 2, 2048, dtype=torch.uint8)[..., ::2], ValueError),  # not contiguous
    (3, torch.zeros(1, 1, 1024, dtype=torch.uint8).expand(3, 2, 1024), ValueError),
    (3, torch.zeros(3, 2, 1024, dtype=torch.int8), TypeError),
    (4, torch.ones(3, 2, 16, dtype=BF), ValueError),  # groups of 128 for a layer of 64
    (4, torch.ones(2, 3, 16, dtype=BF), ValueError),
    (4, torch.ones(3, 16, 3, dtype=BF).transpose(1, 2), ValueError),
    (4, torch.ones(3, 3, 16), TypeError),
    (5, torch.zeros(39, dtype=BF), ValueError),
    (5, torch.zeros(80, dtype=BF)[::2], ValueError),
    (5, torch.zeros(40, dtype=torch.float16), TypeError),
    (5, torch.zeros(40, dtype=BF, device="meta"), ValueError),
    (2, 48, NotImplementedError),
    (2, 128, NotImplementedError),  # does not divide the inputs
    (0, 0, NotImplementedError),
    (1, 0, NotImplementedError),
])
def test_other_buffers_are_refused(at, value, err):
    args = _parts()
    args[at] = value
    with pytest.raises(err):
        QuantLinear4(*args)


@pytest.mark.gpu
def test_buffers_replaced_after_construction(cuda):
    """What a layer holds at the call counts, not what it was built with. Nothing is launched."""
    w = torch.randn(40, 192, device=cuda).to(BF)
    x = torch.randn(3, 192, device=cuda).to(BF)
    for name, value, err in [("packed", lambda t: t[:2], ValueError), ("packed", lambda t: t[:, :1], ValueError),
                             ("scales", lambda t: t[:, :2], ValueError), ("bias", lambda t: t[:8], ValueError),
                             ("packed", lambda t: t.view(torch.int8), TypeError)]:
        lin = QuantLinear4.from_weight(w, torch.zeros(40, device=cuda, dtype=BF))
        linear4(x, lin)
        setattr(lin, name, value(getattr(lin, name)))
        for f in (linear4, linear4_partials):
            with pytest.raises(err):
                f(x, lin)
