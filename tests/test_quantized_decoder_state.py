"""A decoder whose Linears are in 4 bits keeps the self-attention's query, key and value in one place, whatever a
program does with the module afterwards."""
import copy
import io

import pytest
import torch

from whisperdrz_amd import QuantLinear4
from whisperdrz_amd.decode_ops import QuantLinear4Rows
from whisperdrz_amd.decoder import TextDecoderStack

N = 64


def _decoder(seed=1, dtype=torch.bfloat16):
    torch.manual_seed(seed)
    return TextDecoderStack(96, 16, N, 1, 2).to(dtype).quantize_linears_(32)


def _one_place(dec):
    for block in dec.blocks:
        a = block.attn
        for i, m in enumerate((a.query, a.key, a.value)):
            assert isinstance(m, QuantLinear4) and (m.in_features, m.out_features, m.group) == (N, N, 32)
            for name, rows in (("packed", N // 16), ("scales", N // 16), ("bias", N)):
                mine, whole = getattr(m, name), getattr(a.qkv4, name)
                if name == "bias" and i == 1:
                    assert mine is None
                    continue
                part = whole[i * rows:(i + 1) * rows]
                assert mine.data_ptr() == part.data_ptr() and mine.dtype == part.dtype and torch.equal(mine, part)
            assert torch.equal(m.dequantize(), a.qkv4.dequantize()[i * N:(i + 1) * N])


def _bytes(dec):
    return sum({b.untyped_storage().data_ptr(): b.untyped_storage().nbytes() for b in dec.buffers()}.values())


def test_conversions_and_copies_keep_one_place():
    dec = _decoder()
    _one_place(dec)
    size = _bytes(dec)
    half = copy.deepcopy(dec).to(torch.float16)
    _one_place(half)
    assert half.blocks[0].attn.query.scales.dtype == torch.float16 and _bytes(half) == size
    same = copy.deepcopy(dec)
    _one_place(same)
    assert same.blocks[0].attn.query.packed.data_ptr() != dec.blocks[0].attn.query.packed.data_ptr()
    meta = copy.deepcopy(dec).to("meta").to_empty(device="cpu")
    meta.load_state_dict(dec.state_dict())
    _one_place(meta)
    assert torch.equal(meta.blocks[1].attn.value.dequantize(), dec.blocks[1].attn.value.dequantize()) and _bytes(meta) == size


@pytest.mark.parametrize("assign", [False, True])
def test_state_dict_holds_the_weights_once(assign):
    a, b = _decoder(1), _decoder(2)
    state = a.state_dict()
    assert not [n for n in state if n.startswith("blocks.0.attn.") and n.split(".")[3] in ("query", "key", "value")]
    assert "blocks.0.attn.qkv4.packed" in state and "blocks.0.cross_attn.query.packed" in state
    file = io.BytesIO()
    torch.save(state, file)
    file.seek(0)
    b.load_state_dict(torch.load(file, weights_only=True), assign=assign)
    _one_place(b)
    for x, y in zip(a.blocks, b.blocks):
        for n in ("query", "key", "value"):
            assert torch.equal(getattr(x.attn, n).dequantize(), getattr(y.attn, n).dequantize())


def test_rows_of_a_layer_are_whole_tiles():
    lin = QuantLinear4.from_weight(torch.randn(48, 64).to(torch.bfloat16), torch.zeros(48, dtype=torch.bfloat16))
    assert torch.equal(QuantLinear4Rows(lin, 16, 32).dequantize(), lin.dequantize()[16:])
    assert QuantLinear4Rows(lin, 0, 16, bias=False).bias is None and not list(QuantLinear4Rows(lin, 0, 16).buffers())
    for first, features in ((8, 16), (0, 8), (0, 0), (-16, 16), (32, 32)):
        with pytest.raises(ValueError, match="whole tiles"):
            QuantLinear4Rows(lin, first, features)
