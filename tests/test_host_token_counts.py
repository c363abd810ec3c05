"""Counts that the C ABI takes in 32 bits are refused beyond, not wrapped: 2^32 + 8 channels are not 8.  (Tensors without memory; nothing is
launched.)"""
import pytest
import torch

from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions

MANY = (1 << 32) + 8


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_channels():
    x = _meta(2, MANY)
    with pytest.raises(ValueError, match="channels: fewer than 2\\^31"):
        LayerNormalization().forward(x, None, None, _meta(2, MANY))
    with pytest.raises(ValueError, match="channels: fewer"):
        rows = _meta(2, dtype=torch.float32)
        LayerNormalization().backward(x, _meta(2, MANY), rows, rows, None, _meta(2, MANY))
    with pytest.raises(ValueError, match="meta"):  # the next thing that is wrong with it
        LayerNormalization().forward(_meta(2, MANY // 4), None, None, _meta(2, MANY // 4))


@pytest.mark.parametrize("shape,what", [((1, 3, MANY, 8), "heads"), ((MANY, 3, 1, 8), "samples")])
def test_heads_and_samples(shape, what):
    with pytest.raises(ValueError, match=f"{what}: fewer"):
        RotaryPositions(8, [4]).forward(_meta(*shape), _meta(1, 3, dtype=torch.int32), _meta(*shape))
    with pytest.raises(ValueError, match=f"{what}: fewer"):
        Attention().forward(_meta(*shape), _meta(*shape), _meta(*shape), _meta(*shape))


def test_key_heads_without_query_heads():
    with pytest.raises(ValueError, match="key heads: fewer"):
        Attention().forward(_meta(1, 3, 0, 8), _meta(1, 3, MANY, 8), _meta(1, 3, MANY, 8), _meta(1, 3, 0, 8))


def test_windows():
    for window in ((1 << 64, 0), (None, (1 << 64) + 5), (1 << 63, None)):
        with pytest.raises(ValueError, match="2\\^63"):
            Attention(window=window)
    assert Attention(window=((1 << 63) - 1, 0)).window == ((1 << 63) - 1, 0)
