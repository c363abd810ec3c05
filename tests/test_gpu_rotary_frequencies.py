"""Frequencies of the caller's own: strided, on the GPU already, changed after they were copied."""
import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_strided_frequencies(where):
    from dihydrogen_amd.tokens import RotaryPositions
    layer = RotaryPositions(16, [3, 2])
    given = torch.linspace(0.1, 1.9, 10, dtype=torch.float64, device=where)[::2]
    layer.frequencies = given
    want = given.clone()
    x = torch.randn(2, 7, 3, 16, device="cuda")
    positions = torch.arange(14, dtype=torch.int32, device="cuda").view(2, 7)
    y, again = torch.empty_like(x), torch.empty_like(x)
    layer.forward(x, positions, y)
    exact = ref.rotary(x, positions.expand(2, -1, -1), want.cuda(), (3, 2), False)
    ref.check(y, exact, ref.rotary_bound(x, exact, (3, 2), False, ref.U, ref.half_step(x.dtype)), "y")
    given.zero_()  # the layer has a copy
    layer.forward(x, positions, again)
    assert torch.equal(y, again)
