"""A layer whose stream is replaced after its first calls: one of another GPU is refused, though plans for the tensors are there; one of the same is
taken."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Elsewhere:
    """What the layers ask a stream of another GPU for (the handle is the current GPU's default stream, so that nothing could go wrong here)."""
    device_index, cuda_stream = 1, 0


def _layers():
    from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions
    x = torch.randn(2, 3, 4, 8, device="cuda")
    rows, positions = torch.empty(2, 3, 4, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")[None]
    out, lse = torch.empty_like(x), torch.empty(2, 4, 3, device="cuda")
    grads = [torch.empty_like(x) for _ in range(3)]
    norm, turn, attention = LayerNormalization(), RotaryPositions(8, [4]), Attention()
    return [(norm, lambda: norm.forward(x, None, None, out, rows, rows.clone())), (turn, lambda: turn.forward(x, positions, out)),
            (attention, lambda: attention.forward(x, x, x, out, lse)),
            (attention, lambda: attention.backward(x, x, x, out, x, lse, *grads))]


def test_replaced_streams():
    stream = torch.cuda.Stream()
    for layer, call in _layers():
        layer.stream = None
        call()
        torch.cuda.synchronize()
        layer.stream = Elsewhere()
        with pytest.raises(ValueError, match="stream is on GPU 1"):
            call()
        layer.stream = stream
        call()
        stream.synchronize()
