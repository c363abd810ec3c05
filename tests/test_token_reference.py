"""The 64-bit forms that the token kernels are compared with: their gradients against differences of their
forward passes, and their masks against small cases written out."""
import math

import pytest
import torch

import token_reference as ref


def _difference(f, x, direction, step=1e-5):
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


def test_layer_norm_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    make = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, dy, w, b = make(5, 7), make(5, 7), make(7), make(7)
    dx, dw, db = ref.norm_gradients(x, dy, w, 1e-3)
    for _ in range(4):
        d = make(5, 7)
        assert math.isclose(_difference(lambda t: (ref.norm(t, w, b, 1e-3)[0] * dy).sum(), x, d), (dx * d).sum(), rel_tol=1e-6, abs_tol=1e-8)
        d = make(7)
        assert math.isclose(_difference(lambda t: (ref.norm(x, t, b, 1e-3)[0] * dy).sum(), w, d), (dw * d).sum(), rel_tol=1e-6, abs_tol=1e-8)
        assert math.isclose(_difference(lambda t: (ref.norm(x, w, t, 1e-3)[0] * dy).sum(), b, d), (db * d).sum(), rel_tol=1e-6, abs_tol=1e-8)


@pytest.mark.parametrize("neighbours", [False, True])
def test_rotary_turns_back_and_keeps_lengths(neighbours):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 4, 10, generator=g, dtype=torch.float64)
    positions = torch.randint(-50, 50, (2, 2, 3), generator=g)
    f = torch.tensor([1.0, 0.1, 1.0, 0.3], dtype=torch.float64)
    y = ref.rotary(x, positions, f, (2, 2), neighbours)
    assert torch.allclose(ref.rotary(y, positions, f, (2, 2), neighbours, inverse=True), x, atol=1e-13)
    assert torch.allclose(y.norm(dim=3), x.norm(dim=3), atol=1e-13) and torch.equal(y[..., 8:], x[..., 8:])
    # one pair by hand
    a = float(positions[1, 0, 2]) * 0.1
    i, j = (2, 3) if neighbours else (1, 5)
    assert math.isclose(float(y[1, 2, 3, i]), float(x[1, 2, 3, i] * math.cos(a) - x[1, 2, 3, j] * math.sin(a)), rel_tol=1e-12)


def test_masks_by_hand():
    seen = ref.visible(1, 3, 4, None, 0, None, None)[0].int().tolist()
    assert seen == [[1, 1, 0, 0], [1, 1, 1, 0], [1, 1, 1, 1]]  # the last query stands at the last key
    assert ref.visible(1, 4, 2, None, 0, None, None)[0].int().tolist() == [[0, 0], [0, 0], [1, 0], [1, 1]]
    assert ref.visible(1, 3, 3, 1, 0, None, None)[0].int().tolist() == [[1, 0, 0], [1, 1, 0], [0, 1, 1]]
    assert ref.visible(2, 2, 3, None, None, [1, 2], [2, 0]).int().tolist() == [[[1, 1, 0], [0, 0, 0]], [[0, 0, 0], [0, 0, 0]]]


@pytest.mark.parametrize("left,right,lengths", [(None, None, False), (None, 0, False), (2, 1, True)])
def test_attention_gradients_against_differences(left, right, lengths):
    g = torch.Generator().manual_seed(3)
    make = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    q, k, v, d_o = make(2, 5, 4, 3), make(2, 6, 2, 3), make(2, 6, 2, 3), make(2, 5, 4, 3)
    seen = ref.visible(2, 5, 6, left, right, [5, 3] if lengths else None, [4, 6] if lengths else None)

    def loss(q, k, v):
        r = ref.AttentionReference(q, k, v, 0.6, seen)
        return (r.o * d_o.transpose(1, 2)).sum(), r

    _, r = loss(q, k, v)
    (dq, _), (dk, _), (dv, _) = r.gradients(d_o, r.o.transpose(1, 2), r.lse, torch.float32)
    for _ in range(3):
        a, b, c = make(2, 5, 4, 3), make(2, 6, 2, 3), make(2, 6, 2, 3)
        assert math.isclose(_difference(lambda t: loss(t, k, v)[0], q, a), (dq * a).sum(), rel_tol=1e-6, abs_tol=1e-8)
        assert math.isclose(_difference(lambda t: loss(q, t, v)[0], k, b), (dk * b).sum(), rel_tol=1e-6, abs_tol=1e-8)
        assert math.isclose(_difference(lambda t: loss(q, k, t)[0], v, c), (dv * c).sum(), rel_tol=1e-6, abs_tol=1e-8)
