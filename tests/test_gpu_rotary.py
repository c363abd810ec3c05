"""Rotary positions with several axes, against the plain form in 64 bits."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float64, torch.bfloat16, torch.float16]


def _case(n, tokens, heads, dim, axes, dtype, per_sample=False, seed=0, far=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(n, tokens, heads, dim, device="cuda").normal_(0, 1, generator=g).to(dtype)
    lo, hi = (-(2 ** 31), 2 ** 31 - 1) if far else (-40, 5000)
    shape = (n, len(axes), tokens) if per_sample else (len(axes), tokens)
    positions = torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=torch.int64).to(torch.int32)
    return x, positions


def _want(layer, x, positions, inverse):
    from dihydrogen_amd.tokens import RotaryPairing
    neighbours = layer.pairing == RotaryPairing.NEIGHBOURS
    p = positions if positions.dim() == 3 else positions.expand(x.shape[0], -1, -1)
    y = ref.rotary(x, p, layer.frequencies.to(x.device), layer.axis_pairs, neighbours, inverse)
    u = 2.0 ** -53 if x.dtype == torch.float64 else ref.U
    # (angles of doubles are not reduced beforehand: they carry half a step of their own magnitude)
    bound = ref.rotary_bound(x, y, layer.axis_pairs, neighbours, u, ref.half_step(x.dtype))
    if x.dtype == torch.float64:
        bound = bound + 4 * u * float(p.double().abs().max()) * x.abs().amax()
    return y, bound


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("pairing", ["HALVES", "NEIGHBOURS"])
@pytest.mark.parametrize("dim,axes", [(2, (1,)), (8, (2, 1)), (64, (8, 12, 12)), (64, (16, 16)), (72, (9, 13, 14)), (80, (10, 12, 10, 8)),
                                      (96, (0, 24, 16)), (128, (16, 24, 24)), (128, (64,)), (51, (7, 9)), (256, (64, 64))])
def test_against_the_plain_form(dtype, pairing, dim, axes):
    from dihydrogen_amd.tokens import RotaryPairing, RotaryPositions
    layer = RotaryPositions(dim, axes, pairing=RotaryPairing[pairing])
    for n, tokens, heads, per_sample in ((1, 1, 1, False), (2, 37, 3, True), (3, 130, 8, False)):
        x, positions = _case(n, tokens, heads, dim, axes, dtype, per_sample)
        buffer, y = ref.ragged(x.shape, dtype, 7.0)
        layer.forward(x, positions, y)
        ref.check(y, *_want(layer, x, positions, False), f"forward {n} {tokens} {heads}")
        layer.backward(x, positions, y)
        ref.check(y, *_want(layer, x, positions, True), f"backward {n} {tokens} {heads}")
        assert ref.outside_untouched(buffer, y, 7.0)
        # in place, the same bits
        z = x.clone()
        layer.backward(z, positions, z)
        assert torch.equal(z, y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,axes", [(64, (8, 12, 12)), (40, (4, 5, 6))])
def test_strides(dtype, dim, axes):
    """Heads of a fused projection, heads first, gaps and odd offsets, positions with gaps."""
    from dihydrogen_amd.tokens import RotaryPairing, RotaryPositions
    x, positions = _case(2, 19, 4, dim, axes, dtype, per_sample=True)
    spaced = torch.full((2, 3, 30), -7, dtype=torch.int32, device="cuda")
    spaced[:, :, :19] = positions
    for pairing in RotaryPairing:
        layer = RotaryPositions(dim, axes, pairing=pairing)
        for order, gap, offset in (((0, 2, 1, 3), 0, 0), ((0, 1, 2, 3), 5, 1), ((1, 0, 2, 3), 8, 8), ((2, 1, 0, 3), 3, 2)):
            view = ref.ragged(x.shape, dtype, math.nan, gap=gap, offset=offset, order=order)[1]
            view.copy_(x)
            buffer, y = ref.ragged(x.shape, dtype, 7.0, gap=gap, offset=offset)
            layer.forward(view, spaced[:, :, :19], y)
            ref.check(y, *_want(layer, x, positions, False), f"{order}")
            assert ref.outside_untouched(buffer, y, 7.0)


def test_far_positions():
    """Positions of 31 bits, where an angle in 32 bits would be off by many turns."""
    from dihydrogen_amd.tokens import RotaryPositions
    layer = RotaryPositions(64, (16, 16))
    x, positions = _case(2, 300, 2, 64, (16, 16), torch.float32, far=True)
    positions[0, :3] = torch.tensor([2 ** 31 - 1, -(2 ** 31), 0], dtype=torch.int32)
    y = torch.empty_like(x)
    layer.forward(x, positions, y)
    ref.check(y, *_want(layer, x, positions, False), "far")


def test_shards_agree_with_the_whole():
    """A grid split between ranks: each shard's tokens are turned as the whole grid's are."""
    from dihydrogen_amd.tensor import Distribution, LocaleVirtual, Tensor
    from dihydrogen_amd.tokens import RotaryPositions, grid_positions
    layer = RotaryPositions(24, (4, 4, 4))
    make = lambda rank, dist, size: Tensor([9, 7, 5, 1, 1], LocaleVirtual(rank, size), dist)
    whole = make(0, Distribution.make_localized_distribution(5), 1)
    x = torch.randn(1, 5 * 7 * 9, 2, 24, device="cuda")
    y = torch.empty_like(x)
    layer.forward(x, grid_positions(whole), y)
    dist = Distribution([2, 2, 1, 1, 1])
    for rank in range(4):
        t = make(rank, dist, 4)
        cut = tuple(slice(o, o + l) for o, l in zip(reversed(t.global_index[:3]), reversed(t.local_shape[:3])))
        part = x.view(5, 7, 9, 2, 24)[cut].reshape(1, -1, 2, 24).contiguous()
        out = torch.empty_like(part)
        layer.forward(part, grid_positions(t), out)
        assert torch.equal(out, y.view(5, 7, 9, 2, 24)[cut].reshape(out.shape))


def test_gradient_against_differences():
    from dihydrogen_amd.tokens import RotaryPositions
    layer = RotaryPositions(16, (4, 3))
    x, positions = _case(2, 5, 3, 16, (4, 3), torch.float64)
    dy, dx, y = torch.randn_like(x), torch.empty_like(x), torch.empty_like(x)
    layer.backward(dy, positions, dx)
    d = torch.randn_like(x)
    loss = []
    for sign in (1, -1):
        layer.forward(x + sign * d, positions, y)
        loss.append(float((y * dy).sum()))
    assert math.isclose((loss[0] - loss[1]) / 2, float((dx * d).sum()), rel_tol=1e-10, abs_tol=1e-10)  # (linear in x)


def test_nothing_to_turn():
    from dihydrogen_amd.tokens import RotaryPositions
    layer = RotaryPositions(8, (4,))
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.empty(shape, device="cuda")
        layer.forward(x, torch.zeros(1, shape[1], dtype=torch.int32, device="cuda"), torch.empty_like(x))
    torch.cuda.synchronize()
