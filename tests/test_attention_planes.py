"""The bounds of tests/attention_planes.py, on the CPU: what the kernels' arithmetic gives lies within them, and without any of the six
products it does not."""
import pytest
import torch

import attention_planes as planes


def _numbers(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(n, generator=g), torch.randn(n, generator=g)


def _error(x, y, without=None):
    """In U of the product."""
    exact = x.double() * y.double()
    return ((planes.product(x, y, without).double() - exact).abs() / exact.abs() / planes.U).max().item()


def test_planes_hold_all_bits():
    x, _ = _numbers(100000, 0)
    a, b, c = planes.split(x)
    assert torch.equal(a.double() + b.double() + c.double(), x.double())
    assert bool((b.abs() <= 2.0 ** -8 * x.abs()).all()) and bool((c.abs() <= 2.0 ** -17 * x.abs()).all())


@pytest.mark.parametrize("rows", [240, 1000])
def test_a_missing_product_shows(rows):
    """Of as many rows as the GPU tests look at."""
    x, y = _numbers(rows, 1)
    assert _error(x, y) <= planes.PRODUCT
    largest = max(planes.LOGARITHM + planes.LOGARITHM_ADDS, planes.OUTPUT, planes.VALUES, planes.QUERIES)
    for without in planes.PAIRS:
        assert _error(x, y, without) > 2 * largest, without


def test_a_missing_product_of_equal_values_shows():
    """Two keys' probabilities times the same value, over their sum."""
    g = torch.Generator().manual_seed(2)
    p, c = torch.rand(240, generator=g), torch.randn(240, generator=g)
    one = torch.ones(240)

    def error(without=None):
        o = (planes.product(c, one, without) + planes.product(c, p, without)) * (1 / (one + p))
        return ((o.double() - c.double()).abs() / c.double().abs() / planes.U).max().item()

    assert error() <= planes.OUTPUT
    for without in planes.PAIRS:
        assert error(without) > 1.5 * planes.OUTPUT, without


def test_rows_with_one_element():
    g = torch.Generator().manual_seed(3)
    x = planes.one_element(200, 2, 96, g, "cpu")
    assert bool(((x != 0).sum(3) == 1).all()) and bool((x != 0).any(1).any(1).all())  # every element is somebody's
