"""What a rotary layer holds: frequencies are one float64 a pair, whatever the caller puts there, since the kernel reads that many; what plans are made
with cannot change.  (Nothing is launched.)"""
import pytest
import torch

from dihydrogen_amd.tokens import RotaryPairing, RotaryPositions


def _layer():
    return RotaryPositions(16, [3, 2])


@pytest.mark.parametrize("bad", [torch.ones(5), torch.ones(5, dtype=torch.int64), torch.ones(4, dtype=torch.float64), torch.ones(6, dtype=torch.float64),
                                 torch.ones(1, 5, dtype=torch.float64), torch.ones((), dtype=torch.float64), [1.0] * 5, None],
                         ids=["float32", "int64", "too few", "too many", "a matrix", "a number", "a list", "none"])
def test_frequencies_of_another_kind_are_refused(bad):
    layer = _layer()
    kept = layer.frequencies
    with pytest.raises(ValueError, match="float64"):
        layer.frequencies = bad
    assert layer.frequencies is kept


def test_frequencies_are_looked_at_again_before_they_are_copied():
    layer = _layer()
    layer.frequencies.resize_(2)
    with pytest.raises(ValueError, match="float64"):
        layer._frequencies(torch.device("cuda", 0))


def test_frequencies_may_be_replaced_until_they_are_copied():
    layer = _layer()
    for given in (torch.arange(5, dtype=torch.float64), torch.arange(10, dtype=torch.float64)[::2]):
        layer.frequencies = given
        assert layer.frequencies is given
    layer._on_device[0] = given  # (as a first call leaves it)
    with pytest.raises(ValueError, match="first call"):
        layer.frequencies = torch.ones(5, dtype=torch.float64)
    assert layer.frequencies is given


@pytest.mark.parametrize("name,value", [("head_dim", 32), ("axis_pairs", [1]), ("pairing", RotaryPairing.NEIGHBOURS)])
def test_what_plans_are_made_with_is_fixed(name, value):
    layer = _layer()
    with pytest.raises(AttributeError):
        setattr(layer, name, value)
    with pytest.raises(TypeError):
        layer.axis_pairs[0] = 1
    assert (layer.head_dim, layer.axis_pairs, layer.pairing) == (16, (3, 2), RotaryPairing.HALVES)
