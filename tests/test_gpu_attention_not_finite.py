"""A query whose scores are not numbers has an output and a logarithm that are not, in every way that a call is run, and its gradients too:
nothing looks like a row that sees no key.  Other rows are as they would be."""
import math

import pytest
import torch

import token_reference as ref
from test_gpu_attention import BF16, DTYPES, F32, Problem

pytestmark = pytest.mark.gpu

# 128 queries a workgroup; keys split among the waves of a workgroup; the same in four parts, and in sixteen
WAYS = pytest.mark.parametrize("queries,keys", [(40, 100), (3, 200), (3, 3000), (2, 17000)], ids=["wide", "split", "4 parts", "16 parts"])


def _check_others(p, o, lse, bad):
    bo, bl = p.want.forward_bounds(p.dtype)
    good = ~bad
    ref.check(o.transpose(1, 2)[good], p.want.o[good], bo[good], "o of the other rows")
    ref.check(lse[good], p.want.lse[good], bl.expand_as(lse)[good], "logarithms of the other rows")


@DTYPES
@WAYS
@pytest.mark.parametrize("dim", [20, 64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf], ids=["nan", "inf"])
def test_a_query_that_is_not_finite(dtype, queries, keys, dim, value):
    p = Problem(1, queries, keys, 2, 1, dim, dtype, window=(None, 0))
    bad = torch.zeros(1, 2, queries, dtype=torch.bool, device="cuda")
    bad[0, 1, queries - 1] = True
    if math.isnan(value):
        p.inputs[0][0, queries - 1, 1, dim // 2] = value
    else:
        p.inputs[0][0, queries - 1, 1] = value  # sums of infinities of both signs
    o, lse = p.forward()
    assert bool(torch.isnan(o.transpose(1, 2)[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    _check_others(p, o, lse, bad)
    dq, dk, dv = p.backward()
    assert bool(torch.isnan(dq[0, queries - 1, 1]).all())
    assert bool(torch.isnan(dk).all()) and bool(torch.isnan(dv).all())  # (the last query sees all keys)
    if queries == 40:  # the other queries' own
        want, bound = p.want.gradients(p.d_o, o.masked_fill(bad.transpose(1, 2)[..., None], 0), lse.masked_fill(bad, 0), dtype)[0]
        good = ~bad.transpose(1, 2)
        ref.check(dq[good], want[good], bound[good], "dq of the other rows")


@DTYPES
@WAYS
def test_scores_that_overflow(dtype, queries, keys):
    """Finite queries and keys whose product is not: no number is what the formula gives, with scores of plus infinity and with nothing but
    minus infinity."""
    p = Problem(1, queries, keys, 2, 1, 64, dtype)
    q, k = p.inputs[:2]
    q[0, 0, 0], k[:] = 2e38, 2.0
    q[0, 0, 1] = -2e38
    o, lse = p.forward()
    assert bool(torch.isnan(o[0, 0]).all()) and bool(torch.isnan(lse[0, 0, 0]).all())
    assert float(lse[0, 1, 0]) == -math.inf  # the logarithm of a sum of nothing
    assert not bool(torch.isnan(o[0, 1:]).any()) and not bool(torch.isnan(lse[0, :, 1:]).any())
    _, _, dv = p.backward()
    assert bool(torch.isnan(dv).all())


@DTYPES
def test_logarithms_that_are_not_numbers_reach_all_gradients(dtype):
    """The backward pass takes the logarithms as they are: one that is NaN is no empty row's."""
    p = Problem(1, 40, 100, 2, 1, 64, dtype)
    p.forward()
    p.lse[0, 0, 7] = math.nan
    dq, dk, dv = p.backward()
    assert bool(torch.isnan(dq[0, 7, 0]).all()) and bool(torch.isnan(dk).all()) and bool(torch.isnan(dv).all())
    assert not bool(torch.isnan(dq[0, :7]).any())
