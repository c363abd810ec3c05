"""Values near the end of the types' range: exact where the sums of the probabilities and values hold them, and rows behind a
sample's queries are zero whatever their neighbours' values are."""
import math

import pytest
import torch

import token_reference as ref
from test_gpu_attention import DTYPES, Problem

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("queries,keys", [(40, 100), (3, 500), (2, 17000)], ids=["wide", "split", "parts"])
def test_large_values(dtype, queries, keys):
    """keys * 2^8 * the largest value stays below 2^128."""
    for dim in (64, 128):
        p = Problem(1, queries, keys, 2, 1, dim, dtype, window=(None, 0))
        p.inputs[2].mul_(2.0 ** 100)
        p.want = ref.AttentionReference(p.inputs[0], p.inputs[1], p.inputs[2], p.scale, p.seen)
        assert keys * 2.0 ** 8 * float(p.inputs[2].abs().max()) < 2.0 ** 128
        p.check_forward()


@DTYPES
@pytest.mark.parametrize("queries,keys,heads", [(128, 4000, 130), (6, 4000, 150), (6, 9000, 2)], ids=["wide", "split", "parts"])
def test_rows_behind_the_queries_are_zero(dtype, queries, keys, heads):
    """A row behind the sample's queries takes part in the products of its wave as a query of zeros, whose flat sum over these values
    overflows.  The sample's own rows each have one key that outweighs the others: their sums, of probabilities up to 2^8, stay in range."""
    for dim in (64, 128):
        p = Problem(1, queries, keys, heads, heads, dim, dtype, lengths=([queries - 3], None))
        q, k, v, _ = p.inputs
        v.fill_(2e35)
        there = queries - 3
        target = torch.arange(there, device="cuda") * 7 % keys
        q[0, :there] = 12 * k[0, target]
        assert keys * 2e35 > 2.0 ** 128 > 4 * 2 ** 8 * 2e35
        p.want = ref.AttentionReference(q, k, v, p.scale, p.seen)
        assert bool((p.want.p[:, :, :there].amax(3) > 0.9).all())
        o, lse = p.forward()
        assert bool((o[0, there:] == 0).all()) and bool((lse[0, :, there:] == -math.inf).all())
        bo, bl = p.want.forward_bounds(dtype)
        ref.check(o[0, :there], p.want.o.transpose(1, 2)[0, :there], bo.transpose(1, 2)[0, :there], "o")
        ref.check(lse[0, :, :there], p.want.lse[0, :, :there], bl.expand_as(lse)[0, :, :there], "lse")
