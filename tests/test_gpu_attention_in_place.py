"""The output of attention over its queries, with the same strides: each workgroup, or the launch that joins the parts, writes only rows whose queries
have been read.  (Other strides are refused: tests/test_host_token_aliases.py.)"""
import pytest
import torch

from test_gpu_attention import DTYPES, Problem

pytestmark = pytest.mark.gpu


@DTYPES
@pytest.mark.parametrize("queries,keys", [(300, 100), (12, 300), (200, 333), (5, 9000)], ids=["wide", "few", "split", "parts"])
@pytest.mark.parametrize("layout", ["tokens", "heads first"])
def test_output_over_the_queries(dtype, queries, keys, layout):
    p = Problem(2, queries, keys, 4, 2, 64, dtype, window=(None, 0), layout=layout)
    want = [t.clone() for t in p.forward()]
    q, k, v, _ = p.inputs
    lse = torch.empty_like(want[1])
    p.layer.forward(q, k, v, q, lse)
    assert torch.equal(q, want[0]) and torch.equal(lse, want[1])
