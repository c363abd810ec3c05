"""Outputs of the token operators over their inputs: refused where a workgroup would overwrite what another has yet to read.  (No kernel runs:
pointers are imaginary, and the file is skipped where a GPU is visible.)"""
import ctypes

import pytest
import torch

from dihydrogen_amd import capi

INVALID = -1
Q, K, V, O, W, L = (ctypes.c_void_p(i << 20) for i in range(1, 7))


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: valid calls would launch on imaginary pointers")


@pytest.mark.parametrize("queries,keys", [(300, 100), (3, 200), (3, 20000)], ids=["wide", "split", "parts"])
def test_output_over_the_queries(queries, keys):
    heads, dim = 4, 64

    def call(o, o_strides, samples=2):
        a = capi.Attention()
        a.dtype, a.head_dim, a.samples, a.query_heads, a.key_heads, a.queries, a.keys = capi.BF16, dim, samples, heads, heads, queries, keys
        a.window_left, a.window_right, a.scale = -1, -1, 0.125
        a.q = capi.TokenStrides(queries * heads * dim, heads * dim, dim)
        a.k = a.v = capi.TokenStrides(keys * heads * dim, heads * dim, dim)
        a.o = capi.TokenStrides(*o_strides)
        return capi.load().h2x_attention_forward(ctypes.byref(a), Q, K, V, None, None, o, L, W, None)

    alike = (queries * heads * dim, heads * dim, dim)
    heads_first = (queries * heads * dim, dim, queries * dim)
    assert call(O, alike) > 0 and call(O, heads_first) > 0  # HIP's own error: there is no GPU
    assert call(Q, alike) > 0
    assert call(Q, heads_first) == INVALID
    assert call(Q, (2 * queries * heads * dim, heads * dim, dim)) == INVALID
    assert call(Q, (2 * queries * heads * dim, heads * dim, dim), samples=1) > 0  # (no element's place goes with that stride)
