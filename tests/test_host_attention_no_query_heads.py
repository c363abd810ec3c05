"""Gradients without query heads: a call that has keys is one that writes their gradients.  (No kernel runs: pointers are imaginary, and the file is
skipped where a GPU is visible; tests/test_gpu_attention_no_query_heads.py looks at what is written.)"""
import ctypes

import pytest
import torch

from dihydrogen_amd import capi

INVALID, TOO_LARGE = -1, -3
P, DK, DV = (ctypes.c_void_p(i << 20) for i in (1, 2, 3))


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: valid calls would launch on imaginary pointers")


def _call(samples=2, key_heads=2, queries=5, keys=6, k=P, dk=DK, dv=DV):
    a = capi.Attention()
    a.dtype, a.head_dim, a.samples, a.query_heads, a.key_heads, a.queries, a.keys = capi.BF16, 8, samples, 0, key_heads, queries, keys
    a.window_left, a.window_right, a.scale = -1, -1, 0.125
    a.k = a.v = a.dk = a.dv = capi.TokenStrides(96, 16, 8)
    a.q = a.o = a.d_o = a.dq = capi.TokenStrides(8, 8, 8)
    lib = capi.load()
    assert lib.h2x_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
    v = ctypes.c_void_p(9 << 20)
    return lib.h2x_attention_backward(ctypes.byref(a), None, k, v, None, None, None, None, None, None, dk, dv, None, None)


def test_without_query_heads():
    assert _call() > 0 and _call(queries=0) > 0  # HIP's own error: there is no GPU
    assert _call(dk=None) == INVALID and _call(dv=None) == INVALID and _call(k=None) == INVALID and _call(dv=DK) == INVALID
    assert _call(samples=0) == 0 and _call(key_heads=0) == 0 and _call(keys=0, k=None, dk=None, dv=None) == 0
    assert _call(samples=1 << 30, key_heads=1 << 30, keys=1 << 30) == TOO_LARGE
