"""Gradients of keys and values that have no query heads are sums of nothing: zeros, not what was there."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("queries,keys,lengths", [(5, 6, False), (0, 40, False), (300, 2000, True)])
def test_no_query_heads(dtype, queries, keys, lengths):
    from dihydrogen_amd.tokens import Attention
    layer = Attention(causal=True)
    q, k = torch.empty(2, queries, 0, 8, dtype=dtype, device="cuda"), torch.ones(2, keys, 2, 8, dtype=dtype, device="cuda")
    v, o, d_o, dq = k.clone(), q.clone(), q.clone(), q.clone()
    lse = torch.empty(2, 0, queries, device="cuda")
    dk, dv = torch.full_like(k, math.nan), torch.full_like(k, math.nan)
    n = {"query_lengths": torch.tensor([queries, 1], dtype=torch.int32, device="cuda"),
         "key_lengths": torch.tensor([keys, 1], dtype=torch.int32, device="cuda")} if lengths else {}
    layer.forward(q, k, v, o, lse, **n)
    layer.backward(q, k, v, o, d_o, lse, dq, dk, dv, **n)
    assert bool((dk == 0).all()) and bool((dv == 0).all())
