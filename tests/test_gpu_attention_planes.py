"""Attention of floats, product by product: inputs that make each result of one product, so that all 24 bits of the numbers show (see
tests/attention_planes.py for the bounds, tests/test_attention_planes.py for what a missing product does to them)."""
import pytest
import torch

import attention_planes as planes
import token_reference as ref

pytestmark = pytest.mark.gpu

# 128 queries a workgroup; single queries and many of them with split keys; keys in parts (and tiles in parts in the backward pass)
WAYS = pytest.mark.parametrize("queries,keys", [(120, 120), (14, 14), (230, 230), (14, 5000), (1100, 1100)],
                               ids=["wide", "few", "split", "key parts", "query parts"])
DIMS = pytest.mark.parametrize("dim", [8, 17, 32, 40, 64, 72, 80, 96, 100, 121, 128])


class Case:
    """Each query sees one key, its own (`more` of them before it too); two query heads, of one key head or of two."""

    def __init__(self, queries, keys, dim, layout, scale, more=0, key_heads=2):
        from dihydrogen_amd.tokens import Attention
        self.g = torch.Generator(device="cuda").manual_seed(queries + keys + dim)
        self.queries, self.keys, self.dim, self.layout, self.key_heads = queries, keys, dim, layout, key_heads
        self.layer = Attention(scale=scale, window=(more, 0))
        self.own = slice(keys - queries, keys)  # the keys that the queries stand at

    def place(self, t):
        gap, offset, order = (0, 0, (0, 1, 2, 3)) if self.layout == "aligned" else (3, 1, (0, 2, 1, 3))
        view = ref.ragged(t.shape, torch.float32, float("nan"), gap=gap, offset=offset, order=order)[1]
        return view.copy_(t)

    def normal(self, tokens, heads):
        return torch.empty(1, tokens, heads, self.dim, device="cuda").normal_(0, 1, generator=self.g)

    def one_element(self):
        return planes.one_element(self.queries, 2, self.dim, self.g, "cuda")

    def of_queries(self, t):
        """The key that each query stands at, for each query head."""
        return t[:, self.own].repeat_interleave(2 // self.key_heads, 2)

    def forward(self, q, k, v):
        o, lse = self.place(torch.zeros_like(q)), torch.empty(1, 2, self.queries, device="cuda")
        self.layer.forward(self.place(q), self.place(k), self.place(v), o, lse)
        return o, lse

    def backward(self, q, k, v, o, d_o, lse):
        out = [self.place(torch.zeros_like(t)) for t in (q, k, v)]
        self.layer.backward(*(self.place(t) for t in (q, k, v, o, d_o)), lse, *out)
        return out


LAYOUTS = pytest.mark.parametrize("layout", ["aligned", "odd"])


@DIMS
@WAYS
@LAYOUTS
def test_scores(queries, keys, dim, layout):
    """The logarithm is the score of the only key: one product."""
    c = Case(queries, keys, dim, layout, 1.0)
    q, k = c.one_element(), c.normal(keys, 2)
    _, lse = c.forward(q, k, c.normal(keys, 2))
    score = (q.double() * c.of_queries(k).double()).sum(3)[0].T[None]
    ref.check(lse, score, planes.LOGARITHM * ref.U * score.abs() + planes.LOGARITHM_ADDS * ref.U, "lse")


@DIMS
@WAYS
@LAYOUTS
def test_outputs(queries, keys, dim, layout):
    """Two keys with the same value: the output is that value."""
    c = Case(queries, keys, dim, layout, dim ** -0.5, more=1)
    value = c.normal(1, 2)
    o, _ = c.forward(c.normal(queries, 2), c.normal(keys, 2), value.expand(1, keys, 2, dim).contiguous())
    ref.check(o, value.double().expand_as(o), planes.OUTPUT * ref.U * value.double().abs().expand_as(o), "o")


def _small_scores(c):
    """Queries, keys, and logarithms of up to 1 in magnitude, beside scores whose error is far below U (2^-14 of sums of `dim` products)."""
    q, k = c.normal(c.queries, 2), c.normal(c.keys, c.key_heads)
    score = (q.double() * c.of_queries(k).double()).sum(3)[0].T[None] * 2.0 ** -14
    lse = torch.empty(1, 2, c.queries, device="cuda").uniform_(-0.9, 0.9, generator=c.g)
    p = torch.exp(score - lse.double())
    return q, k, lse, p.transpose(1, 2)[..., None]  # samples, tokens, heads, 1


def _of_keys(c, t):
    """Numbers of the queries summed over the heads that share a key head, at their keys."""
    out = torch.zeros(1, c.keys, c.key_heads, c.dim, dtype=torch.float64, device="cuda")
    out[:, c.own] = t.view(1, c.queries, c.key_heads, 2 // c.key_heads, c.dim).sum(3)
    return out


@DIMS
@WAYS
@LAYOUTS
@pytest.mark.parametrize("key_heads", [1, 2])
def test_gradients_of_values(queries, keys, dim, layout, key_heads):
    """dv = p d_o."""
    c = Case(queries, keys, dim, layout, 2.0 ** -14, key_heads=key_heads)
    q, k, lse, p = _small_scores(c)
    d_o = c.normal(queries, 2)
    dv = c.backward(q, k, c.normal(keys, key_heads), torch.zeros_like(q), d_o, lse)[2]
    want = p * d_o.double()
    ref.check(dv, _of_keys(c, want), (planes.VALUES + 4) * ref.U * _of_keys(c, want.abs()), "dv")


@DIMS
@WAYS
@LAYOUTS
@pytest.mark.parametrize("key_heads", [1, 2])
def test_gradients_of_queries_and_keys(queries, keys, dim, layout, key_heads):
    """With an output of zero ds = p (d_o v), one product where d_o has one element; dq = ds k, dk = ds q."""
    c = Case(queries, keys, dim, layout, 2.0 ** -14, key_heads=key_heads)
    q, k, lse, p = _small_scores(c)
    v, d_o = c.normal(keys, key_heads), c.one_element()
    dq, dk, _ = c.backward(q, k, v, torch.zeros_like(q), d_o, lse)
    ds = p * (d_o.double() * c.of_queries(v).double()).sum(3, keepdim=True) * 2.0 ** -14
    want = ds * c.of_queries(k).double()
    ref.check(dq, want, planes.QUERIES * ref.U * want.abs(), "dq")
    want = ds * q.double()
    ref.check(dk, _of_keys(c, want), (planes.QUERIES + 4) * ref.U * _of_keys(c, want.abs()), "dk")
