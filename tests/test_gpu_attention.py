"""Attention, forward and backward, against the plain form in 64 bits, with bounds derived in tests/token_reference.py."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


class Problem:
    def __init__(self, n, queries, keys, heads, key_heads, dim, dtype, window=(None, None), lengths=None, scale=None, seed=0, layout="tokens",
                 magnitude=1.0):
        from dihydrogen_amd.tokens import Attention
        g = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: torch.empty(*s, device="cuda").normal_(0, magnitude, generator=g).to(dtype)
        q, k, v, d_o = make(n, queries, heads, dim), make(n, keys, key_heads, dim), make(n, keys, key_heads, dim), make(n, queries, heads, dim)
        self.layer = Attention(scale=scale, window=window)
        self.dtype, self.scale = dtype, dim ** -0.5 if scale is None else scale
        self.lengths = {}
        query_lengths, key_lengths = lengths if lengths else (None, None)
        for name, l, t, most in (("query_lengths", query_lengths, (q, d_o), queries), ("key_lengths", key_lengths, (k, v), keys)):
            if l is not None:
                self.lengths[name] = torch.tensor(l, dtype=torch.int32, device="cuda")
                for x in t:  # what lies behind a sample may hold anything
                    for b in range(n):
                        x[b, min(max(l[b], 0), most):] = math.nan
        gap, offset, order = {"tokens": (0, 0, (0, 1, 2, 3)), "heads first": (0, 0, (0, 2, 1, 3)), "gaps": (8, 8, (0, 1, 2, 3)),
                              "samples inside": (16, 0, (1, 0, 2, 3)), "odd": (3, 1, (0, 2, 1, 3))}[layout]
        place = lambda t, fill: ref.ragged(t.shape, dtype, fill, gap=gap, offset=offset, order=order)
        self.inputs = []
        for t in (q, k, v, d_o):
            view = place(t, math.nan)[1]
            self.inputs.append(view.copy_(t))
        self.outputs = [place(t, 7.0) for t in (q, q, k, k)]  # o, dq, dk, dv
        self.lse = torch.full((n, heads, queries), math.nan, device="cuda")
        self.seen = ref.visible(n, queries, keys, *window, query_lengths, key_lengths)
        self.want = ref.AttentionReference(q, k, v, self.scale, self.seen)
        self.d_o = d_o

    def forward(self):
        q, k, v, _ = self.inputs
        self.layer.forward(q, k, v, self.outputs[0][1], self.lse, **self.lengths)
        return self.outputs[0][1], self.lse

    def backward(self):
        o, dq, dk, dv = (t[1] for t in self.outputs)
        self.layer.backward(*self.inputs[:3], o, self.inputs[3], self.lse, dq, dk, dv, **self.lengths)
        return dq, dk, dv

    def check_forward(self):
        o, lse = self.forward()
        bo, bl = self.want.forward_bounds(self.dtype)
        ref.check(o, self.want.o.transpose(1, 2), bo.transpose(1, 2), "o")
        empty = ~self.seen.any(2).to(o.device)[:, None].expand_as(lse)
        assert bool((lse[empty] == -math.inf).all()) and bool((o.transpose(1, 2)[empty] == 0).all())
        ref.check(lse[~empty], self.want.lse[~empty], bl.expand_as(lse)[~empty], "lse")
        assert ref.outside_untouched(*self.outputs[0], 7.0)

    def check(self):
        self.check_forward()
        got = self.backward()
        for name, g, (want, bound), out in zip(("dq", "dk", "dv"), got, self.want.gradients(self.d_o, self.outputs[0][1], self.lse, self.dtype),
                                              self.outputs[1:]):
            ref.check(g, want, bound, name)
            assert ref.outside_untouched(*out, 7.0), name
        # keys that no query sees, and queries that see no key, have no gradient
        assert bool((got[0].transpose(1, 2)[~self.seen.any(2).to(got[0].device)[:, None].expand(-1, got[0].shape[2], -1)] == 0).all())
        unseen = ~self.seen.any(1).to(got[0].device)
        assert bool((got[1][unseen] == 0).all()) and bool((got[2][unseen] == 0).all())


DTYPES = pytest.mark.parametrize("dtype", [BF16, F32], ids=["bf16", "f32"])


@DTYPES
@pytest.mark.parametrize("dim", [1, 8, 20, 32, 40, 64, 72, 80, 96, 100, 121, 128])
def test_head_sizes(dtype, dim):
    Problem(2, 70, 75, 4, 2, dim, dtype, window=(None, 0)).check()
    Problem(1, 5, 200, 6, 2, dim, dtype).check()


@DTYPES
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 2), (2, 1), (1, 63), (1, 64), (1, 65), (3, 129), (16, 300), (17, 300), (31, 32), (32, 31),
                                          (33, 33), (64, 64), (65, 64), (127, 129), (128, 128), (129, 257), (300, 40), (513, 511)])
def test_lengths(dtype, queries, keys):
    for window in ((None, None), (None, 0), (7, 3), (0, 0)):
        Problem(2, queries, keys, 2, 1, 64, dtype, window=window, seed=queries).check()


@DTYPES
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (3, 3), (8, 2), (7, 1), (64, 1)])
def test_shared_heads(dtype, heads, key_heads):
    Problem(2, 40, 50, heads, key_heads, 32, dtype, window=(None, 0)).check()
    Problem(3, 1, 333, heads, key_heads, 128, dtype, window=(None, 0)).check()
    Problem(1, 9, 70, heads, key_heads, 64, dtype, window=(20, 0)).check()


@DTYPES
@pytest.mark.parametrize("layout", ["heads first", "gaps", "samples inside", "odd"])
@pytest.mark.parametrize("queries", [3, 90])
def test_layouts(dtype, layout, queries):
    for dim in (64, 80):
        Problem(3, queries, 100, 4, 2, dim, dtype, window=(None, 0), layout=layout).check()


@DTYPES
@pytest.mark.parametrize("window", [(None, None), (None, 0), (30, 10), (5, None)])
@pytest.mark.parametrize("queries,keys,query_lengths,key_lengths", [
    (150, 150, [150, 1, 0, 77], [150, 1, 0, 77]),     # a padded batch
    (140, 90, [140, 10, 140, 3], [90, 90, 0, 2]),     # more queries than keys: rows that see nothing; no keys at all
    (2, 500, None, [500, 0, 64, 65]),                 # caches of unlike lengths
    (4, 300, [4, 0, 1, 3], [1, 300, 299, 2]),
    (33, 64, [-5, 40, 33, 0], [64, 70, 1, -1]),       # beyond what the tensors hold: clamped
])
def test_samples_of_unlike_lengths(dtype, window, queries, keys, query_lengths, key_lengths):
    Problem(4, queries, keys, 4, 2, 64, dtype, window=window, lengths=(query_lengths, key_lengths)).check()


@DTYPES
def test_no_keys_no_queries(dtype):
    Problem(2, 5, 0, 2, 2, 32, dtype).check()
    Problem(2, 40, 0, 2, 2, 32, dtype).check()
    Problem(2, 0, 40, 2, 2, 32, dtype).check()
    Problem(0, 4, 40, 2, 2, 32, dtype).check()


@DTYPES
@pytest.mark.parametrize("queries,keys,heads,key_heads,n", [(1, 9000, 4, 1, 1), (2, 20000, 2, 2, 1), (16, 5000, 4, 2, 2), (40, 9000, 2, 1, 1),
                                                           (130, 4500, 1, 1, 1)])
def test_keys_in_parts(dtype, queries, keys, heads, key_heads, n):
    """Few workgroups and many keys: the keys are shared out and the parts joined, some of them empty."""
    for window, lengths in (((None, 0), None), ((100, 0), None), ((None, 0), (None, [keys - 4000] * n)), ((None, 0), (None, [3] * n))):
        p = Problem(n, queries, keys, heads, key_heads, 64, dtype, window=window, lengths=lengths)
        p.check()


@DTYPES
@pytest.mark.parametrize("queries,keys,heads,key_heads,dim,n", [(2500, 100, 4, 1, 64, 1), (70, 4500, 2, 2, 40, 1), (1500, 1300, 8, 1, 128, 1),
                                                                (1100, 1100, 3, 1, 72, 2)])
def test_gradients_in_parts(dtype, queries, keys, heads, key_heads, dim, n):
    """Few blocks of rows and many of the other side: shared out, and summed in order; some parts empty."""
    for window, lengths in (((None, None), None), ((None, 0), None), ((200, 30), None),
                            ((None, 0), ([max(1, queries - 90)] * n, [keys - 60] * n)), ((None, None), ([5] * n, [3] * n))):
        p = Problem(n, queries, keys, heads, key_heads, dim, dtype, window=window, lengths=lengths, layout="gaps")
        p.check()
        first = [t[1].clone() for t in p.outputs[1:]]
        assert all(torch.equal(a, b) for a, b in zip(first, p.backward()))


@DTYPES
@pytest.mark.parametrize("magnitude", [0.01, 30.0])
def test_sharp_and_flat_rows(dtype, magnitude):
    """Scores of a few thousandths, and of hundreds: one key takes all."""
    Problem(1, 70, 200, 2, 1, 64, dtype, window=(None, 0), magnitude=magnitude ** 0.5, scale=0.125 * magnitude).check()
    Problem(1, 3, 200, 2, 1, 64, dtype, magnitude=magnitude ** 0.5, scale=0.125 * magnitude).check()


@DTYPES
def test_rising_scores(dtype):
    """Every key outweighs those before it: the running maximum moves at every tile."""
    for queries in (2, 40):
        p = Problem(1, queries, 700, 1, 1, 32, dtype)
        q, k = p.inputs[0], p.inputs[1]
        q.fill_(1.0)
        k.copy_((torch.arange(700, device="cuda") * 0.02)[None, :, None, None].expand_as(k).to(dtype))
        p.want = ref.AttentionReference(q, k, p.inputs[2], p.scale, p.seen)
        p.check()


@DTYPES
def test_what_no_query_sees_may_hold_anything(dtype):
    """Keys before a window's reach and behind the last query's, a tile or a few keys of them, within the sample's lengths."""
    for queries, window in ((1, (20, 0)), (3, (70, 0)), (40, (10, 0)), (130, (100, 0)), (1, (0, 0))):
        p = Problem(2, queries, 300, 4, 2, 64, dtype, window=window)
        q, k, v, _ = p.inputs
        unseen = ~p.seen.any(1)[0].cuda()
        assert bool(unseen.any())
        clean = [t.clone() for t in (k, v)]
        for t in (k, v):
            t[:, unseen] = torch.tensor([math.nan, math.inf, -math.inf, 1e30], device="cuda").repeat(128)[:int(unseen.sum())].to(dtype)[:, None, None]
        p.check()
        k.copy_(clean[0]), v.copy_(clean[1])


def test_outputs_that_lie_on_themselves_are_refused():
    from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions
    x = torch.ones(2, 3, 4, 8, device="cuda")
    flat = torch.ones(2, 3, 1, 8, device="cuda").expand(2, 3, 4, 8)
    with pytest.raises(ValueError):
        Attention().forward(x, x, x, flat)
    with pytest.raises(ValueError):
        LayerNormalization().forward(x, None, None, flat)
    with pytest.raises(ValueError):
        RotaryPositions(8, [4]).forward(x, torch.zeros(1, 3, dtype=torch.int32, device="cuda"), flat)
    o = torch.empty_like(x)
    Attention().forward(flat, flat, flat, o)  # as inputs they are fine
    assert bool((o == 1).all())


def test_more_than_32_bits_of_offsets():
    """A cache of one sample whose last keys lie beyond 2^31 elements, and 2^32 bytes."""
    from dihydrogen_amd.tokens import Attention
    keys, dim = 34000, 64
    stride = 1024 * dim  # tokens of a cache with many heads, of which this is one
    assert (keys - 1) * stride > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(5)
    buffers = [torch.zeros(keys * stride, dtype=BF16, device="cuda") for _ in range(2)]
    k, v = (b.as_strided((1, keys, 1, dim), (keys * stride, stride, dim, 1)) for b in buffers)
    small = [torch.empty(1, keys, 1, dim, device="cuda").normal_(0, 1, generator=g).to(BF16) for _ in range(2)]
    k.copy_(small[0]), v.copy_(small[1])
    layer = Attention(causal=True)
    for queries in (1, 60):
        q = torch.empty(1, queries, 2, dim, device="cuda").normal_(0, 1, generator=g).to(BF16)
        d_o = torch.randn_like(q)
        outs = []
        for a, b in ((k, v), small):
            o, lse, dq = torch.empty_like(q), torch.empty(1, 2, queries, device="cuda"), torch.empty_like(q)
            dk, dv = torch.empty_like(small[0]), torch.empty_like(small[0])
            layer.forward(q, a, b, o, lse)
            layer.backward(q, a, b, o, d_o, lse, dq, dk, dv)
            outs.append((o, lse, dq, dk, dv))
        assert all(torch.equal(x, y) for x, y in zip(*outs))


@DTYPES
def test_same_bits_every_time(dtype):
    p = Problem(2, 700, 700, 8, 2, 64, dtype, window=(None, 0), seed=3)
    first = None
    for _ in range(3):
        p.forward()
        now = [t.clone() for t in (p.outputs[0][1], p.lse, *p.backward())]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(now, first))


def test_gradients_against_differences():
    """The kernels' own forward pass in 32 bits, along random directions.  The loss is a sum of 2 * 11 * 3 * 16 products of size 1, so its
    error is about 1e-6 of 30, and the difference's 3e-5 / (2 * step); the step's own error goes with its square."""
    p = Problem(2, 11, 13, 3, 3, 16, F32, window=(None, 2))
    p.forward()
    gradients = [t.clone() for t in p.backward()]
    base = [t.clone() for t in p.inputs[:3]]
    step = 0.03
    for which in range(3):
        d = torch.randn_like(base[which])
        d /= d.norm()
        loss = []
        for sign in (1, -1):
            p.inputs[which].copy_(base[which] + sign * step * d)
            loss.append(float((p.forward()[0].double() * p.d_o.double()).sum()))
        p.inputs[which].copy_(base[which])
        assert abs((loss[0] - loss[1]) / (2 * step) - float((gradients[which] * d).sum())) < 5e-3
