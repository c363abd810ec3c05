"""The token operators together, as a transformer block over a volume uses them: layer normalisation, projections (torch's products),
rotary positions over three axes, attention, and back through all of it; against the same chain in 64 bits by torch's own gradients.  And
the same calls on another stream beside busy ones, from two graphs, and refused."""
import ctypes
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu


class Block:
    """x (samples, tokens, channels) -> projection of attention of the normalised x."""

    def __init__(self, n, grid, heads, key_heads, dim, dtype, stream=None, causal=False, seed=0):
        from dihydrogen_amd.tensor import Distribution, LocaleVirtual, Tensor
        from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions, grid_positions
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.n, self.tokens, self.heads, self.key_heads, self.dim, self.dtype = n, math.prod(grid), heads, key_heads, dim, dtype
        self.channels, self.generator = heads * dim, g
        make = lambda *s: torch.empty(*s, device="cuda").normal_(0, 1, generator=g)
        self.x, self.dy = make(n, self.tokens, self.channels).to(dtype), make(n, self.tokens, self.channels).to(dtype)
        width = (heads + 2 * key_heads) * dim
        self.w_qkv = (make(self.channels, width) / self.channels ** 0.5).to(dtype)
        self.w_out = (make(self.channels, self.channels) / self.channels ** 0.5).to(dtype)
        self.scale, self.bias = 1 + 0.1 * make(self.channels), 0.1 * make(self.channels)
        self.positions = grid_positions(Tensor(list(reversed(grid)) + [1, 1], LocaleVirtual(0, 1),
                                               Distribution.make_localized_distribution(len(grid) + 2)))
        pairs = dim // 2 // len(grid)
        self.norm = LayerNormalization(1e-5, stream=stream)
        self.turn = RotaryPositions(dim, [pairs] * len(grid), stream=stream)
        self.attention = Attention(causal=causal, stream=stream)

    def step(self):
        """Output, and gradients of x, both products' weights, scale and bias."""
        n, t, h, kh, d = self.n, self.tokens, self.heads, self.key_heads, self.dim
        e = lambda *s: torch.empty(*s, dtype=self.dtype, device="cuda")
        f = lambda *s: torch.empty(*s, device="cuda")
        normed, mean, rstd = e(n, t, self.channels), f(n, t), f(n, t)
        self.norm.forward(self.x, self.scale, self.bias, normed, mean, rstd)
        qkv = (normed.view(-1, self.channels) @ self.w_qkv).view(n, t, h + 2 * kh, d)
        q, k, v = qkv.split([h, kh, kh], 2)
        turned = qkv[:, :, :h + kh]
        self.turn.forward(turned, self.positions, turned)  # queries and keys at once, in place
        o, lse = e(n, t, h, d), f(n, h, t)
        self.attention.forward(q, k, v, o, lse)
        y = o.view(-1, self.channels) @ self.w_out
        dy = self.dy.view(-1, self.channels)
        d_w_out = o.view(-1, self.channels).t() @ dy
        d_o = (dy @ self.w_out.t()).view(n, t, h, d)
        d_qkv = e(n, t, h + 2 * kh, d)
        dq, dk, dv = d_qkv.split([h, kh, kh], 2)
        self.attention.backward(q, k, v, o, d_o, lse, dq, dk, dv)
        d_turned = d_qkv[:, :, :h + kh]
        self.turn.backward(d_turned, self.positions, d_turned)
        flat = d_qkv.view(n * t, -1)
        d_w_qkv = normed.view(-1, self.channels).t() @ flat
        d_normed = (flat @ self.w_qkv.t()).view(n, t, self.channels)
        dx, d_scale, d_bias = e(n, t, self.channels), f(self.channels), f(self.channels)
        self.norm.backward(self.x, d_normed, mean, rstd, self.scale, dx, d_scale, d_bias)
        return y.view(n, t, self.channels), dx, d_w_qkv, d_w_out, d_scale, d_bias

    def reference(self):
        n, t, h, kh, d = self.n, self.tokens, self.heads, self.key_heads, self.dim
        leaf = lambda a: a.double().requires_grad_(True)
        x, wq, wo, s, b = (leaf(a) for a in (self.x, self.w_qkv, self.w_out, self.scale, self.bias))
        c = x - x.mean(-1, keepdim=True)
        normed = c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * s + b
        qkv = (normed @ wq).view(n, t, h + 2 * kh, d)
        m = d // 2 // self.positions.shape[0] * self.positions.shape[0]
        axis = [a for a in range(self.positions.shape[0]) for _ in range(m // self.positions.shape[0])]
        angle = (self.positions.double()[axis].T * self.turn.frequencies.cuda())[None, :, None]
        z = qkv[:, :, :h + kh]
        u, w, rest = z[..., :m], z[..., m:2 * m], z[..., 2 * m:]
        z = torch.cat([u * angle.cos() - w * angle.sin(), u * angle.sin() + w * angle.cos(), rest], -1).transpose(1, 2)
        q, k = z[:, :h], z[:, h:].repeat_interleave(h // kh, 1)
        v = qkv[:, :, h + kh:].transpose(1, 2).repeat_interleave(h // kh, 1)
        score = q @ k.transpose(2, 3) * d ** -0.5
        if self.attention.window[1] == 0:
            score = score.masked_fill(torch.ones(t, t, device="cuda", dtype=torch.bool).triu(1), -math.inf)
        y = (torch.softmax(score, -1) @ v).transpose(1, 2).reshape(n, t, -1) @ wo
        (y * self.dy.double()).sum().backward()
        return y.detach(), x.grad, wq.grad, wo.grad, s.grad, b.grad


@pytest.mark.parametrize("dtype,steps", [(torch.float32, 400), (torch.bfloat16, 10)], ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_block_against_64_bits(dtype, steps, causal):
    """A chain of about ten roundings to the elements' type, each of half a step of values that go into sums: together a few half steps of
    the results' root mean square (`steps` of them; float32 also accumulates hundreds of terms in 32 bits in every product)."""
    block = Block(2, (3, 6, 8), 6, 2, 24, dtype, causal=causal)
    for name, got, want in zip(("y", "dx", "dw_qkv", "dw_out", "dscale", "dbias"), block.step(), block.reference()):
        error = (got.double() - want).square().mean().sqrt()
        assert error <= steps * ref.half_step(dtype) * want.square().mean().sqrt(), (name, float(error))


def test_on_a_stream_beside_busy_ones():
    expected = [t.clone() for t in Block(2, (4, 8, 8), 4, 2, 32, torch.bfloat16, causal=True).step()]
    stream = torch.cuda.Stream()
    block = Block(2, (4, 8, 8), 4, 2, 32, torch.bfloat16, stream=stream, causal=True)
    torch.cuda.synchronize()
    a = torch.randn(4096, 4096, device="cuda")
    for _ in range(20):
        a = (a @ a).clamp_(-1, 1)  # the default stream is busy
    with torch.cuda.stream(stream):
        got = block.step()
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, expected))
    # layers without a stream of their own go to the current one
    block = Block(2, (4, 8, 8), 4, 2, 32, torch.bfloat16, causal=True)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = block.step()
    stream.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, expected))


def test_two_graphs_of_the_same_layers_at_once():
    """Graphs captured from the same layers share no workspace: their replays may overlap.  Every replay equals the eager result."""
    from dihydrogen_amd.tokens import Attention, LayerNormalization
    attention, norm = Attention(causal=True), LayerNormalization()
    g = torch.Generator(device="cuda").manual_seed(0)
    make = lambda *s: torch.empty(*s, device="cuda").normal_(0, 1, generator=g).to(torch.bfloat16)

    class Work:
        def __init__(self):
            self.q, self.k, self.v = make(2, 1, 4, 64), make(2, 8000, 2, 64), make(2, 8000, 2, 64)  # keys in parts
            self.x, self.dy = make(700, 320), make(700, 320)
            self.tq, self.tk, self.tv, self.d_o = make(1, 300, 4, 64), make(1, 300, 2, 64), make(1, 300, 2, 64), make(1, 300, 4, 64)
            self.o, self.y, self.dx = torch.empty_like(self.q), torch.empty_like(self.x), torch.empty_like(self.x)
            self.mean, self.rstd = torch.empty(700, device="cuda"), torch.empty(700, device="cuda")
            self.w, self.dw, self.db = torch.ones(320, device="cuda"), torch.empty(320, device="cuda"), torch.empty(320, device="cuda")
            self.to, self.lse = torch.empty_like(self.tq), torch.empty(1, 4, 300, device="cuda")
            self.grads = [torch.empty_like(t) for t in (self.tq, self.tk, self.tv)]

        def step(self):
            attention.forward(self.q, self.k, self.v, self.o)
            norm.forward(self.x, self.w, None, self.y, self.mean, self.rstd)
            norm.backward(self.x, self.dy, self.mean, self.rstd, self.w, self.dx, self.dw, self.db)
            attention.forward(self.tq, self.tk, self.tv, self.to, self.lse)
            attention.backward(self.tq, self.tk, self.tv, self.to, self.d_o, self.lse, *self.grads)

        def outputs(self):
            return [t.clone() for t in (self.o, self.y, self.dx, self.dw, self.db, self.to, self.lse, *self.grads)]

    works = [Work(), Work()]
    for w in works:
        w.step()
    torch.cuda.synchronize()
    graphs = []
    for w in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.step()
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in works]
    for turn in range(4):
        for w in works:
            for t in (w.q, w.k, w.v, w.x, w.dy, w.tq, w.d_o):
                t.copy_(make(*t.shape))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for w in works:
            replayed = w.outputs()
            w.step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(replayed, w.outputs())), turn


def test_calls_on_two_streams_at_once():
    from dihydrogen_amd.tokens import Attention
    layer = Attention()
    make = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
    q, k, v = ([make(1, 2, 4, 128) for _ in range(2)], [make(1, 30000, 1, 128) for _ in range(2)], [make(1, 30000, 1, 128) for _ in range(2)])
    want = [torch.empty_like(t) for t in q]
    for i in range(2):
        layer.forward(q[i], k[i], v[i], want[i])
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[torch.empty_like(q[i]) for _ in range(10)] for i in range(2)]
    torch.cuda.synchronize()
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                layer.forward(q[i], k[i], v[i], got[i][turn])
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_refusals_launch_nothing():
    """What the C ABI refuses leaves real buffers alone (the list of refusals: tests/test_host_token_refusals.py)."""
    from dihydrogen_amd import capi
    lib = capi.load()
    out = torch.full((64, 64), 7.0, device="cuda")
    x = torch.ones(64, 64, device="cuda")
    p, o = x.data_ptr(), out.data_ptr()
    assert lib.h2x_layer_norm_forward(capi.F32, capi.F64, 64, 64, None, None, p, None, None, o, None, None, 1e-5, None) == -2
    assert lib.h2x_layer_norm_forward(capi.F32, capi.F32, 64, 64, None, None, p, None, None, o, o, None, 1e-5, None) == -1
    assert lib.h2x_layer_norm_backward(capi.F32, capi.F32, 64, 64, None, None, None, p, p, p, p, p, o, o, o, None, None) == -1
    r = capi.Rotary()
    r.head_dim, r.heads, r.samples, r.num_axes, r.tokens = 64, 1, 1, 1, 64
    r.axis_pairs[0] = 33
    assert lib.h2x_rotary_apply(ctypes.byref(r), p, p, p, 0, o, None) == -1
    a = capi.Attention()
    a.dtype, a.head_dim, a.samples, a.query_heads, a.key_heads, a.queries, a.keys, a.scale = capi.F16, 64, 1, 1, 1, 64, 64, 1.0
    for name in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
        setattr(a, name, capi.TokenStrides(0, 64, 0))
    assert lib.h2x_attention_forward(ctypes.byref(a), p, p, p, None, None, o, None, None, None) == -2
    a.dtype, a.dk = capi.F32, capi.TokenStrides(0, 63, 0)
    assert lib.h2x_attention_backward(ctypes.byref(a), p, p, p, p, p, p, None, None, o, o, o, p, None) == -1
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())


def test_layers_refuse_what_is_elsewhere():
    from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions
    x, host = torch.ones(2, 3, 4, 8, device="cuda"), torch.ones(2, 3, 4, 8)
    with pytest.raises(ValueError):
        LayerNormalization().forward(x, None, None, host)
    with pytest.raises(ValueError):
        Attention().forward(x, x, host, x)
    with pytest.raises(ValueError):
        RotaryPositions(8, [4]).forward(x, torch.zeros(1, 3, dtype=torch.int32), x)
