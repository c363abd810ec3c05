"""Calls of the token operators that have to be refused, by the C ABI before any launch and by the Python
layers with an error that says why.  (No kernel runs: pointers are imaginary, and the file is skipped where a GPU is
visible.)"""
import ctypes

import pytest
import torch

from dihydrogen_amd import capi

INVALID, UNSUPPORTED, TOO_LARGE = -1, -2, -3
P = ctypes.c_void_p(1 << 20)


@pytest.fixture(autouse=True)
def no_gpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: valid calls would launch on imaginary pointers")


def _geometry(shape, strides):
    g = capi.TensorGeometry()
    g.num_dims = len(shape)
    for i, (e, s) in enumerate(zip(shape, strides)):
        g.local_shape[i], g.strides[i] = e, s
    return ctypes.byref(g)


def test_layer_norm():
    lib = capi.load()
    F, B, O = lib.h2x_layer_norm_forward, lib.h2x_layer_norm_backward, ctypes.c_void_p(2 << 20)

    def fwd(dtype=capi.F32, weights=capi.F32, rows=4, c=8, xg=None, yg=None, x=P, y=P, mean=P, rstd=P, eps=1e-5):
        return F(dtype, weights, rows, c, xg, yg, x, P, P, y, mean, rstd, eps, None)

    assert fwd() > 0  # HIP's own error: there is no GPU
    assert fwd(dtype=4) == UNSUPPORTED and fwd(dtype=-1) == UNSUPPORTED
    assert fwd(weights=capi.F64) == UNSUPPORTED and fwd(weights=capi.BF16) == UNSUPPORTED
    assert fwd(dtype=capi.F64, weights=capi.F32) == UNSUPPORTED and fwd(dtype=capi.F16, weights=capi.BF16) == UNSUPPORTED
    assert fwd(c=0) == INVALID and fwd(c=-3) == INVALID and fwd(eps=-1.0) == INVALID and fwd(eps=float("nan")) == INVALID
    assert fwd(mean=None) == INVALID and fwd(rstd=None) == INVALID and fwd(x=None) == INVALID and fwd(y=None) == INVALID
    assert fwd(rows=1 << 31) == TOO_LARGE and fwd(c=(1 << 26) + 1) == TOO_LARGE
    assert fwd(rows=0, x=None, y=None, mean=None, rstd=None) == 0
    assert fwd(xg=_geometry((8, 4), (1, 8))) > 0
    assert fwd(xg=_geometry((8, 4), (1, 16))) == INVALID  # in place, but laid out otherwise
    assert fwd(xg=_geometry((8, 4), (1, 16)), y=ctypes.c_void_p(2 << 20)) > 0
    assert B(capi.F32, capi.F32, 4, 8, None, _geometry((8, 4), (1, 16)), None, P, O, P, P, P, O, None, None, None, None) == INVALID
    assert fwd(xg=_geometry((8, 5), (1, 8))) == INVALID  # not four rows
    assert fwd(xg=_geometry((7, 4), (1, 8))) == INVALID and fwd(yg=_geometry((8, 4), (2, 8))) == INVALID
    assert fwd(xg=_geometry((8, 4, -1), (1, 8, 8))) == INVALID
    assert fwd(xg=_geometry((8,) * 6, (1,) * 6)) == INVALID
    assert B(capi.F32, capi.F32, 4, 8, None, None, None, P, P, P, P, P, P, P, P, None, None) == INVALID  # no workspace
    assert B(capi.F32, capi.F32, 4, 8, None, None, None, P, P, None, P, P, P, None, None, None, None) == INVALID
    assert B(capi.F32, capi.F32, 4, 8, None, None, None, P, P, P, P, P, None, None, None, None, None) == 0  # nothing asked for
    assert lib.h2x_layer_norm_workspace_bytes(9, 4, 8) == 0 and lib.h2x_layer_norm_workspace_bytes(capi.F32, 4, 0) == 0
    assert lib.h2x_layer_norm_workspace_bytes(capi.F32, 0, 8) >= 2 * 8 * 4


def _rotary(**changes):
    r = capi.Rotary()
    r.dtype, r.pairing, r.head_dim, r.heads, r.samples, r.num_axes, r.tokens = capi.F32, 0, 8, 2, 1, 2, 3
    r.axis_pairs[:2] = [2, 1]
    r.positions_axis_stride = 3
    r.x = r.y = capi.TokenStrides(48, 16, 8)
    for name, value in changes.items():
        if name == "axis_pairs":
            r.axis_pairs[:len(value)] = value
        else:
            setattr(r, name.split("_strides")[0], value)
    return r


def test_rotary():
    F = capi.load().h2x_rotary_apply

    def call(x=P, positions=P, frequencies=P, y=P, **changes):
        return F(ctypes.byref(_rotary(**changes)), x, positions, frequencies, 0, y, None)

    assert call() > 0
    assert F(None, P, P, P, 0, P, None) == INVALID
    assert call(dtype=7) == UNSUPPORTED and call(head_dim=257) == UNSUPPORTED
    assert call(head_dim=5) == INVALID and call(axis_pairs=[3, 2]) == INVALID and call(axis_pairs=[-1, 2]) == INVALID
    assert call(axis_pairs=[2 ** 31 - 1, 2 ** 31 - 1]) == INVALID
    assert call(num_axes=5) == INVALID and call(num_axes=-1) == INVALID and call(pairing=2) == INVALID
    assert call(heads=-1) == INVALID and call(samples=-1) == INVALID and call(tokens=-1) == INVALID
    assert call(tokens=1 << 31) == TOO_LARGE
    assert call(y_strides=capi.TokenStrides(48, 8, 24)) == INVALID  # in place, but laid out otherwise
    assert call(y_strides=capi.TokenStrides(48, 8, 24), y=ctypes.c_void_p(2 << 20)) > 0
    assert call(x=None) == INVALID and call(y=None) == INVALID and call(positions=None) == INVALID and call(frequencies=None) == INVALID
    assert call(tokens=0, x=None, y=None) == 0 and call(heads=0) == 0 and call(samples=0) == 0


def _attention(**changes):
    a = capi.Attention()
    a.dtype, a.head_dim, a.samples, a.query_heads, a.key_heads, a.queries, a.keys = capi.BF16, 64, 2, 4, 2, 40, 50
    a.window_left, a.window_right, a.scale = -1, 0, 0.125
    for name, heads, tokens in (("q", 4, 40), ("o", 4, 40), ("d_o", 4, 40), ("dq", 4, 40), ("k", 2, 50), ("v", 2, 50), ("dk", 2, 50),
                                ("dv", 2, 50)):
        setattr(a, name, capi.TokenStrides(tokens * heads * 64, heads * 64, 64))
    for name, value in changes.items():
        setattr(a, name.split("_strides")[0], value)
    return a


def test_attention():
    lib = capi.load()

    O, A, B, C = (ctypes.c_void_p(i << 20) for i in (2, 3, 4, 5))

    def fwd(q=P, k=P, v=P, o=O, ws=None, **changes):
        return lib.h2x_attention_forward(ctypes.byref(_attention(**changes)), q, k, v, None, None, o, P, ws, None)

    def bwd(q=P, lse=P, dq=A, dv=B, ws=P, **changes):
        return lib.h2x_attention_backward(ctypes.byref(_attention(**changes)), q, P, P, P, P, lse, None, None, dq, C, dv, ws, None)

    for call in (fwd, bwd):
        assert call() > 0, call
        assert call(dtype=capi.F16) == UNSUPPORTED and call(dtype=capi.F64) == UNSUPPORTED and call(dtype=9) == UNSUPPORTED
        assert call(head_dim=129) == UNSUPPORTED and call(head_dim=0) == INVALID
        assert call(key_heads=3) == INVALID and call(key_heads=0) == INVALID and call(samples=-1) == INVALID
        assert call(queries=-1) == INVALID and call(keys=-1) == INVALID
        assert call(queries=2 ** 31 - 1) == TOO_LARGE and call(keys=2 ** 31 - 1) == TOO_LARGE
        for scale in (0.0, -1.0, float("nan"), float("inf")):
            assert call(scale=scale) == INVALID
        assert call(k_strides=capi.TokenStrides(0, 63, 0)) == INVALID  # tokens on one another
        assert call(k_strides=capi.TokenStrides(0, (1 << 21) + 1, 0)) == UNSUPPORTED
        assert call(q=None) == INVALID
        assert call(queries=0, keys=0) == 0 and call(samples=0) == 0 and call(query_heads=0, key_heads=0) == 0
    assert lib.h2x_attention_forward(None, P, P, P, None, None, P, P, None, None) == INVALID
    assert fwd(o=None) == INVALID
    assert fwd(o=O) > 0 and fwd(o=P) == INVALID
    a = _attention()
    a.o = capi.TokenStrides(4 * 64, 4 * 64, 32)  # heads of the output on one another
    assert lib.h2x_attention_forward(ctypes.byref(a), P, P, P, None, None, P, P, None, None) == INVALID
    assert bwd(lse=None) == INVALID and bwd(dq=None) == INVALID and bwd(dv=None) == INVALID and bwd(ws=None) == INVALID
    # outputs where inputs or other outputs lie
    others = [ctypes.c_void_p((i + 2) << 20) for i in range(8)]
    run = lambda p: lib.h2x_attention_backward(ctypes.byref(_attention()), *p[:5], P, None, None, *p[5:], P, None)
    assert run(others) > 0
    for out in (5, 6, 7):
        for other in range(8):
            if other != out:
                assert run([others[other] if i == out else p for i, p in enumerate(others)]) == INVALID
    assert lib.h2x_attention_forward(ctypes.byref(_attention()), others[0], P, others[1], None, None, P, None, None, None) == INVALID
    # keys in parts need a workspace
    long = _attention(queries=1, keys=1 << 17, samples=1)
    for name in ("k", "v"):
        setattr(long, name, capi.TokenStrides(0, 128, 64))
    assert lib.h2x_attention_forward_workspace_bytes(ctypes.byref(long)) > 0
    assert lib.h2x_attention_forward(ctypes.byref(long), P, P, P, None, None, P, P, None, None) == INVALID
    assert lib.h2x_attention_forward_workspace_bytes(ctypes.byref(_attention(dtype=9))) == 0
    assert lib.h2x_attention_backward_workspace_bytes(ctypes.byref(_attention(dtype=9))) == 0
    assert lib.h2x_attention_forward_workspace_bytes(None) == 0


def test_older_entry_points_refuse_the_new_types():
    lib = capi.load()
    for dtype in (capi.BF16, capi.F16):
        assert lib.h2x_bn_channel_sums_and_sqsums(dtype, 2, 4, 8, 8, P, P, P, P, None) == UNSUPPORTED
        assert lib.h2x_softmax_channel_forward(dtype, 2, 4, 8, P, P, None) == UNSUPPORTED
        assert lib.h2x_softmax_instance_max(dtype, 2, 8, P, P, P, None) == UNSUPPORTED
        assert lib.h2x_halo_clear(dtype, P, 4, capi.i64_array((10, 8, 3, 2)), 1, 1, None) == UNSUPPORTED


# ---- the layers' own checks: they come before any launch --------------------------------------------------------

def test_layer_checks():
    from dihydrogen_amd.tokens import Attention, LayerNormalization, RotaryPositions
    empty = lambda *s, dtype=torch.float32: torch.empty(*s, dtype=dtype)
    norm = LayerNormalization(1e-5)
    x, w, rows = empty(4, 8), empty(8), empty(4)
    bad_norm = [dict(x=empty(4, 8, dtype=torch.int32), y=empty(4, 8, dtype=torch.int32)), dict(y=empty(4, 7)), dict(y=empty(4, 8, dtype=torch.float64)),
                dict(w=empty(7)), dict(w=empty(8, dtype=torch.bfloat16)), dict(x=empty(8, 4).t(), y=empty(8, 4).t()),
                dict(mean=empty(4)), dict(mean=empty(5), rstd=empty(5)), dict(mean=empty(4, dtype=torch.float64), rstd=rows)]
    for change in bad_norm:
        a = dict(x=x, y=empty(4, 8), w=w, mean=None, rstd=None)
        a.update(change)
        with pytest.raises(ValueError):
            norm.forward(a["x"], a["w"], empty(8), a["y"], a["mean"], a["rstd"])
    with pytest.raises(ValueError, match="cpu"):  # all is well but for the device
        norm.forward(x, w, empty(8), empty(4, 8))
    with pytest.raises(ValueError):
        LayerNormalization(-1.0)

    for bad in (dict(axis_pairs=[]), dict(axis_pairs=[1] * 5), dict(axis_pairs=[3, 2]), dict(axis_pairs=[0, 0]), dict(axis_pairs=[-1, 3])):
        with pytest.raises(ValueError):
            RotaryPositions(8, **bad)
    turn = RotaryPositions(8, [2, 1])
    x, pos = empty(2, 3, 4, 8), empty(2, 3, dtype=torch.int32)
    for a, p, b in ((x, pos.long(), x), (x, empty(3, 3, dtype=torch.int32), x), (x, pos, empty(2, 3, 4, 7)), (x[0], pos, x[0]),
                    (x, empty(3, 2, dtype=torch.int32).t(), x), (empty(2, 3, 4, 6), pos, empty(2, 3, 4, 6))):
        with pytest.raises(ValueError):
            turn.forward(a, p, b)
    with pytest.raises(ValueError, match="cpu"):
        turn.forward(x, pos, x)

    att = Attention()
    q, k = empty(2, 5, 4, 16), empty(2, 6, 2, 16)
    good = dict(query=q, key=k, value=k, output=q, logsumexp=empty(2, 4, 5), query_lengths=None, key_lengths=None)
    half = lambda t: t.to(torch.float16)
    for change in (dict(query=half(q), key=half(k), value=half(k), output=half(q)), dict(query=q.double()), dict(key=empty(2, 6, 3, 16)),
                   dict(value=empty(2, 7, 2, 16)), dict(output=empty(2, 5, 4, 8)), dict(logsumexp=empty(2, 5, 4)),
                   dict(key_lengths=empty(2)), dict(key_lengths=empty(3, dtype=torch.int32)), dict(query=q.transpose(2, 3)),
                   dict(key=empty(3, 6, 2, 16))):
        with pytest.raises(ValueError):
            att.forward(**{**good, **change})
    with pytest.raises(ValueError, match="cpu"):
        att.forward(**good)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(window=(-1, None)), dict(causal=True, window=(None, 3))):
        with pytest.raises(ValueError):
            Attention(**bad)


def test_positions_of_a_shard():
    from dihydrogen_amd.tensor import Distribution, LocaleVirtual, Tensor
    from dihydrogen_amd.tokens import grid_positions
    t = Tensor([7, 5, 4, 3, 2], LocaleVirtual(3, 4), Distribution([2, 2, 1, 1, 1]), device="cpu")  # W, H, D, C, N
    p = grid_positions(t)
    assert p.shape == (3, 4 * t.local_shape[1] * t.local_shape[0]) and p.dtype == torch.int32
    w, h = t.local_shape[:2]
    at = (2 * h + 1) * w + 2  # plane 2, row 1, column 2 of the shard
    assert p[:, at].tolist() == [2, t.global_index[1] + 1, t.global_index[0] + 2]
    assert grid_positions(t, [0]).tolist() == [list(range(t.global_index[0], 7))]


def test_scales_that_32_bits_do_not_hold():
    from dihydrogen_amd.tokens import Attention
    lib = capi.load()
    for scale, status in ((1e-60, INVALID), (9e-31, INVALID), (1e-30, 0), (1e30, 0), (2e30, INVALID)):
        a = _attention(scale=scale, samples=0)  # (nothing to launch)
        assert lib.h2x_attention_forward(ctypes.byref(a), P, P, P, None, None, ctypes.c_void_p(2 << 20), P, None, None) == status
        if status:
            with pytest.raises(ValueError):
                Attention(scale=scale)
        else:
            Attention(scale=scale)


def test_most_channels():
    """The sums of the weights' gradients take 64 threads a channel, of fewer than 2^32."""
    lib = capi.load()
    most, O = 1 << 25, ctypes.c_void_p(2 << 20)
    fwd = lambda c: lib.h2x_layer_norm_forward(capi.F32, capi.F32, 1, c, None, None, P, P, P, O, P, P, 1e-5, None)
    bwd = lambda c: lib.h2x_layer_norm_backward(capi.F32, capi.F32, 1, c, None, None, None, P, P, P, P, P, O, P, P, P, None)
    for call in (fwd, bwd):
        assert call(most) > 0 and call(most + 1) == TOO_LARGE and call(1 << 26) == TOO_LARGE


def test_more_heads_than_any_grid_has():
    """Products of the sizes that pass 64 bits are refused, not wrapped."""
    lib, most = capi.load(), 2 ** 31 - 1
    for samples, heads, queries in ((1 << 30, 1 << 30, 1 << 4), (most, most, most - 256), (1 << 16, 1 << 16, 1 << 30), (1, most, most - 256)):
        a = _attention(samples=samples, query_heads=heads, key_heads=heads, queries=queries)
        for name in ("q", "k", "v", "o", "d_o", "dq", "dk", "dv"):
            setattr(a, name, capi.TokenStrides(64, 64, 64))
        p = [ctypes.c_void_p((i + 1) << 20) for i in range(9)]
        assert lib.h2x_attention_forward(ctypes.byref(a), *p[:3], None, None, p[3], P, P, None) == TOO_LARGE
        assert lib.h2x_attention_backward(ctypes.byref(a), *p[:5], P, None, None, *p[5:8], P, None) == TOO_LARGE
