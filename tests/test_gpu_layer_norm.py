"""Layer normalisation through the Python layer and the C ABI, against the plain form in 64 bits, with bounds derived in
tests/token_reference.py."""
import math

import pytest
import torch

import token_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.float64, torch.float64), (torch.bfloat16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float16, torch.float16)]
# one element; less than a wave's vectors; around the rows that a wave, 256 and 1024 threads hold; beyond all of them
CHANNELS = [1, 3, 8, 63, 64, 256, 257, 511, 1000, 1024, 2047, 2049, 4099, 8192, 8200, 16385, 20001]


def _inputs(rows, channels, dtype, weights, seed=0, mean=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * rows + channels)
    n = lambda *s: torch.empty(*s, device="cuda").normal_(0, 1, generator=g)
    return ((n(rows, channels) + mean).to(dtype), n(rows, channels).to(dtype), (1 + 0.2 * n(channels)).to(weights),
            (0.1 * n(channels)).to(weights))


def _compare(x, dy, w, b, epsilon, y, mean, rstd, dx, dw, db, what):
    double = x.dtype == torch.float64
    u = 2.0 ** -53 if double else ref.U
    wt = w.dtype if w is not None else x.dtype
    by, bdx, bdw, bdb = ref.norm_bounds(x, dy, w, b, epsilon, u, ref.half_step(x.dtype), ref.half_step(wt))
    want_y, want_mean, want_rstd = ref.norm(x, w, b, epsilon)[:3]
    want_dx, want_dw, want_db = ref.norm_gradients(x, dy, w, epsilon)
    ref.check(y, want_y, by, f"y {what}")
    ref.check(mean, want_mean[:, 0], ref.ADDS * u * (1 / want_rstd + want_mean.abs())[:, 0], f"mean {what}")
    ref.check(rstd, want_rstd[:, 0], ref.ADDS * u * (1 + want_mean.abs() * want_rstd)[:, 0] * want_rstd[:, 0], f"rstd {what}")
    ref.check(dx, want_dx, bdx, f"dx {what}")
    if dw is not None:
        ref.check(dw, want_dw, bdw, f"dscale {what}")
        ref.check(db, want_db, bdb, f"dbias {what}")


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).split(".")[1] for x in t))
@pytest.mark.parametrize("channels", CHANNELS)
def test_against_the_plain_form(types, channels):
    from dihydrogen_amd.tokens import LayerNormalization
    dtype, weights = types
    layer = LayerNormalization(1e-5)
    kept = torch.float64 if dtype == torch.float64 else torch.float32
    for rows in (1, 5, 37) if channels > 2000 else (1, 6, 300):
        x, dy, w, b = _inputs(rows, channels, dtype, weights)
        fill = 7.0
        yb, y = ref.ragged((rows, channels), dtype, fill)
        dxb, dx = ref.ragged((rows, channels), dtype, fill)
        mean, rstd = (torch.full((rows,), math.nan, dtype=kept, device="cuda") for _ in range(2))
        dw, db = (torch.full((channels,), math.nan, dtype=weights, device="cuda") for _ in range(2))
        layer.forward(x, w, b, y, mean, rstd)
        layer.backward(x, dy, mean, rstd, w, dx, dw, db)
        _compare(x, dy, w, b, 1e-5, y, mean, rstd, dx, dw, db, f"{rows} x {channels}")
        assert ref.outside_untouched(yb, y, fill) and ref.outside_untouched(dxb, dx, fill)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(str(x).split(".")[1] for x in t))
@pytest.mark.parametrize("channels", [16, 17, 33, 100, 128, 130, 300, 700, 1500, 6145, 12000, 12289])
def test_rows_of_every_share(types, channels):
    """Rows that 8, 16 and 32 lanes hold, several to a wave, and those around the other shares' ends."""
    test_against_the_plain_form(types, channels)


@pytest.mark.parametrize("channels", [24, 40, 1155, 9001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_rows_apart(dtype, channels):
    """Rows with gaps, off alignment, in another order of dimensions; between them lies what may not be read."""
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization(1e-3)
    kept = torch.float64 if dtype == torch.float64 else torch.float32
    shape = (2, 3, 4, channels)
    flat = lambda t: t.reshape(-1, channels)
    x, dy, w, b = _inputs(24, channels, dtype, dtype)
    for order, gap, offset in (((0, 1, 2, 3), 3, 1), ((1, 0, 2, 3), 0, 0), ((2, 1, 0, 3), 5, 3)):
        views = [ref.ragged(shape, dtype, math.nan, gap=gap, offset=offset, order=order)[1] for _ in range(2)]
        views[0].copy_(x.view(shape)), views[1].copy_(dy.view(shape))
        yb, y = ref.ragged(shape, dtype, 7.0, gap=2, offset=1, order=order)
        dxb, dx = ref.ragged(shape, dtype, 7.0, gap=1, offset=5)
        mean, rstd = (torch.empty(2, 3, 4, dtype=kept, device="cuda") for _ in range(2))
        dw, db = torch.empty_like(w), torch.empty_like(b)
        layer.forward(views[0], w, b, y, mean, rstd)
        layer.backward(views[0], views[1], mean, rstd, w, dx, dw, db)
        _compare(x, dy, w, b, 1e-3, flat(y), mean.view(-1), rstd.view(-1), flat(dx), dw, db, f"{order}")
        assert ref.outside_untouched(yb, y, 7.0) and ref.outside_untouched(dxb, dx, 7.0)


def test_interior_of_a_haloed_tensor():
    from dihydrogen_amd.tensor import Distribution, LocaleVirtual, Tensor
    from dihydrogen_amd.tokens import LayerNormalization
    dist = Distribution.make_overlapped_distribution([1, 2, 2, 1], [0, 1, 1, 0])
    make = lambda: Tensor([20, 12, 10, 3], LocaleVirtual(1, 4), dist).allocate()  # channel, W, H, sample
    x, y, dx = make(), make(), make()
    x.data.fill_(math.nan), y.data.fill_(7.0), dx.data.fill_(7.0)
    inner = x.interior_view()
    rows = inner.numel() // 20
    a, dy, w, b = _inputs(rows, 20, torch.float32, torch.float32)
    inner.copy_(a.view(inner.shape))
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    dw, db = torch.empty_like(w), torch.empty_like(b)
    layer = LayerNormalization()
    layer.forward(x, w, b, y, mean, rstd)
    layer.backward(x, dy.view(inner.shape), mean, rstd, w, dx, dw, db)
    _compare(a, dy, w, b, 1e-5, y.interior_view().reshape(rows, 20), mean, rstd, dx.interior_view().reshape(rows, 20), dw, db, "halo")
    for t in (y, dx):
        assert int((t.real_view() == 7.0).sum()) >= t.get_local_real_size() - t.get_local_size()
        t.interior_view().fill_(7.0)
        assert bool((t.data == 7.0).all())  # nothing but the interior was written


@pytest.mark.parametrize("channels", [100, 5000, 40000])
def test_without_weights_in_place_and_alone(channels):
    """No scale or bias; outputs on inputs; one gradient alone; without what the backward pass keeps."""
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization(1e-5)
    x, dy, w, b = _inputs(19, channels, torch.bfloat16, torch.float32)
    y, plain = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(19, device="cuda"), torch.empty(19, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    layer.forward(x, w, b, y, mean, rstd)
    layer.forward(x, w, b, plain)
    assert torch.equal(y, plain)
    layer.forward(x, None, None, plain, mean, rstd)
    layer.backward(x, dy, mean, rstd, None, dx, dw, db)
    _compare(x, dy, None, None, 1e-5, plain, mean, rstd, dx, None, None, "no weights")
    layer.backward(x, dy, mean, rstd, w, dx, dw, db)
    for given in ((dw, None), (None, db), (None, None)):
        got = [None if g is None else torch.full_like(g, math.nan) for g in given]
        dx2 = torch.full_like(dx, math.nan)
        layer.backward(x, dy, mean, rstd, w, dx2, *got)
        assert torch.equal(dx2, dx)
        assert all(g is None or torch.equal(g, want) for g, want in zip(got, (dw, db)))
    for target in ("x", "dy"):
        x2, dy2 = x.clone(), dy.clone()
        dw2, db2 = torch.empty_like(w), torch.empty_like(b)
        layer.backward(x2, dy2, mean, rstd, w, x2 if target == "x" else dy2, dw2, db2)
        assert torch.equal(x2 if target == "x" else dy2, dx) and torch.equal(dw2, dw) and torch.equal(db2, db)
    x2 = x.clone()
    layer.forward(x2, w, b, x2)
    assert torch.equal(x2, y)


@pytest.mark.parametrize("channels", [96, 3000, 30000])
def test_far_from_zero_and_constant_rows(channels):
    """A mean a thousand times the deviation; rows without deviation; and a row of infinities or NaN that spoils only itself."""
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization(1e-5)
    x, dy, w, b = _inputs(6, channels, torch.float32, torch.float32, mean=1000.0)
    x[1] = 3.25
    x[2, channels // 2] = math.inf
    x[3, 0] = math.nan
    y = torch.empty_like(x)
    mean, rstd = torch.empty(6, device="cuda"), torch.empty(6, device="cuda")
    layer.forward(x, w, b, y, mean, rstd)
    fine = torch.tensor([0, 1, 4, 5], device="cuda")
    bound = ref.norm_bounds(x[fine], None, w, b, 1e-5, ref.U, ref.half_step(torch.float32), 0)
    ref.check(y[fine], ref.norm(x[fine], w, b, 1e-5)[0], bound, "fine rows")
    assert torch.isnan(y[3]).all() and torch.isnan(y[2]).any()


def test_no_rows():
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization()
    x, w = torch.empty(0, 40, device="cuda"), torch.ones(40, device="cuda")
    none = torch.empty(0, device="cuda")
    dw, db = torch.full_like(w, math.nan), torch.full_like(w, math.nan)
    layer.forward(x, w, w, x, none, none)
    layer.backward(x, x, none, none, w, x, dw, db)
    assert bool((dw == 0).all()) and bool((db == 0).all())


def test_many_rows_of_few_channels():
    """More rows than one grid of workgroups takes at four rows each."""
    from dihydrogen_amd.tokens import LayerNormalization
    rows = (1 << 25) + 3
    x = torch.empty(rows, 4, dtype=torch.bfloat16, device="cuda").normal_()
    y = torch.full_like(x, math.nan)
    layer = LayerNormalization()
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    layer.forward(x, None, None, y, mean, rstd)
    dx = torch.full_like(x, math.nan)
    layer.backward(x, x, mean, rstd, None, dx)
    for part in (slice(0, 1000), slice(rows // 2, rows // 2 + 1000), slice(rows - 1000, rows)):
        a = x[part]
        by, bdx, _, _ = ref.norm_bounds(a, a, None, None, 1e-5, ref.U, ref.half_step(torch.bfloat16), 0)
        ref.check(y[part], ref.norm(a, None, None, 1e-5)[0], by, "y")
        ref.check(dx[part], ref.norm_gradients(a, a, None, 1e-5)[0], bdx, "dx")
    assert not torch.isnan(y).any() and not torch.isnan(dx).any()


def test_gradients_against_differences():
    """The kernels' own forward pass, in 64 bits, along random directions."""
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization(1e-3)
    x, dy, w, b = _inputs(7, 33, torch.float64, torch.float64)
    mean, rstd = (torch.empty(7, dtype=torch.float64, device="cuda") for _ in range(2))
    y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)

    def loss(x, w, b):
        layer.forward(x, w, b, y, mean, rstd)
        return float((y * dy).sum())

    loss(x, w, b)
    layer.backward(x, dy, mean.clone(), rstd.clone(), w, dx, dw, db)
    e = 1e-5
    for _ in range(3):
        d, dv = torch.randn_like(x), torch.randn_like(w)
        # differences of 64-bit values of magnitude 100: 1e-14 * 100 / 1e-5, and e^2 times a third derivative of magnitude 100
        assert math.isclose((loss(x + e * d, w, b) - loss(x - e * d, w, b)) / (2 * e), float((dx * d).sum()), rel_tol=1e-6, abs_tol=1e-6)
        assert math.isclose((loss(x, w + e * dv, b) - loss(x, w - e * dv, b)) / (2 * e), float((dw * dv).sum()), rel_tol=1e-6, abs_tol=1e-6)
        assert math.isclose((loss(x, w, b + e * dv) - loss(x, w, b - e * dv)) / (2 * e), float((db * dv).sum()), rel_tol=1e-6, abs_tol=1e-6)


def test_same_bits_every_time():
    from dihydrogen_amd.tokens import LayerNormalization
    layer = LayerNormalization()
    x, dy, w, _ = _inputs(3001, 770, torch.bfloat16, torch.float32)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = torch.empty(3001, device="cuda"), torch.empty(3001, device="cuda")
    layer.forward(x, w, None, y, mean, rstd)
    runs = []
    for _ in range(3):
        dw, db = torch.empty_like(w), torch.empty_like(w)
        layer.backward(x, dy, mean, rstd, w, dx, dw, db)
        runs.append((dx.clone(), dw, db))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))
