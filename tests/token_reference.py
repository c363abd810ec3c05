"""The token operators in 64 bits, plainly (not collected by pytest), and bounds of their errors.

u is half a step of float32, h half a step of the elements' type; both relative to the value."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def ragged(shape, dtype, fill, device="cuda", gap=0, offset=0, order=None):
    """A tensor of `shape` in a buffer full of `fill`: `gap` elements behind each last dimension, `offset` before it all,
    dimensions in memory in `order` (None: as they are).  Returns (the buffer, the view)."""
    order = list(range(len(shape))) if order is None else list(order)
    assert order[-1] == len(shape) - 1
    in_memory = [shape[d] for d in order]
    padded = in_memory[:-1] + [in_memory[-1] + gap]
    buffer = torch.full((offset + math.prod(padded) + 64,), fill, dtype=dtype, device=device)
    view = buffer[offset:offset + math.prod(padded)].view(padded).narrow(-1, 0, in_memory[-1])
    return buffer, view.permute([order.index(d) for d in range(len(shape))])


def outside_untouched(buffer, view, fill):
    """Whether all of the buffer that is not in the view still holds `fill`."""
    saved = view.clone()
    view.fill_(fill)
    same = bool((buffer == fill).all())
    view.copy_(saved)
    return same


# ---- layer normalisation -----------------------------------------------------------------------------------

def norm(x, scale, bias, epsilon):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean) ** 2).mean(-1, keepdim=True).add(epsilon).rsqrt()
    h = (x - mean) * rstd
    w = torch.ones_like(x[0]) if scale is None else scale.double()
    b = torch.zeros_like(x[0]) if bias is None else bias.double()
    return h * w + b, mean, rstd, h, w, b


def norm_gradients(x, dy, scale, epsilon):
    _, _, rstd, h, w, _ = norm(x, scale, None, epsilon)
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx, (dy * h).sum(0), dy.sum(0)


# A row's sum is made of at most 64 numbers a thread (32 in registers, as many partial ones), 6 steps of a wave and 16 waves: 86 roundings.
ADDS = 96


def norm_bounds(x, dy, scale, bias, epsilon, u, h_elements, h_weights):
    """Bounds of y, dx, dscale, dbias.  The mean is off by ADDS u times the mean magnitude (at most 1 / rstd + |mean|), so h by ADDS u (1 +
    |mean| rstd) and by its share of rstd's error, of which half a sum's error and the square root's."""
    y, mean, rstd, h, w, b = norm(x, scale, bias, epsilon)
    dh = ADDS * u * (1 + mean.abs() * rstd + h.abs())
    by = dh * w.abs() + 4 * u * (y.abs() + b.abs()) + h_elements * y.abs()
    if dy is None:
        return by
    dx, dscale, dbias = norm_gradients(x, dy, scale, epsilon)
    dy = dy.double()
    g = (dy * w).abs()
    size = (g ** 2).mean(-1, keepdim=True).sqrt()  # at least the mean of |g|, and of |g h|, as h has mean square 1
    d = dh.amax(-1, keepdim=True)
    bdx = rstd * (4 * u * g + ADDS * u * size * (1 + h.abs()) + 2 * d * size * (1 + h.abs()) + dh * size) + 8 * u * dx.abs() \
        + h_elements * dx.abs()
    rows = x.shape[0]
    bds = (dy.abs() * (dh + (rows + 8) * u * h.abs())).sum(0) + h_weights * dscale.abs()
    bdb = (rows + 8) * u * dy.abs().sum(0) + h_weights * dbias.abs()
    return by, bdx, bds, bdb


# ---- rotary positions -------------------------------------------------------------------------------------------

def rotary(x, positions, frequencies, axis_pairs, neighbours, inverse=False):
    """positions: (samples, axes, tokens)."""
    x = x.double()
    axis = [a for a, m in enumerate(axis_pairs) for _ in range(m)]
    angle = positions.double()[:, axis].transpose(1, 2) * frequencies  # samples, tokens, pairs
    angle = (-angle if inverse else angle)[:, :, None]
    m, y = len(axis), x.clone()
    first = slice(0, 2 * m, 2) if neighbours else slice(0, m)
    second = slice(1, 2 * m, 2) if neighbours else slice(m, 2 * m)
    u, v = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
    return y


def rotary_bound(x, y, axis_pairs, neighbours, u, h):
    """An angle of 64 bits is off by its rounding and that of its reduction (2 ** -50 of up to 2 ** 31 turns: below u), what is left of it is
    rounded to u of half a turn (3 u), sine and cosine to two steps of theirs: 8 u in all, and two operations."""
    m = sum(axis_pairs)
    size = torch.zeros_like(y)
    first = slice(0, 2 * m, 2) if neighbours else slice(0, m)
    second = slice(1, 2 * m, 2) if neighbours else slice(m, 2 * m)
    size[..., first] = size[..., second] = x.double()[..., first].abs() + x.double()[..., second].abs()
    return 10 * u * size + h * y.abs()


# ---- attention --------------------------------------------------------------------------------------------------

def visible(n, queries, keys, left, right, query_lengths, key_lengths):
    """Which keys each query sees: (samples, queries, keys), on the CPU."""
    seen = torch.zeros(n, queries, keys, dtype=torch.bool)
    for b in range(n):
        nq = queries if query_lengths is None else min(max(int(query_lengths[b]), 0), queries)
        nk = keys if key_lengths is None else min(max(int(key_lengths[b]), 0), keys)
        for i in range(nq):
            place = i + nk - nq
            lo = 0 if left is None else max(0, place - left)
            hi = nk if right is None else min(nk, place + right + 1)
            if lo < hi:
                seen[b, i, lo:hi] = True
    return seen


def _heads(t, heads):
    """samples, tokens, heads, elements -> samples, heads, tokens, elements, shared heads repeated."""
    t = t.double().transpose(1, 2)
    return t.repeat_interleave(heads // t.shape[1], 1)


def _clean(t, seen_rows):
    """Rows that nobody sees may hold anything."""
    return torch.where(seen_rows[:, None, :, None], t, torch.zeros((), dtype=t.dtype, device=t.device))


class AttentionReference:
    """Everything (samples, heads, queries, ...) in 64 bits."""

    def __init__(self, q, k, v, scale, seen):
        self.heads, self.key_heads, self.dim = q.shape[2], k.shape[2], q.shape[3]
        self.scale, self.seen = scale, seen.to(q.device)
        used_q, used_k = self.seen.any(2), self.seen.any(1)
        self.q, self.k, self.v = (_clean(_heads(t, self.heads), used) for t, used in ((q, used_q), (k, used_k), (v, used_k)))
        hidden = ~self.seen[:, None]
        self.s = (self.q @ self.k.transpose(2, 3) * scale).masked_fill(hidden, -math.inf)
        self.lse = torch.logsumexp(self.s, 3) if k.shape[1] else torch.full(self.s.shape[:3], -math.inf, device=q.device).double()
        self.p = torch.exp(self.s - self.lse.masked_fill(self.lse == -math.inf, 0)[..., None])
        self.o = self.p @ self.v
        # a score: rounding of its products' sum, of its scaling, and of what is taken from it; the exponential two steps
        size = self.q.abs() @ self.k.abs().transpose(2, 3) * scale
        top = lambda t: t.amax(3, keepdim=True) if t.shape[3] else torch.zeros_like(t[..., :1].sum(3, keepdim=True))
        self.e_score = (self.dim + 8) * U * top(size) + 8 * U * (1 + self.lse.masked_fill(self.lse == -math.inf, 0).abs()[..., None])

    def forward_bounds(self, dtype):
        """Of o and lse.  Probabilities of 16 bits are off by half a step each for the product with v; their sum is made of the unrounded
        ones; sums go over all keys."""
        half = half_step(dtype) if dtype == torch.bfloat16 else 0.0
        keys = self.k.shape[2]
        size = self.p @ self.v.abs()
        bo = size * (half + 2 * self.e_score + (2 * keys + 64) * U) + half_step(dtype) * self.o.abs()
        bl = self.e_score[..., 0] + (keys + 64) * U + 4 * U * self.lse.masked_fill(self.lse == -math.inf, 0).abs()
        return bo, bl

    def gradients(self, d_o, o, lse, dtype):
        """From what the backward pass is given: (value, bound) of dq, dk, dv, laid out as the inputs."""
        half = half_step(dtype) if dtype == torch.bfloat16 else 0.0
        used_q = self.seen.any(2)
        d_o, o = _clean(_heads(d_o, self.heads), used_q), _clean(_heads(o, self.heads), used_q)
        lse = lse.double()
        p = torch.where(self.seen[:, None], torch.exp(self.s - lse.masked_fill(lse == -math.inf, 0)[..., None]), torch.zeros_like(self.s))
        dp, delta = d_o @ self.v.transpose(2, 3), (d_o * o).sum(3, keepdim=True)
        ds = p * (dp - delta)
        e_dp = (self.dim + 8) * U * (d_o.abs() @ self.v.abs().transpose(2, 3) + (d_o * o).abs().sum(3, keepdim=True))
        e_ds = ds.abs() * (half + 2 * self.e_score) + p * e_dp * (1 + half)
        n, queries = self.q.shape[0], self.q.shape[2]
        keys, group = self.k.shape[2], self.heads // max(self.key_heads, 1)

        def shared(t):  # sums over the heads of a group
            return t.view(n, self.key_heads, group, keys, self.dim).sum(2)

        tr = lambda t: t.transpose(2, 3)
        # (a bf16 zero or the smallest numbers: an absolute error of the smallest normal number does no harm)
        tiny = 1e-37
        adds_q, adds_k = (keys + 64) * U, (queries * group + 64) * U
        dq, bq = ds @ self.k * self.scale, (e_ds + adds_q * ds.abs()) @ self.k.abs() * self.scale
        dk = shared(tr(ds) @ self.q) * self.scale
        bk = shared(tr(e_ds + adds_k * ds.abs()) @ self.q.abs()) * self.scale
        dv = shared(tr(p) @ d_o)
        bv = shared(tr(p * (half + 2 * self.e_score + adds_k)) @ d_o.abs())
        return [(t.transpose(1, 2), (b + half_step(dtype) * t.abs() + 4 * U * t.abs() + tiny).transpose(1, 2))
                for t, b in ((dq, bq), (dk, bk), (dv, bv))]


def check(got, want, bound, what=""):
    """got within bound of want, elementwise; nothing is NaN."""
    # Below the smallest normal number 2^m a type's numbers lie 2^m eps apart, however small: rounding is off by up to 2^m eps / 2 there,
    # which is more than half a step relative to the value (float16: 2.9e-5 lies between multiples of 2^-24, and may be off by 2^-25 = 3e-8,
    # where eps / 2 of it is 1.4e-8).
    bound = bound + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert not torch.isnan(got).any(), f"{what}: NaN"
    error = (got - want).abs()
    worst = (error - bound)
    if worst.numel() and bool((worst > 0).any()):
        at = int(worst.argmax())
        raise AssertionError(f"{what}: {got.flatten()[at]} against {want.flatten()[at]}, bound {bound.flatten()[at]}, "
                             f"{int((worst > 0).sum())} of {worst.numel()} beyond theirs")
