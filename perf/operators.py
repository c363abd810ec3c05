"""Performance cases of the token operators: layer normalisation, rotary positions over a grid, and
attention, forward and backward.  A network over images or volumes uses them once it treats the cells
of its grid as tokens.

Shapes are written outermost first: samples, tokens, heads, elements of a head.
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16, "float16": torch.float16}
_EPSILON = 1e-5


def _norm(name, rows, cols, dtype="bfloat16", weights="float32", step="train"):
    return {"name": name, "kind": "norm", "rows": rows, "cols": cols, "dtype": dtype, "weights": weights, "step": step}


def _rotary(name, n, grid, heads, dim, pairs, dtype="bfloat16", pairing="halves", step="forward"):
    """grid: cells along depth, height and width; pairs: rotated pairs that belong to each of these axes."""
    return {"name": name, "kind": "rotary", "n": n, "gd": grid[0], "gh": grid[1], "gw": grid[2], "heads": heads, "dim": dim,
            "pd": pairs[0], "ph": pairs[1], "pw": pairs[2], "dtype": dtype, "pairing": pairing, "step": step}


def _attention(name, n, queries, keys, heads, key_heads, dim, dtype="bfloat16", step="forward", left=-1, right=-1,
               ragged=False):
    """left, right: how many keys before and behind its own position a query sees (-1: all).  ragged: samples of
    unlike lengths in a padded batch."""
    return {"name": name, "kind": "attention", "n": n, "queries": queries, "keys": keys, "heads": heads,
            "key_heads": key_heads, "dim": dim, "dtype": dtype, "step": step, "left": left, "right": right, "ragged": ragged}


def listed():
    return [
        # Serving one image of 14 x 14 patches: the smallest calls, bound by latency.
        _norm("norm_infer_one_image", 196, 768, step="forward"),
        # A training step's normalisation of a batch of 64 x 64 grids, weights kept in 32 bits.
        _norm("norm_train_tokens", 8 * 4096, 1024),
        # Single precision, an odd number of channels: no row but every fourth starts on a vector.
        _norm("norm_train_odd_f32", 3 * 1369, 1155, dtype="float32"),
        # Gradient of the queries and keys of an image in single precision, neighbours paired.
        _rotary("rotary_image_f32", 1, (1, 24, 24), 24, 64, (0, 16, 16), dtype="float32", pairing="neighbours", step="backward"),
        # Queries and keys of a video or a volume, three axes.
        _rotary("rotary_video", 2, (16, 32, 32), 32, 128, (16, 24, 24)),
        # Serving one image.
        _attention("attention_one_image", 1, 196, 196, 12, 12, 64),
        # Serving single tokens: one query a sample against caches of unlike lengths, key heads shared by four.
        _attention("attention_single_queries", 16, 1, 16384, 32, 8, 128, ragged=True),
        # A video's or a volume's tokens, all against all: the largest forward pass.
        _attention("attention_volume", 1, 16384, 16384, 16, 16, 128),
        # Single precision, an ordered sequence of odd length, heads of 80.
        _attention("attention_ordered_f32", 2, 1001, 1001, 8, 8, 80, dtype="float32", right=0),
        # A training step's gradients, ordered tokens, key heads shared by four.
        _attention("attention_train_ordered", 4, 4096, 4096, 16, 4, 128, step="backward", right=0),
        # Gradients of local attention over a long sequence.
        _attention("attention_train_window", 1, 16384, 16384, 12, 12, 64, step="backward", left=512, right=512),
        # Gradients in single precision of a padded batch of unlike samples.
        _attention("attention_train_ragged_f32", 3, 577, 577, 12, 12, 72, dtype="float32", step="backward", ragged=True),
    ]


# ---- drawn cases ---------------------------------------------------------------------------------------

_MOST_NORM = 8 * 4096 * 1024
_MOST_ROTARY = 2 * 16384 * 32 * 128
_MOST_PAIRS = 16384 * 16384 * 16 * 128  # (visible pairs of a query and a key) x elements of a head


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_norm(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float32", "float16", "float64"])
    weights = dtype if dtype == "float64" or rng.random() < 0.4 else "float32"
    while True:
        rows, cols = _log(rng, 16, 200_000), _log(rng, 32, 16384)
        if rng.random() < 0.6:
            cols = max(8, cols // 8 * 8)
        if 20_000 <= rows * cols <= _MOST_NORM // (2 if dtype == "float64" else 1):
            return _norm("", rows, cols, dtype, weights, "forward" if rng.random() < 0.3 else "train")


def _draw_rotary(rng):
    dtype = rng.choice(["bfloat16", "bfloat16", "float32", "float16"])
    while True:
        three_d = rng.random() < 0.6
        grid = [_log(rng, 2, 48) if three_d else 1, _log(rng, 4, 80), _log(rng, 4, 80)]
        dim, heads, n = rng.choice([32, 64, 72, 80, 96, 128]), _log(rng, 2, 64), _log(rng, 1, 8)
        if 50_000 <= n * math.prod(grid) * heads * dim <= _MOST_ROTARY // (2 if dtype == "float32" else 1):
            break
    half = dim // 2
    first = half // 4 if three_d else 0
    h = (half - first) // 2
    w = half - first - h - (4 if rng.random() < 0.2 else 0)  # now and then the last elements are not rotated
    return _rotary("", n, grid, heads, dim, (first, h, w), dtype, rng.choice(["halves", "neighbours"]),
                   "backward" if rng.random() < 0.4 else "forward")


def _draw_attention(rng):
    serving = rng.random() < 0.3
    dtype = "float32" if not serving and rng.random() < 0.25 else "bfloat16"
    while True:
        key_heads = _log(rng, 1, 16)
        heads = key_heads * rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
        n = _log(rng, 1, 32)
        left = right = -1
        step, ragged = "forward", rng.random() < 0.35
        if serving:
            keys, queries = _log(rng, 64, 32768), rng.choice([1, 1, 1, 2, 5])
            right = 0
        else:
            keys = _log(rng, 32, 16384)
            queries = keys if rng.random() < 0.7 else max(1, round(keys * rng.uniform(0.1, 1.5)))
            step = "backward" if rng.random() < 0.6 else "forward"
            form = rng.random()
            if form < 0.4:
                right = 0
            elif form < 0.55:
                left, right = _log(rng, 16, 1024), rng.choice([0, 64, 512])
        case = _attention("", n, queries, keys, heads, key_heads, dim, dtype, step, left, right, ragged)
        cost = _pairs(case) * dim * (10 if dtype == "float32" else 1) * (2.5 if step == "backward" else 1)
        buffers = n * (queries * heads + keys * key_heads) * dim
        # (and no more pairs than a plain pass can go through in a second)
        if 1_000_000 <= cost <= _MOST_PAIRS and buffers <= 150_000_000 and n * heads * queries * keys <= 16 * 16384 ** 2:
            return case


def draw(rng):
    kind = rng.choice(["norm", "rotary", "attention", "attention", "attention"])
    case = {"norm": _draw_norm, "rotary": _draw_rotary, "attention": _draw_attention}[kind](rng)
    del case["name"]
    return case


# ---- what the operators are given ------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, dtype, generator, std=1.0, mean=0.0):
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=generator).to(dtype)


def _prepare_norm(case, seed):
    g, dtype, weights = _generator(seed), _DTYPES[case["dtype"]], _DTYPES[case["weights"]]
    rows, cols, train = case["rows"], case["cols"], case["step"] == "train"
    kept = torch.float64 if dtype == torch.float64 else torch.float32
    s = {"x": _normal((rows, cols), dtype, g, mean=0.2), "scale": _normal((cols,), weights, g, 0.2, 1.0),
         "bias": _normal((cols,), weights, g, 0.1), "train": train, "y": torch.empty((rows, cols), dtype=dtype, device="cuda"),
         "mean": None, "rstd": None}
    if train:
        s.update(dy=_normal((rows, cols), dtype, g), dx=torch.empty_like(s["x"]),
                 mean=torch.empty(rows, dtype=kept, device="cuda"), rstd=torch.empty(rows, dtype=kept, device="cuda"),
                 dscale=torch.empty_like(s["scale"]), dbias=torch.empty_like(s["bias"]))
    if own:
        from dihydrogen_amd.tokens import LayerNormalization
        s["layer"] = LayerNormalization(_EPSILON)
    return s


def _grid(case):
    return [case["gd"], case["gh"], case["gw"]]


def _rotary_parts(case):
    """The axes that have pairs, and how many each."""
    pairs = [case["pd"], case["ph"], case["pw"]]
    axes = [a for a in range(3) if pairs[a]]
    return axes, [pairs[a] for a in axes]


def _prepare_rotary(case, seed):
    g, dtype = _generator(seed), _DTYPES[case["dtype"]]
    grid, (axes, pairs) = _grid(case), _rotary_parts(case)
    tokens = math.prod(grid)
    # the block that this rank holds lies somewhere in a larger grid
    origin = [int(v) for v in torch.randint(0, 4096, (3,), device="cuda", generator=g).tolist()]
    cells = torch.meshgrid(*[torch.arange(e, dtype=torch.int32, device="cuda") + o for e, o in zip(grid, origin)], indexing="ij")
    positions = torch.stack([cells[a].reshape(-1) for a in axes]).contiguous()
    x = _normal((case["n"], tokens, case["heads"], case["dim"]), dtype, g)
    s = {"x": x, "y": torch.empty_like(x), "positions": positions, "pairs": pairs, "pairing": case["pairing"],
         "inverse": case["step"] == "backward"}
    if own:
        from dihydrogen_amd.tokens import RotaryPairing, RotaryPositions
        s["layer"] = RotaryPositions(case["dim"], pairs, base=10000.0, pairing=RotaryPairing[case["pairing"].upper()])
    return s


def _lengths(case):
    """Queries and keys of each sample of a padded batch; the first sample has them all."""
    n, queries, keys = case["n"], case["queries"], case["keys"]
    if not case["ragged"]:
        return [queries] * n, [keys] * n
    key_lengths = [max(1, keys - keys * 3 * i // (4 * n)) for i in range(n)]
    # serving: every sample has its queries; else the samples' queries get fewer as their keys do
    return [min(queries, max(1, queries * k // keys)) if queries > 8 else queries for k in key_lengths], key_lengths


def _prepare_attention(case, seed):
    g, dtype, dim = _generator(seed), _DTYPES[case["dtype"]], case["dim"]
    n, queries, keys, heads, key_heads = (case[k] for k in ("n", "queries", "keys", "heads", "key_heads"))
    if queries == keys:
        # parts of what one projection has written
        fused = _normal((n, queries, heads + 2 * key_heads, dim), dtype, g)
        q, k, v = fused.split([heads, key_heads, key_heads], dim=2)
    elif case["queries"] <= 8:
        # a cache, head by head
        q = _normal((n, queries, heads, dim), dtype, g)
        k, v = (_normal((n, key_heads, keys, dim), dtype, g).transpose(1, 2) for _ in range(2))
    else:
        q = _normal((n, queries, heads, dim), dtype, g)
        k, v = (_normal((n, keys, key_heads, dim), dtype, g) for _ in range(2))
    s = {"q": q, "k": k, "v": v, "o": torch.empty((n, queries, heads, dim), dtype=dtype, device="cuda"),
         "lse": torch.empty((n, heads, queries), device="cuda"), "left": case["left"], "right": case["right"],
         "query_lengths": None, "key_lengths": None, "step": case["step"]}
    if case["ragged"]:
        order = torch.randperm(n, device="cuda", generator=g)
        s["query_lengths"], s["key_lengths"] = (torch.tensor(l, dtype=torch.int32, device="cuda")[order] for l in _lengths(case))
    if case["step"] == "backward":
        o, lse = _plain_attention(s)
        s["o"].copy_(o)
        s["lse"].copy_(lse)
        s["do"] = _normal((n, queries, heads, dim), dtype, g)
        s.update(dq=torch.empty((n, queries, heads, dim), dtype=dtype, device="cuda"),
                 dk=torch.empty((n, keys, key_heads, dim), dtype=dtype, device="cuda"),
                 dv=torch.empty((n, keys, key_heads, dim), dtype=dtype, device="cuda"))
    if own:
        from dihydrogen_amd.tokens import Attention
        s["layer"] = Attention(window=tuple(None if w < 0 else w for w in (case["left"], case["right"])))
    return s


def prepare(case, seed):
    s = {"norm": _prepare_norm, "rotary": _prepare_rotary, "attention": _prepare_attention}[case["kind"]](case, seed)
    s["kind"] = case["kind"]
    return s


# ---- the framework's calls -----------------------------------------------------------------------------------

def _own_norm(s):
    s["layer"].forward(s["x"], s["scale"], s["bias"], s["y"], s["mean"], s["rstd"])
    if not s["train"]:
        return s["y"]
    s["layer"].backward(s["x"], s["dy"], s["mean"], s["rstd"], s["scale"], s["dx"], s["dscale"], s["dbias"])
    return s["y"], s["dx"], s["dscale"], s["dbias"]


def _own_rotary(s):
    if s["inverse"]:
        s["layer"].backward(s["x"], s["positions"], s["y"])
    else:
        s["layer"].forward(s["x"], s["positions"], s["y"])
    return s["y"]


def _own_attention(s):
    lengths = {"query_lengths": s["query_lengths"], "key_lengths": s["key_lengths"]}
    if s["step"] == "backward":
        s["layer"].backward(s["q"], s["k"], s["v"], s["o"], s["do"], s["lse"], s["dq"], s["dk"], s["dv"], **lengths)
        return s["dq"], s["dk"], s["dv"]
    s["layer"].forward(s["q"], s["k"], s["v"], s["o"], s["lse"], **lengths)
    return s["o"], s["lse"]


# ---- the plain forms -------------------------------------------------------------------------------------------

def _plain_norm(s):
    wide = torch.float64 if s["x"].dtype == torch.float64 else torch.float32
    x, w, b = s["x"].to(wide), s["scale"].to(wide), s["bias"].to(wide)
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + _EPSILON)
    hat = centred * rstd
    y = (hat * w + b).to(s["x"].dtype)
    if not s["train"]:
        return y
    dy = s["dy"].to(wide)
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * hat).sum(0).to(s["scale"].dtype), dy.sum(0).to(s["bias"].dtype)


def _frequencies(pairs):
    """One for each pair, axis after axis: an axis' frequencies run from 1 down to nearly 1 / 10000."""
    return torch.cat([10000.0 ** (-torch.arange(m, dtype=torch.float64, device="cuda") / m) for m in pairs])


def _plain_rotary(s):
    x, pairs = s["x"], s["pairs"]
    axis = torch.tensor([a for a, m in enumerate(pairs) for _ in range(m)], device="cuda")
    angle = s["positions"].double()[axis].T * _frequencies(pairs)  # tokens, pairs; far positions need 64 bits
    if s["inverse"]:
        angle = -angle
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    cos, sin = angle.cos().to(wide)[:, None, :], angle.sin().to(wide)[:, None, :]
    m, y = sum(pairs), x.to(wide)
    if s["pairing"] == "halves":
        u, v = y[..., :m], y[..., m:2 * m]
        rotated = torch.cat([u * cos - v * sin, u * sin + v * cos, y[..., 2 * m:]], -1)
    else:
        u, v = y[..., 0:2 * m:2], y[..., 1:2 * m:2]
        rotated = torch.cat([torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2), y[..., 2 * m:]], -1)
    return rotated.to(x.dtype)


def _hidden(s, first, last, heads_per):
    """Which keys the queries do not see, for rows first to last of the (sample, key head) pairs; None: they see all."""
    q, k = s["q"], s["k"]
    if s["key_lengths"] is None and s["left"] < 0 and s["right"] < 0:
        return None
    queries, keys, key_heads = q.shape[1], k.shape[1], k.shape[2]
    sample = torch.arange(first, last, device="cuda") // key_heads
    i, j = torch.arange(queries, device="cuda")[None, :, None], torch.arange(keys, device="cuda")[None, None, :]
    if s["key_lengths"] is None:
        nq, nk = queries, keys
        hidden = torch.zeros((1, queries, keys), dtype=torch.bool, device="cuda")
    else:
        nq, nk = s["query_lengths"][sample][:, None, None], s["key_lengths"][sample][:, None, None]
        hidden = (i >= nq) | (j >= nk)
    place = i + nk - nq  # the last query stands at the last key
    if s["left"] >= 0:
        hidden = hidden | (j < place - s["left"])
    if s["right"] >= 0:
        hidden = hidden | (j > place + s["right"])
    return hidden[:, None].expand(-1, heads_per, -1, -1).reshape(hidden.shape[0], heads_per * queries, keys)


def _by_key_head(t, key_heads):
    """samples, tokens, heads, dim -> (sample, key head), (head of the group, token), dim, in 32 bits."""
    n, tokens, heads, dim = t.shape
    return t.float().reshape(n, tokens, key_heads, heads // key_heads, dim).permute(0, 2, 3, 1, 4).reshape(
        n * key_heads, heads // key_heads * tokens, dim)


def _from_key_head(t, n, tokens, heads):
    key_heads, dim = t.shape[0] // n, t.shape[2]
    return t.reshape(n, key_heads, heads // key_heads, tokens, dim).permute(0, 3, 1, 2, 4).reshape(n, tokens, heads, dim)


def _parts(s):
    """Ranges of (sample, key head) pairs whose scores fit 2 GiB."""
    n, queries, heads, _ = s["q"].shape
    keys, key_heads = s["k"].shape[1:3]
    step = max(1, 2 ** 29 // max(1, heads // key_heads * queries * keys))
    return [(a, min(a + step, n * key_heads)) for a in range(0, n * key_heads, step)]


def _plain_attention(s):
    n, queries, heads, dim = s["q"].shape
    key_heads = s["k"].shape[2]
    scale = dim ** -0.5
    q, k, v = (_by_key_head(s[t], key_heads) for t in ("q", "k", "v"))
    o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    for a, b in _parts(s):
        score = torch.bmm(q[a:b] * scale, k[a:b].transpose(1, 2))
        hidden = _hidden(s, a, b, heads // key_heads)
        if hidden is not None:
            score = score.masked_fill(hidden, -math.inf)
        most = score.amax(2, keepdim=True)
        most = most.masked_fill(most == -math.inf, 0.0)  # rows that see nothing
        p = torch.exp(score - most)
        total = p.sum(2, keepdim=True)
        lse[a:b] = (most + torch.log(total))[..., 0]
        o[a:b] = torch.bmm(p, v[a:b]) / total.masked_fill(total == 0, 1.0)
    lse = lse.reshape(n, key_heads, heads // key_heads, queries).reshape(n, heads, queries)
    return _from_key_head(o, n, queries, heads).to(s["q"].dtype), lse


def _plain_attention_backward(s):
    n, queries, heads, dim = s["q"].shape
    keys, key_heads = s["k"].shape[1:3]
    scale = dim ** -0.5
    q, k, v, o, do = (_by_key_head(s[t], key_heads) for t in ("q", "k", "v", "o", "do"))
    lse = s["lse"].reshape(n * key_heads, heads // key_heads * queries, 1)
    lse = lse.masked_fill(lse == -math.inf, 0.0)
    delta = (do * o).sum(2, keepdim=True)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for a, b in _parts(s):
        p = torch.exp(torch.bmm(q[a:b] * scale, k[a:b].transpose(1, 2)) - lse[a:b])
        hidden = _hidden(s, a, b, heads // key_heads)
        if hidden is not None:
            p = p.masked_fill(hidden, 0.0)
        dv[a:b] = torch.bmm(p.transpose(1, 2), do[a:b])
        ds = p * (torch.bmm(do[a:b], v[a:b].transpose(1, 2)) - delta[a:b])
        dq[a:b] = torch.bmm(ds, k[a:b]) * scale
        dk[a:b] = torch.bmm(ds.transpose(1, 2), q[a:b]) * scale
    return (_from_key_head(dq, n, queries, heads).to(s["q"].dtype), _from_key_head(dk, n, keys, key_heads).to(s["q"].dtype),
            _from_key_head(dv, n, keys, key_heads).to(s["q"].dtype))


def run(state):
    kind = state["kind"]
    if own:
        return {"norm": _own_norm, "rotary": _own_rotary, "attention": _own_attention}[kind](state)
    if kind == "norm":
        return _plain_norm(state)
    if kind == "rotary":
        return _plain_rotary(state)
    return _plain_attention_backward(state) if state["step"] == "backward" else _plain_attention(state)


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------

def _exact_norm(case, s):
    x, w, b = s["x"].double(), s["scale"].double(), s["bias"].double()
    c = case["cols"]
    mean = x.sum(1) / c
    rstd = 1.0 / torch.sqrt(((x - mean[:, None]) ** 2).sum(1) / c + _EPSILON)
    y = (x - mean[:, None]) * rstd[:, None]
    if case["step"] != "train":
        return y * w + b
    dy = s["dy"].double()
    along, across = (dy * w).sum(1) / c, (dy * w * y).sum(1) / c
    dx = (dy * w - along[:, None] - y * across[:, None]) * rstd[:, None]
    return y * w + b, dx, torch.einsum("rc,rc->c", dy, y), torch.einsum("rc->c", dy)


def _exact_rotary(case, s):
    axes, pairs = _rotary_parts(case)
    x = s["x"].double()
    out, m, j = x.clone(), sum(pairs), 0
    sign = -1.0 if case["step"] == "backward" else 1.0
    for row, count in enumerate(pairs):
        place = s["positions"][row].double()
        for i in range(count):
            turn = torch.polar(torch.ones_like(place), sign * place * math.pow(10000.0, -i / count))
            first, second = (j, j + m) if case["pairing"] == "halves" else (2 * j, 2 * j + 1)
            z = torch.complex(x[..., first], x[..., second]) * turn[None, :, None]
            out[..., first], out[..., second] = z.real, z.imag
            j += 1
    return out


def _exact_attention(case, s):
    """Sample by sample and head by head, over the sample's own queries and keys, some queries at a time."""
    n, queries, keys, heads, group = (case["n"], case["queries"], case["keys"], case["heads"],
                                      case["heads"] // case["key_heads"])
    backward, scale = case["step"] == "backward", 1.0 / math.sqrt(case["dim"])
    f64 = {"dtype": torch.float64, "device": "cuda"}
    o, lse = torch.zeros(s["q"].shape, **f64), torch.full((n, heads, queries), -math.inf, **f64)
    dq, dk, dv = (torch.zeros(s[t].shape, **f64) for t in ("q", "k", "v")) if backward else (None, None, None)
    query_lengths = [queries] * n if s["query_lengths"] is None else s["query_lengths"].tolist()
    key_lengths = [keys] * n if s["key_lengths"] is None else s["key_lengths"].tolist()
    for b in range(n):
        nq, nk = query_lengths[b], key_lengths[b]
        for h in range(heads):
            q, k, v = s["q"][b, :nq, h].double(), s["k"][b, :nk, h // group].double(), s["v"][b, :nk, h // group].double()
            for lo in range(0, nq, 4096):
                hi = min(nq, lo + 4096)
                t = torch.matmul(q[lo:hi], k.T) * scale
                seen = torch.ones_like(t, dtype=torch.bool)
                if case["right"] >= 0:
                    seen = seen.tril(lo + nk - nq + case["right"])
                if case["left"] >= 0:
                    seen = seen.triu(lo + nk - nq - case["left"])
                if not backward:
                    t = t.where(seen, torch.tensor(-math.inf, **f64))
                    lse[b, h, lo:hi] = torch.logsumexp(t, 1)
                    o[b, lo:hi, h] = torch.nan_to_num(torch.softmax(t, 1)) @ v
                else:
                    p = torch.exp(t - s["lse"][b, h, lo:hi, None].double()).where(seen, torch.tensor(0.0, **f64))
                    do = s["do"][b, lo:hi, h].double()
                    dt = p * (do @ v.T - (do * s["o"][b, lo:hi, h].double()).sum(1, keepdim=True)) * scale
                    dq[b, lo:hi, h] = dt @ k
                    dk[b, :nk, h // group] += dt.T @ q[lo:hi]
                    dv[b, :nk, h // group] += p.T @ do
    return (dq, dk, dv) if backward else (o, lse)


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["kind"]](case, s)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def _pairs(case):
    """Visible pairs of a query and a key, over samples and heads."""
    total = 0
    for nq, nk in zip(*_lengths(case)):
        if case["left"] < 0 and case["right"] < 0:
            total += nq * nk
            continue
        for i in range(nq):
            place = i + nk - nq
            lo = max(0, place - case["left"]) if case["left"] >= 0 else 0
            hi = min(nk, place + case["right"] + 1) if case["right"] >= 0 else nk
            total += max(0, hi - lo)
    return total * case["heads"]


def work(case):
    item = torch.empty((), dtype=_DTYPES[case["dtype"]]).element_size()
    if case["kind"] == "norm":
        elems, weights = case["rows"] * case["cols"], torch.empty((), dtype=_DTYPES[case["weights"]]).element_size() * case["cols"]
        if case["step"] == "forward":
            return {"bytes": 2 * elems * item + 2 * weights, "flops": 8 * elems}
        # forward x -> y, backward x, dy -> dx and the gradients of the weights
        return {"bytes": 5 * elems * item + 5 * weights, "flops": 24 * elems}
    if case["kind"] == "rotary":
        tokens = math.prod(_grid(case))
        axes, pairs = _rotary_parts(case)
        elems = case["n"] * tokens * case["heads"] * case["dim"]
        return {"bytes": 2 * elems * item + 4 * len(axes) * tokens, "flops": 6 * case["n"] * tokens * case["heads"] * sum(pairs)}
    query_lengths, key_lengths = _lengths(case)
    q = sum(query_lengths) * case["heads"] * case["dim"]
    k = sum(key_lengths) * case["key_heads"] * case["dim"]
    pairs, dim, rows = _pairs(case), case["dim"], case["n"] * case["heads"] * case["queries"]
    full_q = rows * dim
    full_k = case["n"] * case["keys"] * case["key_heads"] * dim
    if case["step"] == "forward":
        return {"bytes": (q + 2 * k + full_q) * item + 4 * rows, "flops": 4 * dim * pairs}
    return {"bytes": (3 * q + 2 * k + full_q + 2 * full_k) * item + 4 * rows, "flops": 10 * dim * pairs}
