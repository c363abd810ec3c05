"""Layers for networks that treat the cells of a grid as tokens: layer normalisation, rotary
positions, attention, on top of the C ABI (``include/h2x.h``, where the formulas stand).

Tensors are torch tensors, outermost dimension first, whose last dimension (channels, or the
elements of a head) is contiguous; the others may have any strides, so that parts of a fused
projection, a cache kept head by head, or the interior of a haloed local tensor
(``Tensor.interior_view()``) are taken where they lie.  As with the other layers the caller
brings the outputs, and calls are asynchronous on the layer's stream (or the current one).
Workspaces are made for each call, on its stream: calls on different streams and captured graphs share none.
"""
from __future__ import annotations

import ctypes
import math
from enum import Enum
from typing import Optional, Sequence, Tuple

import torch

from . import capi
from .layers import _buffer_of, _stream_handle
from .tensor import Tensor

_DTYPES = {torch.float32: capi.F32, torch.float64: capi.F64, torch.bfloat16: capi.BF16, torch.float16: capi.F16}


def _require(condition: bool, what: str) -> None:
    if not condition:
        raise ValueError(what)


def _require_int32(**counts: int) -> None:
    """Counts that the C ABI takes in 32 bits, where larger ones would wrap."""
    for what, n in counts.items():
        _require(n < 1 << 31, f"{what.replace('_', ' ')}: fewer than 2^31")


def _current_device() -> int:
    return torch._C._cuda_getDevice() if _initialized() else _first_device()


_initialized = torch.cuda.is_initialized


def _first_device() -> int:
    if not torch.cuda.is_available():
        return -1
    torch.cuda.init()
    return torch._C._cuda_getDevice()


def _on_one_gpu(device: int, stream: Optional[torch.cuda.Stream], *tensors: Optional[torch.Tensor]) -> None:
    """All tensors are on the current GPU, to which the launches go, and the layer's stream too."""
    if stream is not None and stream.device_index != device:
        raise ValueError(f"the layer's stream is on GPU {stream.device_index}, the current one is {device}")
    for t in tensors:
        if t is not None and not (t.is_cuda and t.device.index == device):
            raise ValueError(f"a tensor is on {t.device}, the current GPU is {device}")


class _Plans(dict):
    """What is worked out for tensors of given types, devices, extents and strides, for a bounded number of them."""

    def keep(self, key, plan):
        if len(self) >= 256:
            self.clear()
        self[key] = plan
        return plan


def _key(calls, device: int, stream: Optional[torch.cuda.Stream], *tensors: Optional[torch.Tensor]):
    """Equal for tensors alike, on the same current device, and streams of the same GPU (a layer's may be replaced)."""
    where = device if stream is None else device | (stream.device_index + 1) << 16
    key = calls.layout_key(where, *tensors)
    if key is None:
        key = (where, *((t.dtype, t.device, t.shape, t.stride()) if t is not None else None for t in tensors))
    return key


def _view(t):
    """A torch tensor as it is; of a local tensor its interior."""
    return t.interior_view() if isinstance(t, Tensor) else t


def _rows(t: torch.Tensor) -> Optional[capi.TensorGeometry]:
    """h2x_tensor_geometry of a tensor's rows; None for rows one after another."""
    if t.is_contiguous():
        return None
    _require(t.dim() <= capi.H2X_MAX_DIMS, f"at most {capi.H2X_MAX_DIMS} dimensions")
    _require(t.shape[-1] == 1 or t.stride(-1) == 1, "the channels of a row have to be contiguous")
    g = capi.TensorGeometry()
    g.num_dims = t.dim()
    g.local_shape[:t.dim()] = list(reversed(t.shape))
    g.strides[:t.dim()] = list(reversed(t.stride()))
    g.strides[0] = 1
    return g


def _require_own_memory(*outputs: torch.Tensor) -> None:
    _require(all(n <= 1 or s != 0 for t in outputs for n, s in zip(t.shape, t.stride())), "the elements of an output lie apart")


def _address(struct) -> Optional[int]:
    return None if struct is None else ctypes.addressof(struct)


class LayerNormalization:
    """Normalises each row (the last dimension) of a tensor by its own mean and variance.

    Elements are float32, float64, bfloat16 or float16; scale and bias of the same type or float32
    (float64 with float64), or None.  mean and rstd, which the backward pass needs, hold one float32
    (float64) a row.  Tensors of the framework are taken by their interior, the channel innermost.
    """

    def __init__(self, epsilon: float = 1e-5, stream: Optional[torch.cuda.Stream] = None):
        _require(epsilon >= 0, "epsilon has to be zero or more")
        self.epsilon, self.stream = float(epsilon), stream
        self._calls = capi.calls()
        self._plans = _Plans()

    def _plan(self, key, device: int, weights: Tuple, saved: Tuple, x: torch.Tensor, *others: torch.Tensor):
        """Types, sizes and where rows lie, checked."""
        dtype = _DTYPES.get(x.dtype)
        _require(dtype is not None, f"layer normalisation of {x.dtype} elements is not supported")
        _require(x.dim() >= 1 and x.shape[-1] >= 1, "rows of one element at least")
        channels, rows = x.shape[-1], math.prod(x.shape[:-1])
        _require_int32(channels=channels)
        for t in others:
            _require(t.shape == x.shape and t.dtype == x.dtype, "tensors of one shape and type")
        given = [w for w in weights if w is not None]
        weight_dtype = given[0].dtype if given else torch.float64 if x.dtype == torch.float64 else torch.float32
        _require(weight_dtype in (x.dtype, torch.float32) and (x.dtype != torch.float64 or weight_dtype == x.dtype),
                 "scale and bias are of the elements' type or float32")
        for w in given:
            _require(w.dtype == weight_dtype and w.shape == (channels,) and w.is_contiguous(),
                     "scale, bias and their gradients: one contiguous element of one type a channel")
        kept = torch.float64 if x.dtype == torch.float64 else torch.float32
        _require(len([s for s in saved if s is None]) in (0, len(saved)), "mean and rstd go together")
        for s in saved:
            _require(s is None or (s.dtype == kept and s.numel() == rows and s.is_contiguous()),
                     f"mean and rstd: one contiguous {kept} a row")
        _require_own_memory(others[-1])
        geometries = [_rows(t) for t in (x, *others)]
        _on_one_gpu(device, self.stream, x, *others, *weights, *saved)
        return self._plans.keep(key, (dtype, _DTYPES[weight_dtype], rows, channels, [_address(g) for g in geometries], geometries))

    def forward(self, input, scale: Optional[torch.Tensor], bias: Optional[torch.Tensor], output,
                mean: Optional[torch.Tensor] = None, rstd: Optional[torch.Tensor] = None) -> int:
        x, y, device = _view(input), _view(output), _current_device()
        key = _key(self._calls, device, self.stream, x, y, scale, bias, mean, rstd)
        plan = self._plans.get(key) or self._plan(key, device, (scale, bias), (mean, rstd), x, y)
        dtype, weight_dtype, rows, channels, (xg, yg), _ = plan
        status = self._calls.h2x_layer_norm_forward(dtype, weight_dtype, rows, channels, xg, yg, x, scale, bias, y, mean, rstd,
                                                    self.epsilon, _stream_handle(self.stream))
        if status:
            capi.check(status, "layer normalisation forward")
        return 0

    def backward(self, input, d_output, mean: torch.Tensor, rstd: torch.Tensor, scale: Optional[torch.Tensor], d_input,
                 scale_gradient: Optional[torch.Tensor] = None, bias_gradient: Optional[torch.Tensor] = None) -> int:
        """Gradients; d_input may be input or d_output itself.  Gradients of scale and bias are overwritten."""
        x, dy, dx, device = _view(input), _view(d_output), _view(d_input), _current_device()
        key = _key(self._calls, device, self.stream, x, dy, dx, mean, rstd, scale, scale_gradient, bias_gradient)
        plan = self._plans.get(key)
        if plan is None:
            _require(mean is not None and rstd is not None, "the backward pass needs mean and rstd")
            plan = self._plan(key, device, (scale, scale_gradient, bias_gradient), (mean, rstd), x, dy, dx)
        dtype, weight_dtype, rows, channels, (xg, dyg, dxg), _ = plan
        ws = None
        if scale_gradient is not None or bias_gradient is not None:
            ws = _buffer_of(self.stream, self._calls.h2x_layer_norm_workspace_bytes(dtype, rows, channels), torch.uint8)
        status = self._calls.h2x_layer_norm_backward(dtype, weight_dtype, rows, channels, xg, dyg, dxg, x, dy, mean, rstd, scale,
                                                     dx, scale_gradient, bias_gradient, ws, _stream_handle(self.stream))
        if status:
            capi.check(status, "layer normalisation backward")
        return 0


def _token_strides(t: torch.Tensor) -> capi.TokenStrides:
    """Of (samples, tokens, heads, elements)."""
    return capi.TokenStrides(t.stride(0), t.stride(1), t.stride(2))


def _is_token_tensor(t: torch.Tensor) -> bool:
    return t.dim() == 4 and (t.shape[3] == 1 or t.stride(3) == 1)


class RotaryPairing(Enum):
    """How the elements of a head are paired, with m pairs: (i, i + m), or (2 i, 2 i + 1)."""
    HALVES = capi.ROTARY_HALVES
    NEIGHBOURS = capi.ROTARY_NEIGHBOURS


def grid_positions(tensor: Tensor, dims: Optional[Sequence[int]] = None) -> torch.Tensor:
    """Positions (axes, tokens) of the cells of a local tensor in the global grid: one axis for each dimension of `dims`, innermost
    first as everywhere in the framework, None: all but the last two dimensions.  Cells are counted with the first of the
    dimensions fastest, as they lie in memory, and axes come outermost first (depth, height, width)."""
    dims = list(range(tensor.get_num_dims() - 2)) if dims is None else list(dims)
    outer_first = list(reversed(dims))
    cells = torch.meshgrid(*[torch.arange(tensor.local_shape[d], dtype=torch.int32, device=tensor.device) + tensor.global_index[d]
                             for d in outer_first], indexing="ij")
    return torch.stack([c.reshape(-1) for c in cells]).contiguous()


class RotaryPositions:
    """Turns pairs of a head's elements by angles that grow with a token's position: pair i of an axis
    with m pairs by position * base ** (-i / m).  ``axis_pairs``: how many pairs belong to each axis (time or depth, height, width); elements
    behind the pairs are copied.  ``frequencies``, a float64 tensor of one a pair, may be replaced before the first call, which copies it to the
    GPU; head_dim, axis_pairs and pairing are the layer's for good.

    x: (samples, tokens, heads, head_dim), float32, float64, bfloat16 or float16.  positions: int32, (axes, tokens) for all
    samples or (samples, axes, tokens), tokens contiguous; see grid_positions().
    """

    def __init__(self, head_dim: int, axis_pairs: Sequence[int], base: float = 10000.0,
                 pairing: RotaryPairing = RotaryPairing.HALVES, stream: Optional[torch.cuda.Stream] = None):
        self._head_dim, self._axis_pairs, self._pairing = int(head_dim), tuple(int(m) for m in axis_pairs), RotaryPairing(pairing)
        self.stream = stream
        _require(1 <= len(self.axis_pairs) <= capi.MAX_AXES and min(self.axis_pairs) >= 0, f"1 to {capi.MAX_AXES} axes")
        _require(1 <= 2 * sum(self.axis_pairs) <= self.head_dim, "the pairs of all axes have to fit a head")
        _require(base > 0, "base has to be positive")
        self._on_device = {}  # the frequencies, by the index of a GPU
        self.frequencies = torch.tensor([float(base) ** (-i / m) for m in self.axis_pairs for i in range(m)],
                                        dtype=torch.float64)
        self._calls = capi.calls()
        self._plans = _Plans()

    # (fixed: plans are made with them, and kernels read a frequency for each pair)
    @property
    def head_dim(self) -> int:
        return self._head_dim

    @property
    def axis_pairs(self) -> Tuple[int, ...]:
        return self._axis_pairs

    @property
    def pairing(self) -> RotaryPairing:
        return self._pairing

    @property
    def frequencies(self) -> torch.Tensor:
        return self._given_frequencies

    @frequencies.setter
    def frequencies(self, given: torch.Tensor) -> None:
        _require(not self._on_device, "the frequencies have been copied to a GPU by the first call there")
        self._check_frequencies(given)
        self._given_frequencies = given

    def _check_frequencies(self, given: torch.Tensor) -> None:
        _require(isinstance(given, torch.Tensor) and given.dtype == torch.float64 and tuple(given.shape) == (sum(self.axis_pairs),),
                 f"frequencies: float64, one for each of the {sum(self.axis_pairs)} pairs")

    def _frequencies(self, device: torch.device) -> torch.Tensor:
        kept = self._on_device.get(device.index)
        if kept is None:
            self._check_frequencies(self.frequencies)  # (a tensor can be resized where it is)
            _require(not torch.cuda.is_current_stream_capturing(),
                     "the first call on a GPU copies the frequencies there: make one before a graph is captured")
            own = torch.empty(len(self.frequencies), dtype=torch.float64, device=device)
            kept = self._on_device[device.index] = own.copy_(self.frequencies.detach())  # (whatever its strides were)
            torch.cuda.current_stream(device).synchronize()  # whatever stream comes next finds them
        return kept

    def _plan(self, key, device: int, x: torch.Tensor, positions: torch.Tensor, y: torch.Tensor):
        _require(x.dtype in _DTYPES, f"rotary positions of {x.dtype} elements are not supported")
        _require(_is_token_tensor(x) and _is_token_tensor(y), "(samples, tokens, heads, elements), the elements contiguous")
        _require(x.shape == y.shape and x.dtype == y.dtype, "tensors of one shape and type")
        _require_own_memory(y)
        n, tokens, heads, dim = x.shape
        _require(dim == self.head_dim, f"heads of {self.head_dim} elements, not {dim}")
        _require_int32(samples=n, heads=heads)
        axes = len(self.axis_pairs)
        _require(positions.dtype == torch.int32 and tuple(positions.shape) in ((axes, tokens), (n, axes, tokens)),
                 f"positions: int32, ({axes}, tokens) or (samples, {axes}, tokens)")
        _require(tokens <= 1 or positions.stride(-1) == 1, "positions of an axis have to be contiguous")
        r = capi.Rotary()
        r.dtype, r.pairing, r.head_dim, r.heads, r.samples, r.num_axes, r.tokens = (
            _DTYPES[x.dtype], self.pairing.value, dim, heads, n, axes, tokens)
        r.axis_pairs[:axes] = self.axis_pairs
        r.positions_sample_stride = positions.stride(0) if positions.dim() == 3 else 0
        r.positions_axis_stride = positions.stride(-2)
        r.x, r.y = _token_strides(x), _token_strides(y)
        _on_one_gpu(device, self.stream, x, positions, y)
        return self._plans.keep(key, (ctypes.addressof(r), x.stride() == y.stride(), r, self._frequencies(x.device)))

    def _apply(self, x: torch.Tensor, positions: torch.Tensor, y: torch.Tensor, inverse: int) -> int:
        device = _current_device()
        key = _key(self._calls, device, self.stream, x, positions, y)
        address, alike, _, frequencies = self._plans.get(key) or self._plan(key, device, x, positions, y)
        if not alike:
            _require(x.data_ptr() != y.data_ptr(), "in place: the same strides")
        status = self._calls.h2x_rotary_apply(address, x, positions, frequencies, inverse, y, _stream_handle(self.stream))
        if status:
            capi.check(status, "rotary positions")
        return 0

    def forward(self, x: torch.Tensor, positions: torch.Tensor, y: torch.Tensor) -> int:
        """y may be x itself."""
        return self._apply(x, positions, y, 0)

    def backward(self, dy: torch.Tensor, positions: torch.Tensor, dx: torch.Tensor) -> int:
        """The gradient: the same turn, backwards.  dx may be dy itself."""
        return self._apply(dy, positions, dx, 1)


class Attention:
    """softmax(scale * q k^T) v over the keys that a query sees, forward and backward.

    query: (samples, queries, heads, head_dim); key, value: (samples, keys, key_heads, head_dim), where key_heads divides heads: query
    head h uses key head h // (heads // key_heads).  bfloat16 or float32, heads of up to 128 elements.  (float16 is refused: without
    a scale chosen for them, the gradients of small probabilities fall below its smallest numbers.)

    ``window`` = (left, right): the last query of a sample stands at its last key, and a query sees the keys from `left` before its
    own place to `right` behind it; None: no bound.  ``causal``: no key behind its own place.
    ``query_lengths``, ``key_lengths``: int32 on the GPU, one a sample, for padded batches and caches; None: samples are whole.  Rows behind a
    sample's lengths are not read; their outputs and gradients are zero, as are those of queries that see no key, whose logsumexp is minus infinity.
    Keys and values that any query sees have to be finite (float32: below 3e38), and values times 2^8 times the number of keys below 2^128 (sums are
    in 32 bits, and divided at the end).  A query with a score that is NaN or plus infinity has an
    output and a logsumexp of NaN.
    """

    def __init__(self, scale: Optional[float] = None, causal: bool = False,
                 window: Tuple[Optional[int], Optional[int]] = (None, None), stream: Optional[torch.cuda.Stream] = None):
        left, right = window
        _require(all(w is None or 0 <= w < 1 << 63 for w in (left, right)), "a window reaches zero or more keys to either side, below 2^63")
        _require(scale is None or 1e-30 <= scale <= 1e30, "scale has to be positive, from 1e-30 to 1e30")
        if causal:
            _require(right in (None, 0), "a causal window has no keys behind a query's place")
            right = 0
        self._scale, self._window, self.stream = scale, (left, right), stream  # (fixed: plans are made with them)
        self._calls = capi.calls()
        self._plans = _Plans()

    @property
    def scale(self) -> Optional[float]:
        return self._scale

    @property
    def window(self) -> Tuple[Optional[int], Optional[int]]:
        return self._window

    def _plan(self, key, device: int, q, k, v, o, lse, lengths, gradients=()):
        """h2x_attention for these tensors, checked."""
        tensors = (q, k, v, o, *gradients)
        _require(q.dtype in (torch.bfloat16, torch.float32), f"attention of {q.dtype} elements is not supported")
        _require(all(_is_token_tensor(t) and t.dtype == q.dtype for t in tensors),
                 "(samples, tokens, heads, elements) of one type, the elements contiguous")
        _require_own_memory(*(gradients[1:] or (o,)))
        n, queries, heads, dim = q.shape
        keys, key_heads = k.shape[1:3]
        like_q, like_k = (o, *gradients[:2]), (v, *gradients[2:])
        _require(k.shape == (n, keys, key_heads, dim) and all(t.shape == k.shape for t in like_k)
                 and all(t.shape == q.shape for t in like_q), "shapes of queries, keys, values and outputs do not fit together")
        _require(1 <= dim <= 128, "heads of 1 to 128 elements")
        _require_int32(samples=n, heads=heads, key_heads=key_heads)
        _require(heads == 0 or (key_heads > 0 and heads % key_heads == 0), "the number of key heads has to divide that of heads")
        _require(lse is None or (lse.dtype == torch.float32 and lse.shape == (n, heads, queries) and lse.is_contiguous()),
                 "logsumexp: contiguous float32 (samples, heads, queries)")
        for l in lengths:
            _require(l is None or (l.dtype == torch.int32 and l.shape == (n,) and l.is_contiguous()),
                     "lengths: contiguous int32, one a sample")
        a = capi.Attention()
        a.dtype, a.head_dim, a.samples, a.query_heads, a.key_heads, a.queries, a.keys = (
            _DTYPES[q.dtype], dim, n, heads, key_heads, queries, keys)
        a.window_left, a.window_right = (-1 if w is None else w for w in self._window)
        a.scale = dim ** -0.5 if self._scale is None else self._scale
        for name, t in zip(("q", "k", "v", "o", "d_o", "dq", "dk", "dv"), tensors):
            setattr(a, name, _token_strides(t))
        _on_one_gpu(device, self.stream, *tensors, lse, *lengths)
        address = ctypes.addressof(a)
        count = (self._calls.h2x_attention_backward_workspace_bytes if gradients
                 else self._calls.h2x_attention_forward_workspace_bytes)
        return self._plans.keep(key, (address, count(address), a))

    def forward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, output: torch.Tensor,
                logsumexp: Optional[torch.Tensor] = None, query_lengths: Optional[torch.Tensor] = None,
                key_lengths: Optional[torch.Tensor] = None) -> int:
        """logsumexp, (samples, heads, queries), is for the backward pass.  output may be query itself (the same strides), and overlap no input
        otherwise."""
        device = _current_device()
        alike = _key(self._calls, device, self.stream, query, key, value, output, logsumexp, query_lengths, key_lengths)
        address, nbytes, _ = self._plans.get(alike) or self._plan(alike, device, query, key, value, output, logsumexp,
                                                                  (query_lengths, key_lengths))
        ws = _buffer_of(self.stream, nbytes, torch.uint8) if nbytes else None
        status = self._calls.h2x_attention_forward(address, query, key, value, query_lengths, key_lengths, output, logsumexp, ws,
                                                   _stream_handle(self.stream))
        if status:
            capi.check(status, "attention forward")
        return 0

    def backward(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, output: torch.Tensor,
                 d_output: torch.Tensor, logsumexp: torch.Tensor, d_query: torch.Tensor, d_key: torch.Tensor,
                 d_value: torch.Tensor, query_lengths: Optional[torch.Tensor] = None,
                 key_lengths: Optional[torch.Tensor] = None) -> int:
        """Gradients, from the forward pass' output and logsumexp; they may not overlap the inputs."""
        device = _current_device()
        alike = _key(self._calls, device, self.stream, query, key, value, output, d_output, logsumexp, d_query, d_key, d_value, query_lengths,
                     key_lengths)
        plan = self._plans.get(alike)
        if plan is None:
            _require(logsumexp is not None, "the backward pass needs logsumexp")
            plan = self._plan(alike, device, query, key, value, output, logsumexp, (query_lengths, key_lengths),
                              (d_output, d_query, d_key, d_value))
        address, nbytes, _ = plan
        ws = _buffer_of(self.stream, nbytes, torch.uint8) if nbytes else None
        status = self._calls.h2x_attention_backward(address, query, key, value, output, d_output, logsumexp, query_lengths,
                                                    key_lengths, d_query, d_key, d_value, ws, _stream_handle(self.stream))
        if status:
            capi.check(status, "attention backward")
        return 0
