"""Group normalisation on the sphere, fused with the activation behind it.

The mean and variance of a group are those of a field on the sphere: averages over its channels and grid points with the
latitude quadrature weights of the grid (``QuadratureS2``), so that the many grid points near the poles do not count for more than
their area.  ``weighted=False`` gives the plain averages over grid points of ordinary group normalisation.
"""

import functools
from typing import List, Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .quadrature import precompute_latitudes, trapezoidal_weights

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}


def _latitude_weights(nlat, grid):
    if grid == "equiangular-trapezoidal":
        return trapezoidal_weights(nlat, -1, 1)[1]
    return precompute_latitudes(nlat, grid)[1]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _aligned(t):
    """The kernels read 16 bytes at a time: a view that begins in between is copied."""
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _dense(t):
    """``_lib.dense`` of a real tensor or none, at next to no cost where there is nothing to do."""
    return t if t is None or t.is_contiguous() and not t.is_neg() else _lib.dense(t)


def _call(batch, channels, groups, nlat, nlon, dtype, param_dtype, channels_last, activation, eps):
    """(descriptor, workspace bytes forward, backward): shapes and types only."""
    desc = _lib.GroupNormDesc(batch, channels, groups, nlat, nlon, _DTYPES[dtype], _DTYPES[param_dtype], int(channels_last), _lib.ACTIVATIONS[activation], eps)
    ws = [_lib.load().shtb200_group_norm_workspace_bytes(desc, i) for i in (0, 1)]
    if ws[0] == 0:
        _lib.check(-1, "shtb200_group_norm_workspace_bytes")
    return desc, *ws


def _stats_bytes(batch, groups):
    return (16 * batch * groups + 255) // 256 * 256


def _taken(x):
    """``x`` as the kernels read it: planes or channels last, without a lazy sign, aligned."""
    if x.is_neg():
        x = x.resolve_neg()
    if not (x.is_contiguous() or x.is_contiguous(memory_format=torch.channels_last)):
        x = x.contiguous()
    return _aligned(x)


def _run(call, x, weight, bias, lat, keep):
    """y and (with ``keep``) what the backward pass needs, for a dense ``x``."""
    desc, ws_bytes, _ = call
    dev = x.device
    y = torch.empty_like(x)
    stats_bytes = _stats_bytes(desc.batch, desc.groups)
    stats = torch.empty(stats_bytes if keep else stats_bytes + ws_bytes, dtype=torch.uint8, device=dev)
    if desc.batch == 0:
        return y, stats
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if keep else None
    at = stats.data_ptr()
    with _lib.on_device(dev.index) as stream:
        rc = _lib.load().shtb200_group_norm_forward(
            desc, x.data_ptr(), _ptr(lat), _ptr(weight), _ptr(bias), y.data_ptr(), at, ws.data_ptr() if keep else at + stats_bytes, ws_bytes, stream
        )
    if rc != 0:
        _lib.check(rc, "shtb200_group_norm_forward")
    return y, stats


def _run_backward(call, dy, x, weight, bias, lat, stats, need):
    """dx, dweight, dbias, ``None`` where ``need`` says so."""
    desc, _, ws_bytes = call
    new = torch.empty_like if desc.batch else torch.zeros_like
    dx = torch.empty_like(x) if need[0] else None
    dw = new(weight) if need[1] else None
    db = new(bias) if need[2] else None
    if desc.batch == 0:
        return dx, dw, db
    # the gradient comes in any layout (an expanded scalar, for a sum): the kernel reads it in the layout of x
    dy = _aligned(_lib.dense(dy) if not desc.channels_last else dy.resolve_neg().contiguous(memory_format=torch.channels_last))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    with _lib.on_device(x.device.index) as stream:
        rc = _lib.load().shtb200_group_norm_backward(
            desc, dy.data_ptr(), x.data_ptr(), _ptr(lat), _ptr(weight), _ptr(bias), stats.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), ws.data_ptr(), ws_bytes, stream
        )
    if rc != 0:
        _lib.check(rc, "shtb200_group_norm_backward")
    return dx, dw, db


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, lat, call):
        y, stats = _run(call, x, weight, bias, lat, True)
        ctx.save_for_backward(x, weight, bias, lat, stats)
        ctx.call = call
        return y

    @staticmethod
    def backward(ctx, dy):
        # (where no graph of the gradients is built, there is nothing to guard)
        return _guarded_gradients(ctx, dy) if torch.is_grad_enabled() else _gradients(ctx, dy)


def _gradients(ctx, dy):
    x, weight, bias, lat, stats = ctx.saved_tensors
    return *_run_backward(ctx.call, dy, x, weight, bias, lat, stats, ctx.needs_input_grad), None, None


_guarded_gradients = once_differentiable(_gradients)


# Where torch.compile traces, the call is a custom operator (as the transforms are), so that a network stays one graph.  Eager calls take the function
# above instead: host time of a small call 18 us, as an operator 30, of a small training step 119 and 200.
_traced_call = functools.lru_cache(maxsize=256)(_call)


def _call_of(x, weight, groups, eps, activation):
    return _traced_call(*x.shape[:2], groups, *x.shape[2:], x.dtype, torch.float32 if weight is None else weight.dtype, not x.is_contiguous(), activation, eps)


@torch.library.custom_op("shtb200::group_norm", mutates_args=(), device_types="cuda")
def _group_norm(
    x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], lat: Optional[torch.Tensor], groups: int, eps: float, activation: Optional[str]
) -> Tuple[torch.Tensor, torch.Tensor]:
    x = _taken(x)
    return _run(_call_of(x, weight, groups, eps, activation), x, _dense(weight), _dense(bias), _dense(lat), True)


@torch.library.custom_op("shtb200::group_norm_backward", mutates_args=(), device_types="cuda")
def _group_norm_backward(
    dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], lat: Optional[torch.Tensor], stats: torch.Tensor,
    groups: int, eps: float, activation: Optional[str], need: List[bool],
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:  # fmt: skip
    x, weight, bias = _taken(x), _dense(weight), _dense(bias)
    out = _run_backward(_call_of(x, weight, groups, eps, activation), dy, x, weight, bias, _dense(lat), stats, need)
    return tuple(x.new_empty(0) if t is None else t for t in out)


def _fake_like(x):
    kept = x.is_contiguous() or x.is_contiguous(memory_format=torch.channels_last)
    return torch.empty_like(x, memory_format=torch.preserve_format if kept else torch.contiguous_format)


@_group_norm.register_fake
def _(x, weight, bias, lat, groups, eps, activation):
    return _fake_like(x), x.new_empty(_stats_bytes(x.shape[0], groups), dtype=torch.uint8)


@_group_norm_backward.register_fake
def _(dy, x, weight, bias, lat, stats, groups, eps, activation, need):
    return tuple(make(t) if n else x.new_empty(0) for t, n, make in zip((x, weight, bias), need, (_fake_like, *[lambda p: p.new_empty(p.shape)] * 2)))


def _setup(ctx, inputs, output):
    x, weight, bias, lat, *ctx.how = inputs
    ctx.save_for_backward(x, weight, bias, lat, output[1])


def _traced_gradients(ctx, dy, _):
    x, weight, bias, lat, stats = ctx.saved_tensors
    need = [bool(n) for n in ctx.needs_input_grad[:3]]
    grads = _group_norm_backward(dy, x, weight, bias, lat, stats, *ctx.how, need)
    return *(g if n else None for g, n in zip(grads, need)), None, None, None, None


_group_norm.register_autograd(_traced_gradients, setup_context=_setup)


class GroupNormS2(nn.Module):
    """``(batch, num_channels, nlat, nlon) -> `` the same shape: normalise each of ``num_groups`` groups of consecutive channels
    by its mean and variance over the sphere, scale and shift every channel (``weight``, ``bias``), apply ``activation``.

    ``num_groups = num_channels`` is instance normalisation, ``num_groups = 1`` layer normalisation over (channels, sphere).

    Parameters
    ----------
    img_shape : (nlat, nlon)
    grid : the latitude grid whose quadrature weights are used: "equiangular", "legendre-gauss", "lobatto" or "equiangular-trapezoidal"
    eps : added to the variance
    affine : whether ``weight`` and ``bias`` (num_channels,) exist
    activation : None, "relu", "silu" or "gelu" (z times the normal distribution function, exact form)
    weighted : False: every grid point counts the same, whatever the grid

    The input is float32, bfloat16 or float16, in planes (contiguous) or channels last (``torch.channels_last``); both are read
    where they are, other strides are copied first.  The output has the input's type and layout; statistics, sums and the
    activation are float32 or wider whatever the type, under autocast too.  The parameters may have any of the three types.  The
    gradients can be computed once (no second derivatives).  Calls trace into one graph under ``torch.compile``; ``vmap`` and
    forward-mode derivatives are not there.  ``lat_weights`` may be replaced by other float32 weights (nlat,) of at least 0: rows of weight 0
    (whose values have to be finite) change no statistics and are normalised like the others.

    A field is whole on its device: the tiles of ``distributed`` are not taken, since their statistics would be sums over the ranks.

    Calls may be captured into a CUDA graph.  A backward pass is captured only while no autograd graph of an eager step on the same
    parameters is alive (delete its loss first): torch accumulates gradients on the stream of that step, which ends the capture.
    """

    def __init__(
        self,
        num_groups: int,
        num_channels: int,
        img_shape: Tuple[int],
        grid: Optional[str] = "equiangular",
        eps: Optional[float] = 1e-5,
        affine: Optional[bool] = True,
        activation: Optional[str] = None,
        weighted: Optional[bool] = True,
    ):
        super().__init__()
        if num_groups < 1 or num_channels < 1:
            raise ValueError(f"num_groups ({num_groups}) and num_channels ({num_channels}) must be positive")
        if num_channels % num_groups != 0:
            raise ValueError(f"num_channels ({num_channels}) must be divisible by num_groups ({num_groups})")
        if num_channels > _lib.GROUP_NORM_MAX_CHANNELS:
            raise ValueError(f"num_channels ({num_channels}) must not exceed {_lib.GROUP_NORM_MAX_CHANNELS}")
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"Unknown activation {activation!r}, expected one of {list(_lib.ACTIVATIONS)}")
        if not eps >= 0.0:
            raise ValueError(f"eps must be non-negative, got {eps}")
        self.num_groups = num_groups
        self.num_channels = num_channels
        self.nlat, self.nlon = img_shape
        self.grid = grid
        self.eps = eps
        self.activation = activation
        self.weighted = weighted
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)
        lat = None
        if weighted:
            lat = _latitude_weights(self.nlat, grid)
            lat = (lat / lat.mean()).to(torch.float32)
        self.register_buffer("lat_weights", lat, persistent=False)
        self._calls = {}

    def extra_repr(self):
        return f"num_groups={self.num_groups}, num_channels={self.num_channels}, nlat={self.nlat}, nlon={self.nlon},\n grid={self.grid}, eps={self.eps}, activation={self.activation}, weighted={self.weighted}"

    def _apply(self, fn, *args, **kwargs):
        # the module may be cast to half precision: the latitude weights move with it but stay float32
        lat = self.lat_weights
        out = super()._apply(fn, *args, **kwargs)
        if lat is not None and self.lat_weights.dtype != lat.dtype:
            self.lat_weights = lat.to(device=self.lat_weights.device)
        return out

    def __getstate__(self):
        state = super().__getstate__() if hasattr(super(), "__getstate__") else self.__dict__
        return {**state, "_calls": {}}

    def _affine(self, device, traced=False):
        """``weight`` and ``bias`` as the kernels read them (``traced``: as they are).  They may have been replaced since the module was made."""
        weight, bias = self.weight, self.bias
        if weight is None and bias is None:
            return None, None
        if weight is None or bias is None:
            raise RuntimeError("GroupNormS2: weight and bias must both be there, or neither")
        if weight.device != device or bias.device != device:
            raise RuntimeError(f"GroupNormS2: the input is on {device}, the parameters on {weight.device} and {bias.device}")
        if weight.dtype not in _DTYPES or bias.dtype != weight.dtype:
            raise TypeError(f"GroupNormS2: weight and bias must both be float32, bfloat16 or float16, got {weight.dtype} and {bias.dtype}")
        if weight.shape != (self.num_channels,) or bias.shape != (self.num_channels,):
            raise RuntimeError(f"GroupNormS2: expected weight and bias of shape ({self.num_channels},), got {tuple(weight.shape)} and {tuple(bias.shape)}")
        if traced:
            return weight, bias
        return _dense(weight), _dense(bias)  # (one value expanded to all channels is a copy here, and its gradient a sum)

    def _lat(self, device, traced=False):
        """``lat_weights`` as the kernels read them.  They may have been replaced too (by a mask of rows, for instance)."""
        lat = self._buffers["lat_weights"] if "lat_weights" in self._buffers else self.lat_weights  # (the attribute takes five times as long)
        if lat is None:
            return None
        if lat.device != device:
            raise RuntimeError(f"GroupNormS2: the input is on {device}, the latitude weights on {lat.device}")
        if lat.dtype != torch.float32:
            raise TypeError(f"GroupNormS2: lat_weights must be float32, got {lat.dtype}")
        if lat.shape != (self.nlat,):
            raise RuntimeError(f"GroupNormS2: expected lat_weights of shape ({self.nlat},), got {tuple(lat.shape)}")
        if lat.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("GroupNormS2: lat_weights get no gradient, they must not require one")
        return lat if traced else _dense(lat)

    def _call(self, x, weight):
        param = torch.float32 if weight is None else weight.dtype
        cl = not x.is_contiguous()
        key = (x.shape[0], x.dtype, param, cl, self.eps, self.activation)
        call = self._calls.get(key)
        if call is None:
            call = self._calls[key] = _call(x.shape[0], self.num_channels, self.num_groups, self.nlat, self.nlon, x.dtype, param, cl, self.activation, self.eps)
        return call

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not x.is_cuda:
            raise RuntimeError("GroupNormS2: expected a CUDA tensor; torch_harmonics_b200 has no CPU path")
        if x.dtype not in _DTYPES:
            raise TypeError(f"GroupNormS2: expected dtype torch.float32, torch.bfloat16 or torch.float16, got {x.dtype}")
        if x.dim() != 4:
            raise RuntimeError(f"Expected tensor with 4 dimensions but got {x.dim()} instead")
        if x.shape[1:] != (self.num_channels, self.nlat, self.nlon):
            raise RuntimeError(f"Expected shape (batch, {self.num_channels}, {self.nlat}, {self.nlon}), got {tuple(x.shape)}")
        traced, device = torch.compiler.is_compiling(), x.device
        weight, bias = self._affine(device, traced)
        lat = self._lat(device, traced)
        if traced:
            return _group_norm(x, weight, bias, lat, self.num_groups, self.eps, self.activation)[0]
        x = _taken(x)
        call = self._call(x, weight)
        if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and (weight.requires_grad or bias.requires_grad))):
            return _GroupNorm.apply(x, weight, bias, lat, call)
        return _run(call, x, weight, bias, lat, False)[0]
