"""The global norm of a set of gradients, and clipping to a largest norm, for training the layers of this package: float32,
bfloat16, float16 and complex64 gradients (the weights of ``SpectralConvS2``) together, in two launches whatever their number.

``clip_grad_norm_`` is used like ``torch.nn.utils.clip_grad_norm_``.  Sums of squares are float64, the norm is a float32 scalar on the
gradients' device, and nothing waits for the device.  Where the norm is within the limit the gradients are not touched.

Where parameters are sharded over processes (``distributed.DistributedSpectralConvS2`` keeps its own degrees on each rank), take
``global_norm`` of the sharded and of the replicated gradients on every rank, add the squares of the former over the group,
and hand the joined norm to ``clip_grads_with_norm_``.
"""

import math
from array import array
from operator import attrgetter
from typing import Iterable, Tuple, Union

import torch

from . import _lib

_get_grad, _get_dtype = attrgetter("grad"), attrgetter("dtype")
_get_device, _is_contiguous, _data_ptr, _numel = torch.Tensor.get_device, torch.Tensor.is_contiguous, torch.Tensor.data_ptr, torch.Tensor.numel
_is_conj, _is_neg = torch.Tensor.is_conj, torch.Tensor.is_neg

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.complex64: _lib.C64}


def _norm_kind(norm_type):
    norm_type = float(norm_type)
    if norm_type == 2.0:
        return _lib.NORM_L2
    if norm_type == math.inf:
        return _lib.NORM_INF
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")


def _limit(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be non-negative, got {max_norm}")
    return max_norm


def _fills_memory(t):
    """Whether the entries of ``t`` are a gapless stretch of memory, in any order of the axes."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size != 1:
            if stride != expect:
                return False
            expect *= size
    return True


def _extent(t):
    """First byte of ``t`` and the one behind its last."""
    return t.data_ptr(), t.data_ptr() + (1 + sum(st * (n - 1) for st, n in zip(t.stride(), t.shape))) * t.element_size()


def _meet(spans, distance, other_than_zero=False):
    """Whether ``sum stride_k t_k = distance`` has a solution with every ``t_k``, a difference of two indices, in its range ``lo .. hi``, for ``spans`` of
    ``(stride, lo, hi)``.  (Strides of slices are nested: one or two values of each have to be tried.)"""
    spans = sorted(spans, reverse=True)
    tries = 10000

    def solve(k, rest, zero):
        nonlocal tries
        if k == len(spans):
            return rest == 0 and not zero
        st, lo, hi = spans[k]
        least, most = (sum(q * span[i] for q, *span in spans[k + 1 :]) for i in (0, 1))
        for t in range(max(lo, -((most - rest) // st)), min(hi, (rest - least) // st) + 1):
            tries -= 1
            if tries < 0 or solve(k + 1, rest - st * t, zero and t == 0):  # (strides that need so many are taken to share)
                return True
        return False

    return solve(0, distance, other_than_zero)


def _share(a, b):
    """Whether ``a`` and ``b`` have a byte in common."""
    spans = {}
    for t, lo, hi in ((a, 0, 1), (b, -1, 0)):
        for st, n in (*zip((st * t.element_size() for st in t.stride()), t.shape), (1, t.element_size())):
            if st and n > 1:
                at = spans.setdefault(st, [0, 0])
                at[0] += lo * (n - 1)
                at[1] += hi * (n - 1)
    return _meet([(st, *at) for st, at in spans.items()], b.data_ptr() - a.data_ptr())


def _overlaps_itself(t):
    """Whether two entries of ``t`` have the same place in memory (an expanded axis, windows that overlap)."""
    axes = [(st, n) for st, n in zip(t.stride(), t.shape) if n > 1]
    strides = [st for st, _ in axes]
    return t.numel() > 0 and (0 in strides or len(set(strides)) < len(strides) or _meet([(st, 1 - n, n - 1) for st, n in axes], 0, True))


def _refuse_shared(grads, copies, what):
    """Tensors that are scaled as a copy are written back whole: raise where one shares memory with another tensor, or two of its own entries do.  (Those
    that are scaled where they are are compared by the library.)"""
    if any(g is not c and _overlaps_itself(g) for g, c in zip(grads, copies)):
        raise RuntimeError(f"{what}: two entries of a gradient share memory")
    held = sorted(((*_extent(g), g, g is not c) for g, c in zip(grads, copies) if g.numel()), key=lambda e: e[0])
    near = []  # that reach beyond the first byte of the one at hand
    for lo, hi, g, copied in held:
        near = [e for e in near if e[0] > lo]
        if any((copied or other) and _share(h, g) for _, h, other in near):
            raise RuntimeError(f"{what}: two of the gradients share memory")
        near.append((hi, g, copied))


def _refuse(tensors, what):
    """Raise for the first tensor that cannot be taken."""
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(f"{what}: expected CUDA tensors; torch_harmonics_b200 has no CPU path")
        if t.layout != torch.strided:
            raise TypeError(f"{what}: expected dense tensors, got {t.layout}")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{what}: expected float32, bfloat16, float16 or complex64 tensors, got {t.dtype}")
        if t.device != tensors[0].device:
            raise RuntimeError(f"{what}: all tensors must be on one device, got {tensors[0].device} and {t.device}")


class _List:
    """The tensors of a call, checked, gapless in memory, and as host arrays for the C ABI.

    There may be hundreds of them on every step, and each look at an attribute costs a good part of a microsecond: the checks go through
    the list a few times at C speed, and say which tensor was wrong only once one is."""

    def __init__(self, tensors, what):
        if set(map(_get_device, tensors)) != {tensors[0].get_device()} or tensors[0].get_device() < 0:
            _refuse(tensors, what)
        try:
            self.types = [_DTYPES[t] for t in map(_get_dtype, tensors)]
            self.tensors = tensors
            if not all(map(_is_contiguous, tensors)):
                _refuse(tensors, what)
                # (a slice of a larger tensor is taken as a copy)
                self.tensors = [t if _fills_memory(t) else t.contiguous() for t in tensors]
            pointers = array("Q", map(_data_ptr, self.tensors))
        except (KeyError, RuntimeError):  # (some layouts raise where they have no strides or no pointer)
            _refuse(tensors, what)
            raise
        self.device = tensors[0].device
        self.n = len(tensors)
        self._keep = (pointers, array("q", map(_numel, self.tensors)), array("i", self.types))
        self.src, self.numel, self.dtype = (a.buffer_info()[0] for a in self._keep)


def _workspace(lib, ls):
    nbytes = lib.shtb200_grad_norm_workspace_bytes(ls.n)
    return torch.empty(nbytes, dtype=torch.uint8, device=ls.device), nbytes, torch.empty((), dtype=torch.float32, device=ls.device)


def _norm(ls, kind):
    lib = _lib.load()
    with _lib.on_device(ls.device.index) as stream:
        ws, nbytes, norm = _workspace(lib, ls)
        rc = lib.shtb200_grad_norm(ls.n, ls.src, ls.numel, ls.dtype, kind, norm.data_ptr(), ws.data_ptr(), nbytes, stream)
    _lib.check(rc, "shtb200_grad_norm")
    return norm


def _clip(ls, dst, max_norm, kind, norm=None):
    """dst = the tensors of ``ls`` clipped (``None``: in place); returns the norm, which is computed unless it is given."""
    lib = _lib.load()
    keep = None if dst is None else array("Q", map(_data_ptr, dst))
    to = ls.src if dst is None else keep.buffer_info()[0]
    with _lib.on_device(ls.device.index) as stream:
        if norm is not None:
            rc = lib.shtb200_scale_grads(ls.n, ls.src, to, ls.numel, ls.dtype, max_norm, norm.data_ptr(), stream)
        else:
            ws, nbytes, norm = _workspace(lib, ls)
            rc = lib.shtb200_clip_grads(ls.n, ls.src, to, ls.numel, ls.dtype, kind, max_norm, norm.data_ptr(), ws.data_ptr(), nbytes, stream)
    _lib.check(rc, "shtb200_clip_grads")
    return norm


def _refuse_nonfinite(norm, norm_type):
    if not math.isfinite(norm.item()):
        raise RuntimeError(f"The total norm of order {float(norm_type)} of the gradients is non-finite, so it cannot be clipped.")


def _grads(parameters):
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    return [g for g in map(_get_grad, parameters) if g is not None]


def _clip_in_place(grads, ls, max_norm, kind, what, norm=None):
    if ls.tensors is not grads:
        _refuse_shared(grads, ls.tensors, what)
    norm = _clip(ls, None, max_norm, kind, norm)
    if ls.tensors is not grads:
        for g, h in zip(grads, ls.tensors):
            if h is not g:
                g.copy_(h)
    torch.autograd.graph.increment_version(grads)
    return norm


@torch.no_grad()
def global_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all entries of ``tensors`` together (``norm_type`` 2 or inf), a float32 scalar; zero for no tensors."""
    kind = _norm_kind(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return _norm(_List(tensors, "global_norm"), kind)


@torch.no_grad()
def clip_grad_norm_(
    parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False
) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by ``min(1, max_norm / (norm + 1e-6))`` and return the norm they had.

    Parameters without a gradient are left out; gradients that share memory are refused.  A norm that is not finite makes the gradients zero or NaN, or
    raises with ``error_if_nonfinite`` (which waits for the device), before any gradient is touched."""
    kind, max_norm = _norm_kind(norm_type), _limit(max_norm)
    grads = _grads(parameters)
    if not grads:
        return torch.tensor(0.0)
    ls, norm = _List(grads, "clip_grad_norm_"), None
    if error_if_nonfinite:
        norm = _norm(ls, kind)
        _refuse_nonfinite(norm, norm_type)
    return _clip_in_place(grads, ls, max_norm, kind, "clip_grad_norm_", norm)


@torch.no_grad()
def clip_grads_with_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, total_norm: torch.Tensor) -> None:
    """``clip_grad_norm_`` with a norm that is known: a scalar on the gradients' device, e.g. one joined over several processes."""
    max_norm = _limit(max_norm)
    grads = _grads(parameters)
    if not grads:
        return
    ls = _List(grads, "clip_grads_with_norm_")
    if total_norm.numel() != 1 or total_norm.device != grads[0].device:
        raise RuntimeError(f"clip_grads_with_norm_: expected total_norm as a scalar on {grads[0].device}, got shape {tuple(total_norm.shape)} on {total_norm.device}")
    _clip_in_place(grads, ls, max_norm, _lib.NORM_L2, "clip_grads_with_norm_", _lib.dense(total_norm.to(torch.float32)))


@torch.no_grad()
def clip_by_global_norm(
    tensors: Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False
) -> Tuple[Tuple[torch.Tensor, ...], torch.Tensor]:
    """``(clipped, norm)``: new tensors ``min(1, max_norm / (norm + 1e-6)) * t`` and the norm of ``tensors``, which stay as they are
    (the gradients that ``torch.autograd.grad`` returns, or those of one micro-batch before they are accumulated)."""
    kind, max_norm = _norm_kind(norm_type), _limit(max_norm)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return (), torch.tensor(0.0)
    if any(map(_is_conj, tensors)) or any(map(_is_neg, tensors)):
        tensors = [t.resolve_conj().resolve_neg() for t in tensors]
    ls, norm = _List(tensors, "clip_by_global_norm"), None
    if error_if_nonfinite:
        norm = _norm(ls, kind)
        _refuse_nonfinite(norm, norm_type)
    dst = list(map(torch.empty_like, ls.tensors))
    norm = _clip(ls, dst, max_norm, kind, norm)
    return tuple(dst), norm
