"""CPU-only checks of the normalisation module and of gradient clipping: construction, buffers, refusals before any device work."""

import copy
import ctypes
import math
import pickle

import numpy as np
import pytest
import torch

import torch_harmonics_b200 as th
from oracle import sht_oracle as orc
from torch_harmonics_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


@pytest.mark.parametrize("grid", ["equiangular", "legendre-gauss", "lobatto"])
def test_latitude_weights(grid):
    m = th.GroupNormS2(2, 4, (13, 24), grid=grid)
    w = th.QuadratureS2((13, 24), grid=grid).quad_weight[0, 0, :, 0].double()
    assert m.lat_weights.dtype == torch.float32
    assert np.allclose(m.lat_weights.double().numpy(), (w / w.mean()).numpy(), rtol=1e-6)
    assert th.GroupNormS2(2, 4, (13, 24), grid=grid, weighted=False).lat_weights is None


def test_module_state():
    m = th.GroupNormS2(2, 4, (13, 24), activation="gelu")
    assert set(m.state_dict()) == {"weight", "bias"}
    assert not list(th.GroupNormS2(2, 4, (13, 24), affine=False).parameters())
    lat = m.lat_weights.clone()
    for n in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert torch.equal(n.lat_weights, lat) and n.activation == "gelu"
    m = m.half()
    assert m.weight.dtype == torch.float16 and m.lat_weights.dtype == torch.float32 and torch.equal(m.lat_weights, lat)
    assert "num_groups=2" in repr(m)


def test_construction_refusals():
    for bad in (dict(num_groups=3, num_channels=4), dict(num_groups=0, num_channels=4), dict(num_groups=1, num_channels=0), dict(num_groups=1, num_channels=4097)):
        with pytest.raises(ValueError):
            th.GroupNormS2(**bad, img_shape=(13, 24))
    with pytest.raises(ValueError, match="Unknown activation"):
        th.GroupNormS2(2, 4, (13, 24), activation="tanh")
    with pytest.raises(ValueError, match="Unknown quadrature mode"):
        th.GroupNormS2(2, 4, (13, 24), grid="hexagonal")
    for eps in (-1.0, math.nan):
        with pytest.raises(ValueError, match="eps"):
            th.GroupNormS2(2, 4, (13, 24), eps=eps)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="no CPU path"):
        th.GroupNormS2(2, 4, (13, 24))(torch.zeros(1, 4, 13, 24))
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    for call in (lambda: th.clip_grad_norm_([p], 1.0), lambda: th.clip_by_global_norm([p.grad], 1.0), lambda: th.global_norm(p.grad)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_clipping_arguments():
    p = torch.nn.Parameter(torch.ones(3))
    for bad in (1.0, 0.0, 3, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            th.clip_grad_norm_([p], 1.0, norm_type=bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            th.clip_grad_norm_([p], bad)
        with pytest.raises(ValueError, match="max_norm"):
            th.clip_by_global_norm([torch.ones(3)], bad)
    # nothing to clip
    assert float(th.clip_grad_norm_([p], 1.0)) == 0.0 and float(th.clip_grad_norm_([], 1.0)) == 0.0
    new, n = th.clip_by_global_norm([], 1.0)
    assert new == () and float(n) == 0.0 and float(th.global_norm([])) == 0.0
    assert th.clip_grads_with_norm_([p], 1.0, torch.tensor(1.0)) is None


def test_c_abi_refuses_bad_descriptors(lib):
    good = dict(batch=1, channels=4, groups=2, nlat=8, nlon=16, dtype=0, param_dtype=0, channels_last=0, activation=0, eps=1e-5)
    assert lib.shtb200_group_norm_workspace_bytes(_lib.GroupNormDesc(**good), 0) > 0
    fake = 256  # never read: refused first
    for bad in (dict(batch=-1), dict(channels=0), dict(groups=3), dict(groups=0), dict(nlat=0), dict(nlon=-4), dict(dtype=3), dict(dtype=-1), dict(param_dtype=7),
                dict(activation=9), dict(eps=-1.0), dict(eps=math.nan), dict(batch=1 << 20, channels=1 << 10), dict(nlat=1 << 17, nlon=1 << 17)):  # fmt: skip
        d = _lib.GroupNormDesc(**{**good, **bad})
        assert lib.shtb200_group_norm_workspace_bytes(d, 0) == 0
        assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake, fake, fake, 1 << 30, None) == -1
        assert lib.shtb200_group_norm_backward(d, fake, fake, None, None, None, fake, fake, None, None, fake, 1 << 30, None) == -1
    d = _lib.GroupNormDesc(**good)
    assert lib.shtb200_group_norm_forward(None, fake, None, None, None, fake, fake, fake, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_forward(d, None, None, None, None, fake, fake, fake, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake, fake, fake, 8, None) == -3
    assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake, fake, None, 1 << 30, None) == -3
    assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake + 4, fake, fake, 1 << 30, None) == -1 and b"modulo 16" in lib.shtb200_last_error()
    assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake, fake + 8, fake, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_forward(d, fake, None, None, None, fake, fake, fake + 16, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_backward(d, fake + 4, fake, None, None, None, fake, fake, None, None, fake, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_backward(d, fake, fake, None, None, None, fake, fake + 2, None, None, fake, 1 << 30, None) == -1
    assert lib.shtb200_group_norm_backward(_lib.GroupNormDesc(**{**good, "batch": 0}), fake, fake, None, None, None, fake, fake, None, None, fake, 1 << 30, None) == -1
    # nothing to do: no device is touched
    assert lib.shtb200_group_norm_forward(_lib.GroupNormDesc(**{**good, "batch": 0}), None, None, None, None, None, None, None, 0, None) == 0
    assert lib.shtb200_group_norm_backward(d, fake, fake, None, None, None, fake, None, None, None, fake, 1 << 30, None) == 0


def _lists(tensors):
    """(count, src, numel, dtype) from (address, entries, type) triples that are never read."""
    n = len(tensors)
    return n, (ctypes.c_uint64 * n)(*[t[0] for t in tensors]), (ctypes.c_int64 * n)(*[t[1] for t in tensors]), (ctypes.c_int32 * n)(*[t[2] for t in tensors])


def test_c_abi_refuses_bad_tensor_lists(lib):
    at = 1 << 20
    ws, big = 1 << 16, 1 << 30

    def clip(ts, dst=None, limit=1.0, kind=0, wsb=big):
        n, src, numel, dtype = _lists(ts)
        dst = src if dst is None else (ctypes.c_uint64 * n)(*dst)
        return lib.shtb200_clip_grads(n, src, dst, numel, dtype, kind, limit, ws, ws, wsb, None)

    assert clip([(at, 4, 0), (at + 8, 4, 0)]) == -1 and b"share memory" in lib.shtb200_last_error()
    assert clip([(at, 4, 0), (at, 4, 0)]) == -1
    assert clip([(at, 100, 3), (at + 16, 1, 1)]) == -1
    assert clip([(at, 4, 0), (at + 64, 4, 0)], dst=[at + 64, at + 128]) == -1  # one's result on another's input
    assert clip([(at, 4, 0)], dst=[at + 8]) == -1  # partly on its own input
    assert clip([(at + 2, 4, 0)]) == -1 and b"aligned" in lib.shtb200_last_error()
    assert clip([(at, -1, 0)]) == -1 and clip([(at, 4, 4)]) == -1 and clip([(0, 4, 0)]) == -1
    assert clip([(at, 4, 0)], limit=-1.0) == -1 and clip([(at, 4, 0)], limit=math.nan) == -1 and clip([(at, 4, 0)], kind=5) == -1
    assert clip([(at, 4, 0)], wsb=8) == -3
    assert lib.shtb200_clip_grads(1, None, None, None, None, 0, 1.0, ws, ws, big, None) == -1
    assert lib.shtb200_scale_grads(1, None, None, None, None, 1.0, ws, None) == -1


def test_oracle_agrees_on_the_quadrature():
    """The latitude weights are the oracle's too (independent formulas)."""
    _, w = orc.colatitudes(13, "legendre-gauss")
    m = th.GroupNormS2(1, 1, (13, 24), grid="legendre-gauss")
    assert np.allclose(m.lat_weights.double().numpy(), w / np.mean(w), rtol=1e-6)


def test_replaced_parameters_are_checked():
    def module(weight, bias):
        m = th.GroupNormS2(2, 4, (13, 24))
        m.weight = None if weight is None else torch.nn.Parameter(weight)
        m.bias = None if bias is None else torch.nn.Parameter(bias)
        return m

    cpu = torch.device("cpu")
    assert module(None, None)._affine(cpu) == (None, None)
    for weight, bias in ((torch.ones(3), torch.ones(4)), (torch.ones(4), torch.ones(5)), (torch.ones(()), torch.ones(4)), (torch.ones(1, 4), torch.ones(1, 4))):
        with pytest.raises(RuntimeError, match="of shape"):
            module(weight, bias)._affine(cpu)
    for weight, bias in ((None, torch.ones(4)), (torch.ones(4), None)):
        with pytest.raises(RuntimeError, match="both be there"):
            module(weight, bias)._affine(cpu)
    with pytest.raises(TypeError, match="must both be"):
        module(torch.ones(4), torch.ones(4).half())._affine(cpu)
    with pytest.raises(RuntimeError, match="the parameters on cpu"):
        module(torch.ones(4), torch.ones(4))._affine(torch.device("cuda", 0))
    # read as they are laid out: every other value, one value for all
    weight, bias = module(torch.arange(8.0)[::2], torch.full((1,), 3.0).expand(4))._affine(cpu)
    assert weight.is_contiguous() and bias.is_contiguous()
    assert weight.tolist() == [0.0, 2.0, 4.0, 6.0] and bias.tolist() == [3.0] * 4


def _bytes_of(t):
    at = torch.zeros((), dtype=torch.int64)
    for st, n in zip(t.stride(), t.shape):
        at = at.unsqueeze(-1) + st * torch.arange(n)
    at = (at * t.element_size() + t.data_ptr()).flatten().tolist()
    return {a + i for a in at for i in range(t.element_size())}


def test_shared_memory_is_found_exactly():
    """Against the sets of bytes: boxes of a tensor in any place, with steps, axes in any order, and of two element sizes."""
    from torch_harmonics_b200.gradients import _share

    gen = np.random.default_rng(0)
    base = torch.zeros(7, 9, 11)
    half = base.view(torch.bfloat16)

    def box():
        t = base if gen.integers(3) else half
        sl = []
        for n in t.shape:
            lo = int(gen.integers(n))
            sl.append(slice(lo, int(gen.integers(lo, n)) + 1, int(gen.integers(1, 4))))
        return t[tuple(sl)].permute(*gen.permutation(3).tolist())

    seen = set()
    for _ in range(2000):
        a, b = box(), box()
        want = bool(_bytes_of(a) & _bytes_of(b))
        seen.add(want)
        assert _share(a, b) == want and _share(b, a) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
    assert seen == {True, False}


def test_slices_that_share_memory_are_refused():
    from torch_harmonics_b200.gradients import _refuse_shared

    bucket = torch.zeros(6, 10)
    left, right = bucket[:, :4], bucket[:, 4:]

    def check(*grads):
        _refuse_shared(list(grads), [g if g.is_contiguous() else g.contiguous() for g in grads], "clip_grad_norm_")

    check(left, right, torch.zeros(3))
    check(bucket[0], bucket[1:, 2:], torch.zeros(0))
    check(bucket[::2, 1:], bucket[1::2, 1:])
    for grads in ((left, left), (left, bucket[:, 3:]), (bucket, right), (bucket[1], left, right), (torch.zeros(2), bucket.t()[2:5], right)):
        with pytest.raises(RuntimeError, match="share memory"):
            check(*grads)


def test_replaced_latitude_weights_are_checked():
    """The kernels read nlat float32 values one after the other: anything else would be read beyond its end or as something else."""
    cpu = torch.device("cpu")

    def lat(t):
        m = th.GroupNormS2(2, 4, (13, 24))
        m.lat_weights = t
        return m._lat(cpu)

    assert lat(None) is None and th.GroupNormS2(2, 4, (13, 24), weighted=False)._lat(cpu) is None
    for bad in (torch.ones(12), torch.ones(14), torch.ones(13, 1), torch.ones(()), torch.ones(0)):
        with pytest.raises(RuntimeError, match="of shape"):
            lat(bad)
    for bad in (torch.ones(13).double(), torch.ones(13).half(), torch.ones(13, dtype=torch.int32), torch.ones(13, dtype=torch.complex64)):
        with pytest.raises(TypeError, match="float32"):
            lat(bad)
    with pytest.raises(RuntimeError, match="latitude weights on cpu"):
        th.GroupNormS2(2, 4, (13, 24))._lat(torch.device("cuda", 0))
    with pytest.raises(RuntimeError, match="no gradient"):
        lat(torch.ones(13, requires_grad=True))
    # read as they are laid out: every other value, one value for all, a lazy minus sign
    for t in (torch.arange(26.0)[::2], torch.full((1,), 3.0).expand(13), torch.view_as_complex(torch.randn(13, 2)).conj().imag):
        got = lat(t)
        assert got.is_contiguous() and not got.is_neg() and got.tolist() == t.tolist()


def test_gradients_that_overlap_themselves_are_found_exactly():
    """Against the sets of places: strided views of up to three axes, any strides."""
    from torch_harmonics_b200.gradients import _overlaps_itself, _refuse_shared

    gen = np.random.default_rng(1)
    base, seen = torch.zeros(2000), set()
    for _ in range(3000):
        n = int(gen.integers(1, 4))
        shape, stride = (tuple(int(v) for v in gen.integers(lo, hi, n)) for lo, hi in ((1, 6), (0, 40)))
        t = base.as_strided(shape, stride)
        at = torch.zeros((), dtype=torch.int64)
        for st, k in zip(stride, shape):
            at = at.unsqueeze(-1) + st * torch.arange(k)
        want = at.unique().numel() < t.numel()
        seen.add(want)
        assert _overlaps_itself(t) == want, (shape, stride)
    assert seen == {True, False}
    assert not _overlaps_itself(torch.zeros(0, 3).t()) and not _overlaps_itself(torch.zeros(())) and not _overlaps_itself(base[::2])
    for bad in (torch.zeros(1).expand(5), torch.zeros(3, 1).expand(3, 4), base.as_strided((3, 3), (1, 1)), base.as_strided((4, 4), (2, 1))):
        with pytest.raises(RuntimeError, match="share memory"):
            _refuse_shared([torch.zeros(3), bad], [torch.zeros(3), bad.contiguous()], "clip_grad_norm_")


def test_c_abi_takes_long_tensors_among_many(lib):
    """The length of one tensor is not limited by how many others there are; all of a launch together by what 32 bits count.  (Nothing is launched: two of the tensors
    share memory, which is refused last.)"""
    n, long = 40_000, 1 << 30
    ts = [((1 << 20) + 64 * i, 4, 0) for i in range(n)] + [(1 << 30, long, 0), (1 << 40, long, 3), (1 << 40, long, 3)]

    def clip(ts):
        n, src, numel, dtype = _lists(ts)
        rc = lib.shtb200_clip_grads(n, src, src, numel, dtype, 0, 1.0, 1 << 16, 1 << 16, 1 << 30, None)
        return rc, lib.shtb200_last_error()

    rc, why = clip(ts)
    assert rc == -1 and b"share memory" in why
    rc, why = clip([((i + 1) << 40, 1 << 36, 0) for i in range(300)])  # 2.5e9 units
    assert rc == -1 and b"too many entries" in why
    rc, why = clip([(1 << 20, (1 << 44) + 1, 0)])
    assert rc == -1 and b"length" in why
    # as many units, but in two launches
    rc, why = clip([((i + 1) << 40, 1 << 34, 0) for i in range(1400)] + [(1 << 40, 4, 0)])
    assert rc == -1 and b"share memory" in why


def test_c_abi_refuses_a_norm_inside_the_tensors(lib):
    """Every block reads the norm while others scale: it may not lie in what is written, nor, where it is written itself, in what is read."""
    at, other, ws = 1 << 20, 1 << 21, 1 << 16
    n, src, numel, dtype = _lists([(at, 100, 0), (at + 4096, 100, 3)])
    away = (ctypes.c_uint64 * n)(other, other + 4096)
    for norm in (at, at + 396, at + 4096, at + 4096 + 796):
        assert lib.shtb200_scale_grads(n, src, src, numel, dtype, 1.0, norm, None) == -1 and b"share memory" in lib.shtb200_last_error()
        assert lib.shtb200_clip_grads(n, src, src, numel, dtype, 0, 1.0, norm, ws, 1 << 30, None) == -1 and b"share memory" in lib.shtb200_last_error()
        assert lib.shtb200_clip_grads(n, src, away, numel, dtype, 0, 1.0, norm, ws, 1 << 30, None) == -1
        assert lib.shtb200_scale_grads(n, src, away, numel, dtype, 1.0, norm + (other - at), None) == -1


def test_c_abi_refuses_values_off_their_alignment(lib):
    """All fields a byte off alike: no vector would lie on a 16-byte boundary, wherever it begins."""
    desc = dict(batch=1, channels=4, groups=2, nlat=8, nlon=16, dtype=0, param_dtype=0, channels_last=0, activation=0, eps=1e-5)
    at, ws = 4096, 1 << 20

    def forward(x=0, w=0, lat=0, **k):
        d = _lib.GroupNormDesc(**{**desc, **k})
        return lib.shtb200_group_norm_forward(d, at + x, at + lat, at + w, None, 2 * at + x, at, ws, 1 << 30, None)

    def backward(x=0, w=0, dw=0, **k):
        d = _lib.GroupNormDesc(**{**desc, **k})
        return lib.shtb200_group_norm_backward(d, at + x, 2 * at + x, None, None, at + w, at, 3 * at + x, at + dw, None, ws, 1 << 30, None)

    for rc in (lambda: forward(x=1), lambda: forward(x=2), lambda: forward(x=1, dtype=1), lambda: forward(w=2), lambda: forward(w=1, param_dtype=2), lambda: forward(lat=2),
               lambda: backward(x=3), lambda: backward(x=1, dtype=2), lambda: backward(w=2), lambda: backward(dw=1), lambda: backward(dw=1, param_dtype=1)):  # fmt: skip
        assert rc() == -1 and b"aligned to its element type" in lib.shtb200_last_error()
