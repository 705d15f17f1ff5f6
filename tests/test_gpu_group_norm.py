"""GPU tests of GroupNormS2 (values, gradients, layouts, types, streams, capture) against the formulas in float64.

Tolerances.  In float32 a value of z = weight xh + bias carries at most 168 roundings of 2^-24 relative to |weight xh| + |bias| + 1 (about 128 sequential
additions in a thread's share of a sum, 40 elsewhere), which is 1.0e-5; the gradients likewise, relative to the sizes of the terms they
are sums of.  A result held in fewer bits is off by half a step more: 2^-8 (bfloat16), 2^-11 (float16), 2^-24 (float32)."""

import math
import warnings

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F = 1.0e-5
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0**-25}  # half a step of a subnormal number
FORMATS = {"planes": torch.contiguous_format, "last": torch.channels_last}


def _module(G, C, H, W, **k):
    import torch_harmonics_b200 as th

    return th.GroupNormS2(G, C, (H, W), **k).cuda()


def _act(z, kind):
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if kind == "gelu":
        cdf = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _exact(m, x, dy):
    """y, dx, dweight, dbias and how far each may be off in float32 arithmetic (see above), all float64."""
    B, C, H, W = x.shape
    G = m.num_groups
    a = torch.ones(H, dtype=torch.float64, device=x.device) if m.lat_weights is None else m.lat_weights.double()
    q = (a / (a.sum() * W * (C // G))).view(1, 1, 1, H, 1)
    w = (torch.ones(C, device=x.device) if m.weight is None else m.weight.detach()).double().view(1, G, C // G, 1, 1)
    b = (torch.zeros(C, device=x.device) if m.bias is None else m.bias.detach()).double().view(1, G, C // G, 1, 1)
    v, d = x.double().view(B, G, C // G, H, W), dy.double().view(B, G, C // G, H, W)

    def tot(t):
        return t.sum((2, 3, 4), keepdim=True)

    mu = tot(q * v)
    r = 1 / torch.sqrt(tot(q * (v - mu) ** 2) + m.eps)
    xh = (v - mu) * r
    z = xh * w + b
    y, slope = _act(z, m.activation)
    g = d * slope
    h = g * w
    dx = r * (h - q * (tot(h) + xh * tot(h * xh)))
    size = 1 + (xh * w).abs() + b.abs()
    gs = d.abs() * size
    hs = gs * w.abs()
    tol = [F * size, F * r * (hs + q * (tot(hs) + xh.abs() * tot(hs * (1 + xh.abs()))) * 2)]
    out = [y.reshape(x.shape), dx.reshape(x.shape), (g * xh).sum((0, 3, 4)).reshape(C), g.sum((0, 3, 4)).reshape(C)]
    tol = [t.reshape(x.shape) for t in tol] + [F * (gs * (1 + xh.abs())).sum((0, 3, 4)).reshape(C), F * gs.sum((0, 3, 4)).reshape(C)]
    return out, tol


def _inputs(shape, dtype, fmt, seed=0, level=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, C = shape[:2]
    x = torch.randn(shape, device="cuda", generator=gen) * torch.exp(0.5 * torch.randn(1, C, 1, 1, device="cuda", generator=gen))
    x = (x + 2 * torch.randn(B, C, 1, 1, device="cuda", generator=gen) + level).to(dtype).contiguous(memory_format=FORMATS[fmt])
    dy = torch.randn(shape, device="cuda", generator=gen).to(dtype).contiguous(memory_format=FORMATS[fmt])
    return x, dy


def _parameters(m, seed=1):
    if m.weight is not None:
        gen = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            m.weight.copy_(1 + 0.3 * torch.randn(m.num_channels, device="cuda", generator=gen))
            m.bias.copy_(0.3 * torch.randn(m.num_channels, device="cuda", generator=gen))


def _smooth_at_zero(m, x, dy):
    """No gradient where z is next to relu's corner (a rounding decides the side there)."""
    if m.activation == "relu":
        m.activation = None
        z = _exact(m, x, dy)[0][0]
        m.activation = "relu"
        dy = dy.masked_fill(z.abs() < 1e-3, 0)
    return dy


def _compare(got, want, tol, what=""):
    for name, o, e, t in zip(("y", "dx", "dweight", "dbias"), got, want, tol):
        if o is None:
            continue
        d = (o.double() - e).abs()
        bound = t + HALF[o.dtype] * e.abs() + TINY[o.dtype]
        assert torch.isfinite(o).all(), f"{what} {name} not finite"
        assert (d <= bound).all(), f"{what} {name}: {float((d / bound).max()):.2f} times the bound"


def _step(m, x, dy):
    x = x.detach().requires_grad_(True)
    y = m(x)
    if m.weight is None:
        return [y.detach(), *torch.autograd.grad(y, (x,), dy), None, None]
    return [y.detach(), *torch.autograd.grad(y, (x, m.weight, m.bias), dy)]


# batch, channels, groups, nlat, nlon
SHAPES = [
    (1, 1, 1, 2, 1), (2, 6, 3, 5, 7), (3, 5, 5, 9, 17), (1, 8, 4, 33, 64), (2, 73, 1, 17, 33), (2, 73, 73, 12, 24), (2, 64, 8, 16, 32), (1, 300, 4, 8, 9),
    (2, 520, 8, 6, 10), (1, 3, 1, 129, 257), (1, 1100, 100, 5, 8), (5, 24, 2, 31, 62), (1, 2, 1, 3, 1), (1, 2500, 5, 3, 4), (70, 2, 2, 4, 6), (1, 4, 4, 181, 360), (1, 32, 2, 91, 180),
    (1, 4096, 4096, 3, 4), (1, 4096, 1, 2, 3), (2, 129, 43, 7, 9), (1, 1032, 8, 16, 31), (3, 64, 1, 24, 48),
]  # fmt: skip


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_values_and_gradients(shape, dtype, fmt):
    B, C, G, H, W = shape
    n = SHAPES.index(shape) + (fmt == "last")
    m = _module(G, C, H, W, activation=[None, "relu", "silu", "gelu"][n % 4], grid=["equiangular", "legendre-gauss", "lobatto"][n % 3], weighted=n % 5 != 0, affine=n % 7 != 0)
    _parameters(m)
    x, dy = _inputs((B, C, H, W), dtype, fmt)
    dy = _smooth_at_zero(m, x, dy)
    got = _step(m, x, dy)
    assert got[0].dtype == dtype and got[0].stride() == x.stride() and got[1].stride() == x.stride()
    _compare(got, *_exact(m, x, dy))
    with torch.no_grad():
        assert torch.equal(m(x), got[0])


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_activations(act, dtype, fmt):
    """Every activation over a wide range of z: weights up to 8, so that the tails of the activations are reached."""
    m = _module(4, 16, 45, 90, activation=act)
    with torch.no_grad():
        m.weight.copy_(torch.linspace(-8, 8, 16))
        m.bias.copy_(torch.linspace(3, -3, 16))
    x, dy = _inputs((2, 16, 45, 90), dtype, fmt, seed=3)
    dy = _smooth_at_zero(m, x, dy)
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("param", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_parameter_types(param, fmt):
    m = _module(3, 12, 16, 32, activation="silu")
    _parameters(m)
    m = m.to(param)
    assert m.lat_weights.dtype == torch.float32 and m.weight.dtype == param
    x, dy = _inputs((2, 12, 16, 32), param, fmt)
    got = _step(m, x, dy)
    assert got[2].dtype == param and got[3].dtype == param
    _compare(got, *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_level_far_above_spread(fmt):
    """Fields like surface pressure: a level of 1e5 with a spread of about one.  The inputs are exact, so the bound is the same."""
    m = _module(2, 6, 61, 120, activation="gelu")
    _parameters(m)
    x, dy = _inputs((2, 6, 61, 120), torch.float32, fmt, level=1.0e5)
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("where", ["first", "pole", "middle"])
def test_one_point_far_out(where, fmt):
    """One value of 1e4 spreads; the statistics may not lose the others.  (Same bound: it is relative to |xh|.)"""
    m = _module(2, 6, 61, 120)
    x, dy = _inputs((1, 6, 61, 120), torch.float32, fmt)
    i, j = {"first": (0, 0), "pole": (60, 119), "middle": (30, 7)}[where]
    x[:, :, i, j] = 1.0e4
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_constant_fields_give_the_shift(fmt):
    m = _module(2, 4, 19, 36)
    _parameters(m)
    x = torch.full((2, 4, 19, 36), 1234.567, device="cuda").contiguous(memory_format=FORMATS[fmt])
    y = m(x)
    assert torch.equal(y, m.bias.view(1, 4, 1, 1).expand_as(y))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_nonfinite_values_stay_in_their_group(bad, fmt):
    m = _module(3, 6, 33, 64, activation="relu")
    x, dy = _inputs((2, 6, 33, 64), torch.float32, fmt)
    x[1, 3, 5, 7] = bad
    y, dx = _step(m, x, dy)[:2]
    hit = torch.zeros(2, 6, dtype=torch.bool, device="cuda")
    hit[1, 2:4] = True
    assert torch.equal(torch.isnan(y).any(-1).any(-1), hit) and torch.isnan(y[1, 2:4]).all()
    assert torch.equal(torch.isnan(dx).any(-1).any(-1), hit)


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_gradient_against_differences(fmt):
    """The loss sum(dy y) along a random direction, by central differences of the float64 formulas at the float32 inputs."""
    m = _module(2, 8, 17, 32, activation="gelu")
    _parameters(m)
    x, dy = _inputs((2, 8, 17, 32), torch.float32, fmt, seed=9)
    dx = _step(m, x, dy)[1].double()
    u = torch.randn_like(x)

    def loss(t):
        return (_exact(m, x.double() + t * u.double(), dy)[0][0] * dy.double()).sum()

    e = 1e-4
    slope = (8 * (loss(e) - loss(-e)) - (loss(2 * e) - loss(-2 * e))) / (12 * e)  # (error e^4 times the fifth derivative)
    assert abs(float((dx * u.double()).sum() - slope)) <= 2 * F * float((dx * u.double()).abs().sum())


def test_layouts_and_strides_agree():
    m = _module(2, 6, 20, 40, activation="silu")
    _parameters(m)
    wide = torch.randn(2, 9, 20, 45, device="cuda")
    x = wide[:, 1:7, :, 2:42]  # a slice: neither layout, copied
    y = m(x)
    assert y.is_contiguous() and torch.equal(y, m(x.contiguous()))
    last = m(x.contiguous(memory_format=torch.channels_last))
    assert (y - last).abs().max() <= 2 * F * (1 + y.abs().max())
    flipped = torch.randn(2, 40, 20, 6, device="cuda").permute(0, 3, 2, 1)  # width before height
    assert torch.equal(m(flipped), m(flipped.contiguous()))
    # a gradient in another layout than the input's, and an expanded one
    x = x.contiguous(memory_format=torch.channels_last).requires_grad_(True)
    dy = torch.randn(2, 6, 20, 40, device="cuda")
    (g1,) = torch.autograd.grad(m(x), x, dy)
    (g2,) = torch.autograd.grad(m(x), x, dy.contiguous(memory_format=torch.channels_last))
    assert torch.equal(g1, g2)
    (g3,) = torch.autograd.grad(m(x).sum(), x)
    (g4,) = torch.autograd.grad(m(x), x, torch.ones_like(x))
    assert torch.equal(g3, g4)
    # the imaginary part of a conjugate carries a lazy minus sign
    z = torch.view_as_complex(torch.randn(2, 6, 20, 40, 2, device="cuda"))
    assert torch.equal(m(z.conj().imag), m(-z.imag.contiguous()))


@pytest.mark.parametrize("offset", [1, 3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_views_at_any_alignment(fmt, dtype, offset):
    """A dense tensor that starts at an odd element of its memory."""
    shape = (2, 8, 24, 48)
    m = _module(4, 8, 24, 48, activation="gelu")
    _parameters(m)
    x, dy = _inputs(shape, dtype, fmt)

    def moved(t):
        flat = torch.zeros(t.numel() + 8, dtype=t.dtype, device="cuda")
        v = torch.as_strided(flat, t.shape, t.stride(), offset)
        v.copy_(t)
        return v

    a, b = _step(m, x, dy), _step(m, moved(x), moved(dy))
    _compare(b, *_exact(m, x, dy))
    assert a[0].stride() == b[0].stride()


def test_only_some_gradients():
    m = _module(2, 6, 16, 32, activation="gelu")
    _parameters(m)
    x, dy = _inputs((2, 6, 16, 32), torch.float32, "last")
    _, dx, dw, db = _step(m, x, dy)
    m.bias.requires_grad_(False)
    y = m(x)  # the input needs none
    y.backward(dy)
    assert torch.equal(m.weight.grad, dw) and m.bias.grad is None
    m.weight.requires_grad_(False)
    xg = x.clone().requires_grad_(True)
    m(xg).backward(dy)
    assert torch.equal(xg.grad, dx)
    assert not m(x).requires_grad


def test_empty_batch():
    m = _module(2, 6, 16, 32)
    x = torch.empty(0, 6, 16, 32, device="cuda", requires_grad=True)
    y = m(x)
    assert y.shape == x.shape
    y.sum().backward()
    assert x.grad.shape == x.shape and m.weight.grad.abs().sum() == 0 and m.bias.grad.abs().sum() == 0


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_repeats_exactly_and_on_another_stream(fmt):
    m = _module(4, 24, 61, 120, activation="gelu")
    _parameters(m)
    x, dy = _inputs((3, 24, 61, 120), torch.bfloat16, fmt)
    first = _step(m, x, dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _step(m, x, dy)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for s in streams:  # calls on three streams at once
        with torch.cuda.stream(s):
            outs.append(_step(m, x, dy))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(first, o))


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_captured_and_replayed(fmt):
    """Forward and backward in a graph, replayed on new inputs; two graphs that share a memory pool."""
    m = _module(4, 24, 33, 64, activation="gelu")
    _parameters(m)
    x, dy = _inputs((2, 24, 33, 64), torch.float32, fmt)
    x.requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(m(x), (x, m.weight, m.bias), dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs, results = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            y = m(x)
            results.append([y, *torch.autograd.grad(y, (x, m.weight, m.bias), dy)])
        graphs.append(g)
    for seed in (5, 6):
        nx, ndy = _inputs((2, 24, 33, 64), torch.float32, fmt, seed=seed)
        with torch.no_grad():
            x.copy_(nx)
            dy.copy_(ndy)
        want = _step(m, nx, ndy)
        for g, res in zip(graphs, results):
            g.replay()
            assert all(torch.equal(a.detach(), b) for a, b in zip(res, want))


def test_in_place_use_of_the_input_is_noticed():
    m = _module(2, 6, 16, 32)
    x = torch.randn(1, 6, 16, 32, device="cuda", requires_grad=True)
    h = x * 2
    y = m(h)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_second_derivatives_are_refused():
    m = _module(2, 6, 16, 32)
    x = torch.randn(1, 6, 16, 32, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(m(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_refusals():
    m = _module(2, 6, 16, 32)
    with pytest.raises(TypeError, match="expected dtype"):
        m(torch.zeros(1, 6, 16, 32, device="cuda", dtype=torch.float64))
    with pytest.raises(RuntimeError, match="4 dimensions"):
        m(torch.zeros(6, 16, 32, device="cuda"))
    with pytest.raises(RuntimeError, match="Expected shape"):
        m(torch.zeros(1, 6, 32, 16, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU path"):
        m(torch.zeros(1, 6, 16, 32))
    with pytest.raises(RuntimeError, match="parameters on cpu"):
        m.cpu()(torch.zeros(1, 6, 16, 32, device="cuda"))
    m = m.cuda().double()
    with pytest.raises(TypeError, match="weight and bias"):
        m(torch.zeros(1, 6, 16, 32, device="cuda"))


def test_autocast_keeps_the_input_type():
    m = _module(2, 6, 16, 32, activation="gelu")
    x, dy = _inputs((2, 6, 16, 32), torch.bfloat16, "last")
    want = m(x)
    with torch.autocast(device_type="cuda", dtype=torch.bfloat16):
        assert torch.equal(m(x), want) and m(x.float()).dtype == torch.float32


def test_weights_are_those_of_the_quadrature():
    """The weighted mean of a normalised field over the sphere is zero and its mean square one."""
    import torch_harmonics_b200 as th

    for grid in ("equiangular", "legendre-gauss", "lobatto", "equiangular-trapezoidal"):
        m = _module(5, 5, 33, 64, grid=grid, affine=False, eps=0.0)
        y = m(torch.randn(2, 5, 33, 64, device="cuda") * 3 + 1)
        q = th.QuadratureS2((33, 64), grid=grid, normalize=True).cuda()
        area = q(torch.ones(33, 64, device="cuda"))
        assert q(y).abs().max() <= 10 * F and (q(y * y) / area - 1).abs().max() <= 10 * F


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("channels,groups,dtype", [(73, 73, torch.float32), (73, 1, torch.bfloat16), (32, 4, torch.bfloat16)])
def test_full_resolution(channels, groups, dtype, fmt):
    """721 x 1440.  A thread adds up to 2,000 values one after the other here: the mean of that many roundings of either sign
    stays below 4 sqrt(2000) = 179 half steps, which is the 168 of the bound and its other terms."""
    m = _module(groups, channels, 721, 1440, activation="gelu")
    _parameters(m)
    x, dy = _inputs((1, channels, 721, 1440), dtype, fmt)
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_between_spectral_convolutions_in_training(fmt):
    """A network as it is used: convolution, normalisation with activation, convolution; clipping of all gradients, a step.  Gradients against the
    same chain with the normalisation written out."""
    import torch_harmonics_b200 as th

    torch.manual_seed(0)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        with torch.device("cuda"):
            c1, c2 = th.SpectralConvS2((33, 64), (33, 64), 3, 8), th.SpectralConvS2((33, 64), (33, 64), 8, 3)
    n = _module(4, 8, 33, 64, activation="gelu")
    _parameters(n)
    params = [c1.weight, c2.weight, n.weight, n.bias]
    x, t = torch.randn(2, 3, 33, 64, device="cuda"), torch.randn(2, 3, 33, 64, device="cuda")

    def written_out(h):
        B, C, H, W = h.shape
        q = (n.lat_weights / (n.lat_weights.sum() * W * 2)).view(1, 1, 1, H, 1)
        v = h.view(B, 4, 2, H, W)
        v = v - (q * v).sum((2, 3, 4), keepdim=True)
        v = v / torch.sqrt((q * v * v).sum((2, 3, 4), keepdim=True) + n.eps)
        return torch.nn.functional.gelu(v.view(h.shape) * n.weight.view(1, C, 1, 1) + n.bias.view(1, C, 1, 1))

    grads = []
    for norm in (lambda h: n(h.contiguous(memory_format=FORMATS[fmt])), written_out):
        for p in params:
            p.grad = None
        (c2(norm(c1(x))) - t).square().mean().backward()
        grads.append([p.grad.clone() for p in params])
    for a, b in zip(*grads):
        assert (a - b).abs().max() <= 2e-5 * b.abs().max()
    before = [p.detach().clone() for p in params]
    opt = torch.optim.SGD(params, lr=0.1)
    for p, g in zip(params, grads[0]):
        p.grad = g.clone()
    norm = th.clip_grad_norm_(params, 0.01)
    want = math.sqrt(sum(float(g.abs().double().square().sum()) for g in grads[0]))
    assert abs(float(norm) - want) <= 1e-6 * want and want > 0.01
    opt.step()
    moved = math.sqrt(sum(float((p - b).abs().double().square().sum()) for p, b in zip(params, before)))
    assert abs(moved - 0.1 * 0.01) <= 1e-4 * 0.1 * 0.01 + 1e-7


def _random_bf16(shape, seed):
    x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
    return x.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_more_values_than_32_bits_count(fmt):
    """2,180,304,000 values: the last channels, behind 2^31, against a module of those channels alone (every channel its own group)."""
    C, H, W, tail = 2100, 721, 1440, 3
    if fmt == "planes":
        x, dy = _random_bf16((1, C, H, W), 1), _random_bf16((1, C, H, W), 2)
    else:
        x, dy = (_random_bf16((1, H, W, C), i).permute(0, 3, 1, 2) for i in (1, 2))
    m, small = _module(C, C, H, W, activation="silu"), _module(tail, tail, H, W, activation="silu")
    with torch.no_grad():
        m.weight.normal_(1, 0.3)
        m.bias.normal_(0, 0.3)
        small.weight.copy_(m.weight[-tail:])
        small.bias.copy_(m.bias[-tail:])
    y, dx, dw, db = _step(m, x, dy)
    xs, dys = (t[:, -tail:].contiguous() for t in (x, dy))
    _compare([y[:, -tail:], dx[:, -tail:], dw[-tail:], db[-tail:]], *_exact(small, xs, dys))
    assert torch.isfinite(y[:, ::100]).all() and torch.isfinite(dw).all()


def test_copies_after_use():
    import copy
    import pickle

    m = _module(2, 6, 16, 32, activation="gelu")
    x = torch.randn(1, 6, 16, 32, device="cuda")
    want = m(x)
    for n in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert torch.equal(n(x), want)


def test_inside_a_compiled_function():
    """The surroundings may be compiled; the call itself runs as it is."""
    m = _module(2, 6, 16, 32, activation="gelu")
    _parameters(m)
    x = torch.randn(2, 6, 16, 32, device="cuda", requires_grad=True)

    def f(t):
        return m(t * 2.0) + 1.0

    want = f(x)
    (g,) = torch.autograd.grad(want.square().sum(), x)
    got = torch.compile(f, backend="aot_eager")(x)
    (h,) = torch.autograd.grad(got.square().sum(), x)
    assert torch.equal(got, want) and torch.equal(g, h)


def test_replaced_parameters():
    """Parameters with strides, and one value expanded to all channels, whose gradient is the sum of the channels'."""
    m = _module(2, 6, 16, 32, activation="silu")
    m.weight = torch.nn.Parameter(torch.linspace(0.5, 1.5, 12, device="cuda")[::2])
    m.bias = torch.nn.Parameter(torch.linspace(-1, 1, 18, device="cuda")[::3])
    x, dy = _inputs((2, 6, 16, 32), torch.float32, "planes")
    _compare(_step(m, x, dy), *_exact(m, x, dy))
    one = torch.full((1,), 0.75, device="cuda", requires_grad=True)
    y = torch.func.functional_call(m, {"weight": one.expand(6), "bias": m.bias}, (x,))
    (got,) = torch.autograd.grad(y, (one,), dy)
    with torch.no_grad():
        m.weight.fill_(0.75)
    want, tol = _exact(m, x, dy)
    # (six channels' gradients, each a float32 value, and five additions of them: 6 half steps of the sum of the sizes)
    bound = tol[2].sum() + 6 * HALF[torch.float32] * want[2].abs().sum()
    assert (got.double() - want[2].sum()).abs() <= bound
    m.weight = torch.nn.Parameter(torch.ones(5, device="cuda"))
    with pytest.raises(RuntimeError, match="of shape"):
        m(x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("rows", ["first", "last", "all_but_one", "every_other"])
def test_rows_of_weight_zero(rows, fmt, dtype):
    """Rows that do not count: what they hold, far out here, changes no statistics; they are normalised like the others."""
    m = _module(2, 6, 20, 48, activation="gelu")
    _parameters(m)
    none = {"first": slice(0, 13), "last": slice(11, 20), "all_but_one": slice(0, 19), "every_other": slice(0, 20, 2)}[rows]
    m.lat_weights[none] = 0.0
    x, dy = _inputs((2, 6, 20, 48), dtype, fmt)
    x[:, :, none] += 3
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype,level", [(torch.float32, 101376.0), (torch.bfloat16, 101376.0), (torch.float16, 60000.0), (torch.float16, 1000.0)], ids=["f32", "bf16", "f16", "f16_low"])
def test_constant_fields_give_the_shift_in_every_type(dtype, level, fmt):
    """A constant field has the variance 0: r = eps^(-1/2) multiplies what is left of x - mean, which has to be nothing at all."""
    m = _module(2, 6, 19, 37, affine=True)
    _parameters(m)
    x = torch.full((2, 6, 19, 37), level, device="cuda", dtype=dtype).contiguous(memory_format=FORMATS[fmt])
    _, dy = _inputs((2, 6, 19, 37), dtype, fmt)
    got = _step(m, x, dy)
    assert torch.equal(got[0], m.bias.to(dtype).view(1, 6, 1, 1).expand_as(got[0]))
    _compare(got, *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("dtype,level,step", [(torch.bfloat16, 101376.0, 512.0), (torch.float16, 60000.0, 32.0), (torch.float16, 1000.0, 0.5)], ids=["bf16", "f16", "f16_low"])
def test_one_step_at_one_point(dtype, level, step, act, fmt):
    """Fields that are constant but for the smallest possible step of their type at one of 20,200 points."""
    m = _module(6, 6, 101, 200, activation=act, grid="legendre-gauss")
    _parameters(m)
    x = torch.full((1, 6, 101, 200), level, device="cuda", dtype=dtype)
    x[:, :, 33, 77] += step
    x = x.contiguous(memory_format=FORMATS[fmt])
    _, dy = _inputs((1, 6, 101, 200), dtype, fmt)
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype,level", [(torch.bfloat16, 1.0e3), (torch.float16, 1.0e3), (torch.float16, 3.0e4)], ids=["bf16", "f16", "f16_high"])
def test_level_far_above_spread_in_16_bits(dtype, level, fmt):
    """As with float32 above: the inputs, here a few steps of the type apart, are what is normalised, so the bound is the same."""
    m = _module(2, 6, 61, 120, activation="gelu")
    _parameters(m)
    x, dy = _inputs((2, 6, 61, 120), dtype, fmt, level=level)
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_tail_of_gelu_relative_to_itself(dtype, fmt):
    """gelu of z between -13 and 0, where it falls to 1e-37, against itself rather than against 1.

    z carries the error t = F (1 + |xh w| + |b|) of float32 above.  The logarithmic slope of z Phi(z) is 1 / z + phi(z) / Phi(z), and for z = -a the second
    term lies below (a + sqrt(a^2 + 4)) / 2 <= a + 1 (Mills' ratio), so it is at most |z| + 1 + 1 / |z|.  e^(-z^2 / 2) has an argument of three
    roundings (1.5 z^2 x 2^-24) and an error of 2^-22 of its own, the rest of the product is ten roundings or so: 2^-21 (1 + z^2) together.  The fit is off by
    1.3e-7 (2^-22) before float32 and by 2.9e-5 (2^-15) before 16 bits."""
    m = _module(4, 8, 91, 180, activation="gelu")
    with torch.no_grad():
        m.weight.fill_(2.0)
        m.bias.copy_(torch.linspace(-6, -1, 8))
    x, dy = _inputs((2, 8, 91, 180), dtype, fmt)
    (e, *_), (t, *_) = _exact(m, x, dy)
    m.activation = None
    z = _exact(m, x, dy)[0][0]
    m.activation = "gelu"
    got = m(x).double()
    fit = {torch.float32: 2.0**-22, torch.bfloat16: 2.0**-15, torch.float16: 2.0**-15}[dtype]
    bound = (HALF[dtype] + t * (z.abs() + 1 + 1 / z.abs()) + 2.0**-21 * (1 + z * z) + fit) * e.abs() + TINY[dtype]
    low = (z < -1e-3) & (z > -13.0)
    assert low.sum() > 100_000
    d = ((got - e).abs() / bound)[low]
    assert (d <= 1).all(), f"{float(d.max()):.2f} times the bound"


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("far,rows,channels", [(1.0e4, 1, 73), (1.0e3, 2, 73), (1.0e4, 1, 3), (1.0e5, 1, 32)])
def test_first_rows_far_out(far, rows, channels, fmt):
    """The rows at the pole, a millionth of the weight, are far out (a missing value's mark) and are the first part of the sums, whose mean the others are joined about."""
    m = _module(1, channels, 721, 1440)
    x, dy = _inputs((1, channels, 721, 1440), torch.float32, fmt)
    x[:, :, :rows] += far
    _compare(_step(m, x, dy), *_exact(m, x, dy))


FAR = {"level": (1.0e5, 0.0), "fill": (0.0, 1.0e4), "level_and_fill": (1.0e4, -3.0e4)}


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("rows", ["first", "last", "middle", "every_other"])
@pytest.mark.parametrize("far", list(FAR))
def test_rows_of_weight_zero_in_fields_of_many_chunks(far, rows, fmt):
    """Rows that do not count are whole parts of the sums here (a field is summed in hundreds of parts), the first of them too, and what they hold is far from
    the rest, whose level may be far above its spread.  The bound is that of float32 above: relative to |xh|, so that of the counted rows is tight."""
    level, fill = FAR[far]
    m = _module(8, 32, 256, 512, activation="silu")
    _parameters(m)
    none = {"first": slice(0, 30), "last": slice(226, 256), "middle": slice(100, 150), "every_other": slice(0, 256, 2)}[rows]
    m.lat_weights[none] = 0.0
    x, dy = _inputs((1, 32, 256, 512), torch.float32, fmt, level=level)
    x[:, :, none] += fill
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [slice(0, 1), slice(0, 13), slice(11, 20), slice(0, 19), slice(0, 20, 2), slice(1, 20)], ids=str)
def test_far_values_in_rows_of_weight_zero(rows, dtype, fmt):
    """The same inside one part of the sums: vectors of a thread that do not count come before those that do, and lie across the ends of rows."""
    m = _module(2, 6, 20, 45)
    _parameters(m)
    m.lat_weights[rows] = 0.0
    x, dy = _inputs((2, 6, 20, 45), dtype, fmt)
    x[:, :, rows] += 1.0e4
    _compare(_step(m, x, dy), *_exact(m, x, dy))


def test_replaced_latitude_weights():
    """Weights with strides are read as they are laid out, others are refused, and a change between forward and backward is noticed."""
    m = _module(2, 6, 16, 32)
    x, dy = _inputs((2, 6, 16, 32), torch.float32, "planes")
    m.lat_weights = torch.linspace(0.5, 2.0, 32, device="cuda")[::2]
    _compare(_step(m, x, dy), *_exact(m, x, dy))
    m.lat_weights = torch.full((1,), 3.0, device="cuda").expand(16)
    _compare(_step(m, x, dy), *_exact(m, x, dy))
    m.lat_weights = torch.ones(15, device="cuda")
    with pytest.raises(RuntimeError, match="of shape"):
        m(x)
    m.lat_weights = torch.ones(16, device="cuda")
    y = m(x)
    m.lat_weights[0] = 2.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("fmt", ["planes", "last"])
def test_parameters_with_a_lazy_minus_sign(fmt):
    """A single channel: a view that is contiguous whatever its stride."""
    m = _module(1, 1, 16, 32)
    w, b = (torch.view_as_complex(torch.tensor([[0.5, v]], device="cuda")).conj().imag for v in (1.5, -0.25))
    assert w.is_neg() and w.is_contiguous()
    x, dy = _inputs((2, 1, 16, 32), torch.float32, fmt)
    with torch.no_grad():
        got = torch.func.functional_call(m, {"weight": w, "bias": b}, (x,))
        m.weight.fill_(-1.5)
        m.bias.fill_(0.25)
        assert torch.equal(got, m(x))


def test_lazy_minus_sign_keeps_the_layout():
    m = _module(2, 6, 16, 32)
    x = torch.randn(2, 6, 16, 32, device="cuda").contiguous(memory_format=torch.channels_last)
    n = torch._neg_view(x)
    assert n.is_neg() and n.is_contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        y = m(n)
    assert y.is_contiguous(memory_format=torch.channels_last) and torch.equal(y, m(-x))


@pytest.mark.parametrize("fmt", ["planes", "last", "strided"])
@pytest.mark.parametrize("affine,weighted", [(True, True), (False, True), (True, False)])
def test_traces_into_one_graph(affine, weighted, fmt):
    """Between transforms under torch.compile(fullgraph=True): the same values and gradients as eager, with and without parameters and weights."""
    import torch_harmonics_b200 as th
    from torch_harmonics_b200.normalization import _group_norm, _group_norm_backward

    torch._dynamo.reset()  # (one code object for all cases: its compilations are counted together)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        sht, isht = th.RealSHT(33, 64, grid="equiangular").cuda(), th.InverseRealSHT(33, 64, grid="equiangular").cuda()
    m = _module(2, 6, 33, 64, activation="gelu", affine=affine, weighted=weighted)
    _parameters(m)
    x = torch.randn(2, 6, 33, 64, device="cuda")
    leaves = [x.requires_grad_(True), *m.parameters()]

    def f(t):
        t = isht(sht(t)) * 2
        t = t.contiguous(memory_format=torch.channels_last) if fmt == "last" else torch.cat([t, t], -1)[..., 1:65] if fmt == "strided" else t
        return isht(sht(m(t).contiguous())).square()

    want = f(x)
    grads = torch.autograd.grad(want.sum(), leaves)
    got = torch.compile(f, fullgraph=True, backend="aot_eager")(x)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got.sum(), leaves), grads))
    with torch.no_grad():
        assert torch.equal(torch.compile(f, fullgraph=True, backend="aot_eager")(x), want)
    t = x.detach()
    t = t.contiguous(memory_format=torch.channels_last) if fmt == "last" else torch.cat([t, t], -1)[..., 1:65] if fmt == "strided" else t
    how = (m.weight, m.bias, m.lat_weights, 2, m.eps, "gelu")
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(_group_norm, (t.clone().requires_grad_(True), *how), test_utils=checks)
    y, stats = _group_norm(t, *how)
    assert torch.equal(y, m(t)) and y.stride() == m(t).stride()
    torch.library.opcheck(_group_norm_backward, (torch.randn_like(y), t, *how[:3], stats, *how[3:], [True, affine, False]), test_utils=checks[:2])


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape", [(1, 16, 4, 721, 1440), (2, 32, 8, 256, 512)], ids=lambda s: "x".join(map(str, s)))
def test_errors_in_the_mean_square(shape, act, fmt):
    """float32, where the bound for single values above leaves room for several bits: root-mean-square errors relative to the results'.

    A value of z has three roundings and the errors of m and r, four more at most: 7 x 2^-24.  Activations and slopes add a fit and two approximate
    instructions, 2^-22 each: 7 x 2^-24 + 3 x 2^-22 = 1.2 x 2^-20, of single values, whose mean square is a third of it (uniform): 2^-20 is left for y and dx.
    Sums over a channel of terms of either sign grow like their errors, with n terms by sqrt(n).  To them add the roundings of a thread's running sum: of 2,000
    terms, sqrt(2000) x 0.2 x 2^-24 = 2^-20.8 of its own size.  2^-19 for dweight and dbias."""
    B, C, G, H, W = shape
    m = _module(G, C, H, W, activation=act)
    _parameters(m)
    x, dy = _inputs((B, C, H, W), torch.float32, fmt)
    for name, o, e, bound in zip(("y", "dx", "dweight", "dbias"), _step(m, x, dy), _exact(m, x, dy)[0], (2.0**-20, 2.0**-20, 2.0**-19, 2.0**-19)):
        off = float((o.double() - e).norm() / e.norm())
        assert off <= bound, f"{name}: {off:.2e}"


# channels, groups, nlat, nlon: one or a few vectors a thread, rows shorter than a vector, numbers of channels that do and do not divide a warp
FAR_SHAPES = [(115, 23, 15, 31), (16, 4, 25, 51), (3, 3, 30, 1), (38, 38, 24, 49), (63, 21, 50, 72), (184, 23, 14, 28), (6, 3, 7, 3), (32, 2, 17, 36), (4, 4, 6, 12)]


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype,level", [(torch.float32, 0.0), (torch.float32, 3.0e4), (torch.float16, 1.0e3)], ids=["f32", "f32_high", "f16"])
@pytest.mark.parametrize("where", ["first", "pole", "last", "middle"])
@pytest.mark.parametrize("shape", FAR_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_one_point_far_out_in_small_fields(shape, where, dtype, level, fmt):
    """A value of 3,000 spreads that may be all that a thread, a column or a channel's first slot has to begin with, at a pole with a hundredth of the others' weight or
    less.  The bound is that of float32 above."""
    C, G, H, W = shape
    m = _module(G, C, H, W, activation="silu")
    _parameters(m)
    x, dy = _inputs((2, C, H, W), dtype, fmt, level=level)
    i, j = {"first": (0, 0), "pole": (0, W // 2), "last": (H - 1, W - 1), "middle": (H // 2, W // 3)}[where]
    x[:, :, i, j] += 3.0e3
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["f32", "f16"])
@pytest.mark.parametrize("shape", FAR_SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_rows_of_very_different_weight(shape, dtype, fmt):
    """Weights between 1e-6 and 1, neighbours too, with a value far out in the lightest row."""
    C, G, H, W = shape
    m = _module(G, C, H, W, activation="gelu")
    _parameters(m)
    m.lat_weights[:] = torch.exp(-14 * torch.rand(H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(H)))
    x, dy = _inputs((2, C, H, W), dtype, fmt, level=10.0)
    x[:, :, int(m.lat_weights.argmin()), W // 2] += 3.0e3
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [slice(0, 9), slice(5, 20), slice(0, 20, 2)], ids=str)
def test_fill_values_in_rows_of_weight_zero(rows, dtype, fmt):
    """The largest fill value in use (9.97e36), where the gradient is zero: it reaches neither the statistics nor a gradient."""
    m = _module(2, 6, 20, 45, activation="silu")
    _parameters(m)
    m.lat_weights[rows] = 0.0
    x, dy = _inputs((2, 6, 20, 45), dtype, fmt)
    x[:, :, rows] = 9.96921e36
    dy[:, :, rows] = 0.0
    _compare(_step(m, x, dy), *_exact(m, x, dy))


@pytest.mark.parametrize("fmt", ["planes", "last"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nlon", [541, 1080, 2160])
@pytest.mark.parametrize("column", [5, 400])
def test_heavy_rows_after_light_ones(column, nlon, dtype, fmt):
    """The same in fields of many vectors a thread: every other row weighs a millionth and has a value far out, the next row follows at any of a thread's rounds."""
    m = _module(2, 4, 90, nlon, activation="silu")
    m.lat_weights[0::2] = 1.0e-6
    m.lat_weights[1::2] = 1.0
    x, dy = _inputs((1, 4, 90, nlon), dtype, fmt)
    x[:, :, 0::2, column] += 1.0e7
    _compare(_step(m, x, dy), *_exact(m, x, dy))
