"""GPU tests of the gradient norm and clipping against float64.

Tolerances.  The sums are float64 and the norm is rounded once, with a square root: 2^-23 relative.  The factor is a float32 quotient of float32
values (norm, sum with 1e-6, quotient: 4 x 2^-24 relative), and a clipped value is rounded once more to its type."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0**-24, torch.complex64: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 1e-44, torch.complex64: 1e-44, torch.bfloat16: 5e-41, torch.float16: 2.0**-25}


def _wide(t):
    return t.to(torch.complex128 if t.is_complex() else torch.float64)


def _norm(ts, kind):
    vals = [float(torch.linalg.vector_norm(_wide(t), ord=kind)) for t in ts if t.numel()]
    return (max(vals, default=0.0)) if kind == math.inf else math.sqrt(sum(v * v for v in vals))


def _tensors(spec, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for shape, dt in spec:
        if dt.is_complex:
            out.append(torch.view_as_complex(torch.randn(*shape, 2, device="cuda", generator=gen) * scale))
        else:
            out.append((torch.randn(shape, device="cuda", generator=gen) * scale).to(dt))
    return out


def _clipped_right(new, old, norm64, max_norm):
    f = min(1.0, max_norm / (norm64 + 1e-6))
    for n, o in zip(new, old):
        assert n.dtype == o.dtype and n.shape == o.shape
        e = torch.view_as_real(_wide(o) * f) if o.is_complex() else _wide(o) * f
        v = torch.view_as_real(_wide(n.resolve_conj())) if n.is_complex() else _wide(n)
        assert ((v - e).abs() <= (HALF[o.dtype] + 2.0**-21) * e.abs() + TINY[o.dtype]).all()


F32, BF16, F16, C64 = torch.float32, torch.bfloat16, torch.float16, torch.complex64
SPECS = {
    "one": [((1,), F32)],
    "scalar": [((), F32)],
    "odd": [((7,), F32), ((13, 3), BF16), ((1, 5, 2), F16), ((3, 3), C64), ((8191,), F32), ((8193,), BF16)],
    "mixed": [((1, 16, 16, 33), C64), ((64, 32), BF16), ((64,), BF16), ((32,), F32), ((32, 64), F16)],
    "empty_inside": [((0,), F32), ((5,), F32), ((3, 0), BF16), ((4,), C64)],
    "long": [(((1 << 21) + 3,), F32), (((1 << 20) + 1,), BF16), ((1, 33, 65, 129), C64)],
    "many": [((n % 37 + 1, n % 5 + 1), [F32, BF16, F16, C64][n % 4]) for n in range(2000)],
}


@pytest.mark.parametrize("kind", [2.0, math.inf], ids=["l2", "inf"])
@pytest.mark.parametrize("name", list(SPECS))
def test_norm(name, kind):
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS[name])
    n = th.global_norm(ts, kind)
    assert n.dtype == torch.float32 and n.shape == () and n.is_cuda
    want = _norm(ts, kind)
    assert abs(float(n) - want) <= 2.0**-22 * want


@pytest.mark.parametrize("ratio", [0.5, 3.0])
@pytest.mark.parametrize("kind", [2.0, math.inf], ids=["l2", "inf"])
@pytest.mark.parametrize("name", list(SPECS))
def test_clipping(name, kind, ratio):
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS[name], seed=2, scale=0.1)
    old = [t.clone() for t in ts]
    want = _norm(ts, kind)
    limit = want / ratio
    new, n = th.clip_by_global_norm(ts, limit, kind)
    assert isinstance(new, tuple) and abs(float(n) - want) <= 2.0**-22 * want
    assert all(torch.equal(a, b) for a, b in zip(ts, old))
    assert all(a.data_ptr() != b.data_ptr() for a, b in zip(new, ts) if a.numel())
    _clipped_right(new, old, want, limit)
    params = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, t in zip(params, ts):
        p.grad = t
    n2 = th.clip_grad_norm_(params + [torch.nn.Parameter(torch.zeros(3, device="cuda"))], limit, kind)
    assert torch.equal(n, n2)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, new))
    if ratio < 1:
        assert all(torch.equal(p.grad, b) for p, b in zip(params, old))


def test_clipping_with_a_given_norm():
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS["mixed"])
    params = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, t in zip(params, ts):
        p.grad = t.clone()
    given = torch.tensor(50.0, device="cuda", dtype=torch.float64)  # e.g. joined over ranks: larger than this rank's own
    assert th.clip_grads_with_norm_(params, 2.0, given) is None
    _clipped_right([p.grad for p in params], ts, 50.0, 2.0)
    with pytest.raises(RuntimeError, match="total_norm"):
        th.clip_grads_with_norm_(params, 2.0, torch.tensor(50.0))
    with pytest.raises(RuntimeError, match="total_norm"):
        th.clip_grads_with_norm_(params, 2.0, torch.ones(2, device="cuda"))


@pytest.mark.parametrize("scale", [1e-30, 1e25])
def test_squares_outside_the_range_of_float32(scale):
    import torch_harmonics_b200 as th

    for dt in (F32, C64, BF16):
        ts = _tensors([((1000, 7), dt)], scale=scale)
        want = _norm(ts, 2.0)
        assert abs(float(th.global_norm(ts)) - want) <= 2.0**-22 * want
        want = _norm(ts, math.inf)
        assert abs(float(th.global_norm(ts, math.inf)) - want) <= 2.0**-22 * want


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("dt", [F32, BF16, F16, C64], ids=["f32", "bf16", "f16", "c64"])
def test_bucket_views_at_any_alignment(dt, offset):
    """Views of one flat bucket; what lies between and around them stays as it was."""
    import torch_harmonics_b200 as th

    (flat,) = _tensors([((200_001,), dt)], seed=4)
    before = flat.clone()
    cuts = [(offset, 7), (offset + 8, 1), (offset + 9, 66_001), (offset + 66_013, 100_003)]
    params = []
    for at, n in cuts:
        p = torch.nn.Parameter(torch.zeros(n, dtype=dt, device="cuda"))
        p.grad = flat[at : at + n]
        params.append(p)
    old = [before[at : at + n] for at, n in cuts]
    want = _norm(old, 2.0)
    n = th.clip_grad_norm_(params, want / 2)
    assert abs(float(n) - want) <= 2.0**-22 * want
    _clipped_right([p.grad for p in params], old, want, want / 2)
    keep = torch.ones(200_001, dtype=torch.bool, device="cuda")
    for at, k in cuts:
        keep[at : at + k] = False
    assert torch.equal(flat[keep], before[keep])


def test_orders_of_axes_slices_and_lazy_conjugates():
    import torch_harmonics_b200 as th

    a = _tensors([((6, 7, 8), F32)])[0].permute(2, 0, 1)  # gapless, axes in another order
    b = _tensors([((10, 12), BF16)], seed=1)[0][1:7, 2:9]  # a slice: clipped in a copy
    c = _tensors([((4, 5), C64)], seed=2)[0].conj()
    d = _tensors([((4, 5), C64)], seed=3)[0].conj().imag
    ts = [a, b, c, d]
    want = _norm([t.resolve_conj().resolve_neg() for t in ts], 2.0)
    new, n = th.clip_by_global_norm(ts, want / 3)
    assert abs(float(n) - want) <= 2.0**-22 * want
    _clipped_right(new, [t.resolve_conj().resolve_neg() for t in ts], want, want / 3)
    assert new[0].stride() == a.stride()
    base = _tensors([((10, 12), BF16)], seed=1)[0]
    p = torch.nn.Parameter(torch.zeros(6, 7, dtype=BF16, device="cuda"))
    p.grad = base[1:7, 2:9]
    old = base.clone()
    th.clip_grad_norm_(p, 0.5)  # a single parameter
    _clipped_right([p.grad], [old[1:7, 2:9]], _norm([old[1:7, 2:9]], 2.0), 0.5)
    base[1:7, 2:9] = old[1:7, 2:9]
    assert torch.equal(base, old)


@pytest.mark.parametrize("kind", [2.0, math.inf], ids=["l2", "inf"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_norms_that_are_not_finite(bad, kind):
    import torch_harmonics_b200 as th

    for dt in (F32, C64, BF16):
        ts = _tensors([((1000,), dt), ((77,), F32)])
        ts[0][3] = bad
        old = [t.clone() for t in ts]
        new, n = th.clip_by_global_norm(ts, 1.0, kind)
        ref_n = torch.stack([torch.linalg.vector_norm(t, ord=kind).float() for t in old])
        assert torch.isnan(n) if math.isnan(bad) else float(n) == math.inf
        f = 1.0 / (n + 1e-6)
        assert all(torch.equal(torch.isnan(a), torch.isnan(o * f)) for a, o in zip(new, old)) and ref_n.shape == (2,)
        p = torch.nn.Parameter(torch.zeros_like(ts[0]))
        p.grad = ts[0]
        with pytest.raises(RuntimeError, match="non-finite"):
            th.clip_grad_norm_(p, 1.0, kind, error_if_nonfinite=True)
        assert torch.equal(torch.isnan(p.grad), torch.isnan(old[0]))
        with pytest.raises(RuntimeError, match="non-finite"):
            th.clip_by_global_norm(ts, 1.0, kind, error_if_nonfinite=True)


def test_error_if_nonfinite_clips_the_same():
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS["mixed"])
    a, n = th.clip_by_global_norm(ts, 1.0)
    b, k = th.clip_by_global_norm(ts, 1.0, error_if_nonfinite=True)
    assert torch.equal(n, k) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_zero_gradients_and_zero_limit():
    import torch_harmonics_b200 as th

    z = torch.zeros(1000, device="cuda")
    new, n = th.clip_by_global_norm([z], 1.0)
    assert float(n) == 0 and torch.equal(new[0], z)
    new, _ = th.clip_by_global_norm([z + 1], 0.0)
    assert torch.equal(new[0], z)
    new, _ = th.clip_by_global_norm([z + 1], math.inf)
    assert torch.equal(new[0], z + 1)


def test_versions_and_saved_tensors():
    import torch_harmonics_b200 as th

    p = torch.nn.Parameter(torch.ones(10, device="cuda"))
    p.grad = torch.ones(10, device="cuda")
    v = p.grad._version
    th.clip_grad_norm_(p, 1.0)
    assert p.grad._version > v


def test_captured_and_replayed():
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS["mixed"], scale=0.1)
    th.clip_by_global_norm(ts, 1.0)
    torch.cuda.synchronize()
    graphs, res = [], []
    for _ in range(2):  # two graphs that share a pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            res.append(th.clip_by_global_norm(ts, 1.0))
        graphs.append(g)
    for seed in (7, 8):
        for t, s in zip(ts, _tensors(SPECS["mixed"], seed=seed, scale=0.1)):
            t.copy_(s)
        want, n = th.clip_by_global_norm(ts, 1.0)
        for g, (new, k) in zip(graphs, res):
            g.replay()
            assert torch.equal(k, n) and all(torch.equal(a, b) for a, b in zip(new, want))


def test_on_several_streams_at_once():
    import torch_harmonics_b200 as th

    ts = _tensors(SPECS["long"])
    want, n = th.clip_by_global_norm(ts, 1.0)
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs.append(th.clip_by_global_norm(ts, 1.0))
    torch.cuda.synchronize()
    for new, k in outs:
        assert torch.equal(k, n) and all(torch.equal(a, b) for a, b in zip(new, want))


def test_refusals():
    import torch_harmonics_b200 as th

    g = torch.ones(10, device="cuda")
    p, q = torch.nn.Parameter(g.clone()), torch.nn.Parameter(g.clone())
    p.grad = q.grad = g
    with pytest.raises(RuntimeError, match="share memory"):
        th.clip_grad_norm_([p, q], 1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        th.clip_grad_norm_([p, p], 1.0)
    assert torch.equal(g, torch.ones(10, device="cuda"))
    assert abs(float(th.global_norm([g, g])) - math.sqrt(20)) <= 1e-6  # (a norm may count a tensor twice)
    with pytest.raises(RuntimeError, match="no CPU path"):
        th.global_norm([g, torch.ones(3)])
    with pytest.raises(TypeError, match="float64"):
        th.global_norm([g.double()])
    with pytest.raises(TypeError, match="dense"):
        th.global_norm([g.to_sparse()])


def test_slices_of_one_tensor():
    """Columns of one tensor, neither of them gapless: clipped apart from one another, refused where they share a column."""
    import torch_harmonics_b200 as th

    base = _tensors([((6, 10), F32)])[0]
    old = base.clone()
    ps = [torch.nn.Parameter(torch.zeros(6, n, device="cuda")) for n in (4, 6)]
    ps[0].grad, ps[1].grad = base[:, :4], base[:, 4:]
    th.clip_grad_norm_(ps, 0.5)
    _clipped_right([base], [old], _norm([old], 2.0), 0.5)
    ps[1].grad = base[:, 3:9]
    old = base.clone()
    for clip in (lambda: th.clip_grad_norm_(ps, 0.5), lambda: th.clip_grads_with_norm_(ps, 0.5, torch.tensor(3.0, device="cuda"))):
        with pytest.raises(RuntimeError, match="share memory"):
            clip()
    assert torch.equal(base, old)


def test_expanded_gradients():
    """One value expanded to all entries: counted as often as it is seen, clipped into a new tensor, and refused in place before any gradient is touched."""
    import torch_harmonics_b200 as th

    (a,), one = _tensors([((50,), F32)]), torch.full((1,), 2.0, device="cuda")
    wide = one.expand(30)
    want = _norm([a, wide], 2.0)
    new, n = th.clip_by_global_norm([a, wide], want / 2)
    assert abs(float(n) - want) <= 2.0**-22 * want
    _clipped_right(new, [a, wide], want, want / 2)
    ps = [torch.nn.Parameter(torch.zeros(k, device="cuda")) for k in (50, 30)]
    ps[0].grad, ps[1].grad = a, wide
    old = a.clone()
    for clip in (lambda: th.clip_grad_norm_(ps, want / 2), lambda: th.clip_grads_with_norm_(ps, want / 2, n), lambda: th.clip_grad_norm_(ps, want / 2, error_if_nonfinite=True)):
        with pytest.raises(RuntimeError, match="share memory"):
            clip()
        assert torch.equal(a, old) and float(one) == 2.0


def test_norm_that_is_a_gradient_itself():
    """The norm of a single scalar parameter is its gradient: refused as it stands, taken as a copy."""
    import torch_harmonics_b200 as th

    p = torch.nn.Parameter(torch.zeros((), device="cuda"))
    p.grad = torch.full((), 3.0, device="cuda")
    with pytest.raises(RuntimeError, match="share memory"):
        th.clip_grads_with_norm_(p, 1.0, p.grad)
    assert float(p.grad) == 3.0
    th.clip_grads_with_norm_(p, 1.0, p.grad.clone())
    _clipped_right([p.grad], [torch.full((), 3.0, device="cuda")], 3.0, 1.0)


def test_norm_with_a_lazy_minus_sign():
    import torch_harmonics_b200 as th

    norm = torch.view_as_complex(torch.tensor([0.5, -8.0], device="cuda")).conj().imag  # 8, held as -8
    assert norm.is_neg() and norm.is_contiguous()
    (g,) = _tensors([((100,), F32)])
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = g.clone()
    th.clip_grads_with_norm_(p, 2.0, norm)
    _clipped_right([p.grad], [g], 8.0, 2.0)
