"""Cases, plain forms and exact values of the training-side operators: group normalisation with an activation on fields over the
sphere (``GroupNormS2``), and the global norm of a set of gradients with clipping (``clip_grad_norm_``, ``clip_by_global_norm``).

Group normalisation of x (B, C, nlat, nlon) in G groups of C / G channels, a = latitude weights normalised to mean 1:
    mu = avg(a x), v = avg(a (x - mu)^2) over a group, xh = (x - mu) / sqrt(v + eps), z = weight_c xh + bias_c, y = act(z)
and with g = dy act'(z), h = weight_c g, n = grid points * channels of the group:
    d bias_c = sum g, d weight_c = sum g xh, dx = (h - (a / n) (sum h + xh sum h xh)) / sqrt(v + eps).
Clipping: N = (sum over all tensors and entries |g|^2)^(1/2) or max |g|, factor min(1, max_norm / (N + 1e-6)).
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5


def _gn(name, train, batch, channels, groups, nlat, nlon, dtype, layout, activation, grid):
    return {"name": name, "op": "norm", "train": train, "batch": batch, "channels": channels, "groups": groups, "nlat": nlat, "nlon": nlon,
            "dtype": dtype, "layout": layout, "activation": activation, "grid": grid}


def _clip(name, layers, channels, degrees, dtype, inplace, ratio, norm):
    return {"name": name, "op": "clip", "layers": layers, "channels": channels, "degrees": degrees, "dtype": dtype, "inplace": inplace,
            "ratio": ratio, "norm": norm}


def listed():
    return [
        # a few channels on a 33 x 64 grid, one sample at a time: a rollout of a small surrogate, where the latency of the call counts
        _gn("infer_33x64_c8_fp32", False, 1, 8, 4, 33, 64, "fp32", "contiguous", "gelu", "equiangular"),
        # one sample between pointwise (channels-last) layers at half precision
        _gn("infer_128x256_c32_bf16_cl", False, 1, 32, 8, 128, 256, "bf16", "channels_last", "silu", "legendre-gauss"),
        # 73 fields of the 0.25 degree grid, normalised one by one, straight behind an inverse transform
        _gn("infer_721x1440_c73_fp32", False, 1, 73, 73, 721, 1440, "fp32", "contiguous", "gelu", "equiangular"),
        # training at an odd grid with ragged rows: planes and rows are not multiples of a vector
        _gn("train_129x257_c24_fp16", True, 4, 24, 3, 129, 257, "fp16", "contiguous", "none", "uniform"),
        # training a medium network in float32, channels last
        _gn("train_256x512_c32_fp32_cl", True, 2, 32, 8, 256, 512, "fp32", "channels_last", "gelu", "legendre-gauss"),
        # a wide hidden layer at half resolution under mixed precision
        _gn("train_361x720_c256_bf16_cl", True, 1, 256, 32, 361, 720, "bf16", "channels_last", "gelu", "equiangular"),
        # all 73 fields of a sample normalised together (layer normalisation of the input), an odd number of channels last
        _gn("train_721x1440_c73_bf16_cl", True, 1, 73, 1, 721, 1440, "bf16", "channels_last", "silu", "equiangular"),
        # the largest: a full-resolution hidden layer in float32
        _gn("train_721x1440_c64_fp32", True, 1, 64, 16, 721, 1440, "fp32", "contiguous", "gelu", "equiangular"),
        # a small network of two spectral layers, its norm below the limit (an ordinary step late in training)
        _clip("clip_2x8_small", 2, 8, 32, "fp32", True, 0.5, "2"),
        # 40 pointwise blocks under bf16 training: several hundred small odd tensors, views of one bucket at any alignment
        _clip("clip_40_blocks_bf16", 40, 73, 0, "bf16", True, 0.4, "2"),
        # spectral layers of 73 channels and 720 degrees with bf16 pointwise layers, clipped into new tensors
        _clip("clip_8x73_spectral", 8, 73, 720, "bf16", False, 2.0, "2"),
        # wide spectral layers (256 channels): 1.5 GB of gradients below the limit
        _clip("clip_4x256_spectral", 4, 256, 720, "fp32", True, 0.7, "2"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.7:
        train = rng.random() < 0.6
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        nlat = _log(rng, 17, 721)
        nlon = max(17, 2 * nlat + rng.choice([-2, -1, 0, 0, 0, 1, 6]))
        batch = rng.choice([1, 1, 2, 3, 4])
        most = 60_000_000 // (nlat * nlon)
        while batch > 1 and batch > most:
            batch -= 1
        per = _log(rng, 1, 32)
        groups = _log(rng, 1, 64)
        while per * groups * batch > most and (per > 1 or groups > 1):
            per, groups = max(1, per // 2), max(1, groups - groups // 3 - 1)
        return {"op": "norm", "train": train, "batch": batch, "channels": per * groups, "groups": groups, "nlat": nlat, "nlon": nlon, "dtype": dtype,
                "layout": rng.choice(["channels_last", "channels_last", "contiguous"]), "activation": rng.choice(["gelu", "silu", "none"] if train else ["gelu", "silu", "relu", "none"]),  # (relu's derivative jumps: z next to 0 says nothing)
                "grid": rng.choice(["equiangular", "legendre-gauss", "uniform"])}
    inplace = rng.random() < 0.4
    layers = _log(rng, 1, 40 if inplace else 8)
    channels = _log(rng, 5, 256)
    degrees = rng.choice([0, _log(rng, 9, 720)])
    while layers * channels * channels * (8 * degrees + 16) > 1.3e9:
        layers, channels = max(1, layers - 1), channels - channels // 5
    return {"op": "clip", "layers": layers, "channels": channels, "degrees": degrees, "dtype": rng.choice(["fp32", "bf16", "fp16"]), "inplace": inplace,
            "ratio": round(rng.uniform(0.2, 0.8) if inplace else rng.uniform(1.3, 6.0), 3), "norm": rng.choice(["2", "2", "2", "inf"])}


# ------------------------------------------------------------------------------------------------------------------ inputs

def _lat_weights(nlat, grid):
    """Quadrature weights of the latitude rows, mean 1, float64."""
    if grid == "uniform":
        return np.ones(nlat)
    if grid == "legendre-gauss":
        w = np.polynomial.legendre.leggauss(nlat)[1]
    else:  # Clenshaw-Curtis on nlat equally spaced colatitudes
        n = nlat - 1
        k = np.arange(nlat)
        w = np.ones(nlat)
        for j in range(1, n // 2 + 1):
            w -= (1.0 if 2 * j == n else 2.0) / (4.0 * j * j - 1.0) * np.cos(2.0 * np.pi * j * k / n)
        w *= 2.0 / n
        w[0] *= 0.5
        w[-1] *= 0.5
    return w / w.mean()


def _grad_shapes(case):
    """(shape, dtype) of every gradient of `layers` blocks: a spectral weight, two pointwise products with biases, a norm's scale and shift."""
    c, dt = case["channels"], DTYPES[case["dtype"]]
    out = []
    for i in range(case["layers"]):
        if case["degrees"]:
            out.append(((1, c, c, case["degrees"]), torch.complex64))
        out += [((2 * c, c), dt), ((2 * c,), dt), ((c, 2 * c), dt), ((c,), dt), ((c,), torch.float32), ((c,), torch.float32)]
        if i % 3 == 0:
            out.append(((1, 2 * c + 1, 3), dt))
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, device=dev, generator=gen, dtype=torch.float32)

    if case["op"] == "norm":
        B, C, H, W, dt = case["batch"], case["channels"], case["nlat"], case["nlon"], DTYPES[case["dtype"]]
        fmt = torch.channels_last if case["layout"] == "channels_last" else torch.contiguous_format
        # hidden fields: every channel with its own level and spread, as behind a convolution or a residual sum
        x = randn(B, C, H, W).mul_(torch.exp(0.5 * randn(1, C, 1, 1))).add_(2.0 * randn(B, C, 1, 1))
        st = {"case": case, "x": x.to(dt).contiguous(memory_format=fmt), "weight": 1.0 + 0.3 * randn(C), "bias": 0.3 * randn(C),
              "lat": torch.from_numpy(_lat_weights(H, case["grid"])).to(dev)}
        if case["train"]:
            st["dy"] = randn(B, C, H, W).to(dt).contiguous(memory_format=fmt)
            st["x"].requires_grad_(True)
        if own:
            import torch_harmonics_b200 as th

            act = None if case["activation"] == "none" else case["activation"]
            m = th.GroupNormS2(case["groups"], C, (H, W), grid="equiangular" if case["grid"] == "uniform" else case["grid"], eps=EPS,
                               activation=act, weighted=case["grid"] != "uniform").to(dev)
            with torch.no_grad():
                m.weight.copy_(st["weight"])
                m.bias.copy_(st["bias"])
            st["module"] = m
        return st

    grads, reals = [], 0
    for n, (shape, dt) in enumerate(_grad_shapes(case)):
        s = 1e-3 * math.exp(math.sin(3.0 * n))  # layers differ in the size of their gradients
        if dt.is_complex:
            g = torch.view_as_complex(randn(*shape, 2).mul_(s))
        else:
            g = randn(*shape).mul_(s).to(dt)
        reals += s * s * g.numel() * (2 if dt.is_complex else 1)
        grads.append(g)
    expect = math.sqrt(reals) if case["norm"] == "2" else 6.5 * 2.72e-3
    st = {"case": case, "grads": grads, "max_norm": expect / case["ratio"], "norm_type": 2.0 if case["norm"] == "2" else math.inf}
    if case["inplace"]:
        # one flat bucket for each type with the gradients as views, as data-parallel training keeps them
        st["buckets"], st["grads"] = [], [None] * len(grads)
        for dt in sorted({g.dtype for g in grads}, key=str):
            mine = [n for n, g in enumerate(grads) if g.dtype == dt]
            bucket, at = torch.cat([grads[n].reshape(-1) for n in mine]), 0
            for n in mine:
                st["grads"][n] = bucket[at : at + grads[n].numel()].view(grads[n].shape)
                at += grads[n].numel()
            st["buckets"].append(bucket)
        if own:
            st["params"] = [torch.nn.Parameter(torch.zeros_like(g)) for g in st["grads"]]
            for p, g in zip(st["params"], st["grads"]):
                p.grad = g
    return st


# ------------------------------------------------------------------------------------------------------------- plain forms

def _act(z, kind):
    """act(z) and act'(z) in float32."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if kind == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    cdf = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_norm(st):
    case, x = st["case"], st["x"].detach()
    B, C, H, W = x.shape
    G = case["groups"]
    f64 = torch.float64
    xf = x.float().reshape(B, G, C // G, H, W)
    a = st["lat"].float()[:, None]
    n = float((C // G) * H * W)
    mean = ((xf * a).sum((2, 3, 4), keepdim=True, dtype=f64) / n).float()
    d = xf - mean
    var = ((d * d * a).sum((2, 3, 4), keepdim=True, dtype=f64) / n).float()
    r = 1.0 / torch.sqrt(var + EPS)
    xh = d * r
    w, b = st["weight"].reshape(1, G, C // G, 1, 1), st["bias"].reshape(1, G, C // G, 1, 1)
    y, dact = _act(xh * w + b, case["activation"])
    y = y.reshape(B, C, H, W).to(x.dtype)
    if not case["train"]:
        return y
    g = st["dy"].float().reshape(B, G, C // G, H, W) * dact
    gb = g.sum((0, 3, 4), dtype=f64).float().reshape(C)
    gw = (g * xh).sum((0, 3, 4), dtype=f64).float().reshape(C)
    h = g * w
    s1 = (h.sum((2, 3, 4), keepdim=True, dtype=f64) / n).float()
    s2 = ((h * xh).sum((2, 3, 4), keepdim=True, dtype=f64) / n).float()
    gx = (r * (h - a * (s1 + xh * s2))).reshape(B, C, H, W).to(x.dtype)
    return y, gx, gw, gb


def _plain_clip(st):
    case, grads = st["case"], st["grads"]
    parts = []
    for g in grads:
        f = torch.view_as_real(g) if g.is_complex() else g.float()
        sq = f * f
        if case["norm"] == "2":
            parts.append(sq.sum(dtype=torch.float64))
        else:
            parts.append((sq.sum(-1) if g.is_complex() else sq).max().to(torch.float64))
    parts = torch.stack(parts)
    norm = torch.sqrt(parts.sum() if case["norm"] == "2" else parts.max()).float()
    factor = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    out = [(g * factor) if g.dtype in (torch.float32, torch.complex64) else (g.float() * factor).to(g.dtype) for g in grads]
    if case["inplace"]:
        for g, o in zip(grads, out):
            g.copy_(o)
        out = st["buckets"]
    return [norm] + list(out)


# -------------------------------------------------------------------------------------------------------------------- a pass

def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_norm(state) if case["op"] == "norm" else _plain_clip(state)
    import torch_harmonics_b200 as th

    if case["op"] == "norm":
        m = state["module"]
        if not case["train"]:
            with torch.no_grad():
                return m(state["x"])
        y = m(state["x"])
        gx, gw, gb = torch.autograd.grad(y, (state["x"], m.weight, m.bias), state["dy"])
        return y.detach(), gx, gw, gb
    if case["inplace"]:
        norm = th.clip_grad_norm_(state["params"], state["max_norm"], norm_type=state["norm_type"])
        return [norm] + state["buckets"]
    clipped, norm = th.clip_by_global_norm(state["grads"], state["max_norm"], norm_type=state["norm_type"])
    return [norm] + list(clipped)


def work(case):
    if case["op"] == "norm":
        n = case["batch"] * case["channels"] * case["nlat"] * case["nlon"]
        es = 4 if case["dtype"] == "fp32" else 2
        c = case["channels"]
        # forward: x in, y out; training as well dy in, dx out, and the parameters' gradients
        return {"bytes": (4 if case["train"] else 2) * n * es + (16 if case["train"] else 8) * c, "flops": (40 if case["train"] else 14) * n}
    total, reals = 0, 0
    for shape, dt in _grad_shapes(case):
        n = math.prod(shape)
        total += n * {torch.complex64: 8, torch.float32: 4}.get(dt, 2)
        reals += n * (2 if dt.is_complex else 1)
    # below the limit the gradients stay as they are: they are read once
    below = case["inplace"] and case["ratio"] < 1
    return {"bytes": total if below else 2 * total, "flops": (2 if below else 3) * reals}


# ------------------------------------------------------------------------------------------------------------ exact values

def exact(case, seed):
    """The definitions in float64; the gradients by automatic differentiation."""
    st = prepare(case, seed)
    if case["op"] == "norm":
        x = st["x"].detach().double().requires_grad_(case["train"])
        w = st["weight"].double().requires_grad_(case["train"])
        b = st["bias"].double().requires_grad_(case["train"])
        B, C, H, W = x.shape
        G = case["groups"]
        p = (st["lat"] / st["lat"].sum() / (W * (C // G))).reshape(1, 1, 1, H, 1)
        with torch.set_grad_enabled(bool(case["train"])):
            v = x.reshape(B, G, C // G, H, W)
            mu = torch.sum(p * v, dim=(2, 3, 4), keepdim=True)
            c = v - mu
            sigma = torch.sqrt(torch.sum(p * c.square(), dim=(2, 3, 4), keepdim=True) + EPS)
            z = (c / sigma).reshape(B, C, H, W) * w[:, None, None] + b[:, None, None]
            if case["activation"] == "relu":
                y = z.clamp(min=0)
            elif case["activation"] == "silu":
                y = z * torch.sigmoid(z)
            elif case["activation"] == "gelu":
                y = 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
            else:
                y = z
        if not case["train"]:
            return y
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), st["dy"].double())
        return y.detach(), gx, gw, gb
    two = case["norm"] == "2"
    total = 0.0
    for g in st["grads"]:
        m = torch.linalg.vector_norm(g.to(torch.complex128 if g.is_complex() else torch.float64), ord=2 if two else math.inf).item()
        total = math.hypot(total, m) if two else max(total, m)
    factor = min(1.0, st["max_norm"] / (total + 1e-6))
    out = [torch.tensor(total, dtype=torch.float64)]
    for g in st["buckets"] if case["inplace"] else st["grads"]:
        out.append(g.to(torch.complex128 if g.is_complex() else torch.float64) * factor)
    return out
