"""Plain 64-bit forms of the layer operators on the CPU, and how far a right implementation may be from them.

u = half a step of a type (finfo.eps / 2).  Every bound is a sum over the roundings that the operators' documentation allows: sums and epilogues in
fp32 (fp64 for fp64), dz rounded to the element type, act' kept in fp16 for bf16, in fp32 for fp16, one rounding of each output."""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def wide_of(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def smallest(dtype):
    """Half a step below the normal numbers: what a rounding costs there."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def f64(t):
    return None if t is None else t.detach().cpu().double()


def activate(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "tanh":
        return torch.tanh(z), 1 / torch.cosh(z.clamp(-300, 300)) ** 2
    if act == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    gate = torch.sigmoid(z)
    return z * gate, gate * (1 + z * (1 - gate))


def product_error(p, q, depth, u):
    """A sum of `depth` products, each addition off by at most one step (2 u: the matrix pipe need not round to nearest)."""
    return (depth + 8) * 2 * u * (p.abs() @ q.abs())


def dense(x, kernel, bias, residual, act, scale, dy, dtype):
    """{name: (value, bound)} of y, slope, dx, dkernel, dbias."""
    kept = {torch.bfloat16: torch.float16, torch.float16: torch.float32}.get(dtype, dtype)
    u, uw, us = half_step(dtype), half_step(wide_of(dtype)), half_step(kept)
    tiny, tiny_s = smallest(dtype), smallest(kept)
    x, kernel, bias, residual, dy = map(f64, (x, kernel, bias, residual, dy))
    k, n, rows = kernel.shape[0], kernel.shape[1], x.shape[0]
    z = x @ kernel + (bias if bias is not None else 0)
    ez = product_error(x, kernel, k, uw) + (2 * uw * (z.abs() + bias.abs()) if bias is not None else 0)
    a, slope = activate(z, act)
    ea = 1.13 * ez + (0 if act == "none" else 16 * uw * (a.abs() + (1 if act == "tanh" else z.abs())))   # |act'| <= 1.13; the functions to 16 half steps
    y = scale * a + (residual if residual is not None else 0)
    ey = abs(scale) * (ea + 2 * uw * a.abs()) + 2 * uw * y.abs() + u * (y.abs() + abs(scale) * ea) + tiny
    out = {"y": (y, ey)}
    eslope = (0 if act == "none" else 0.8 * ez + 16 * uw * (1 + z.abs() * (z.abs() < 8))) + us * slope.abs() + tiny_s      # |act''| <= 0.8
    eslope = eslope if act != "none" else torch.zeros_like(z)
    out["slope"] = (slope, eslope)
    if dy is None:
        return out
    dz = scale * slope * dy
    wide_dz = abs(scale) * dy.abs() * eslope + 3 * uw * dz.abs()
    edz = wide_dz + u * (dz.abs() + wide_dz) + tiny
    if act == "none" and scale == 1:
        edz, wide_dz = torch.zeros_like(dz), torch.zeros_like(dz)
    dx = dz @ kernel.t()
    edx = edz @ kernel.t().abs() + product_error(dz.abs() + edz, kernel.t(), n, uw)
    dkernel = x.t() @ dz
    edk = x.t().abs() @ edz + product_error(x.t(), dz.abs() + edz, rows, uw)
    dbias = dz.sum(0)
    edb = wide_dz.sum(0) + (rows + 8) * uw * (dz.abs() + wide_dz).sum(0)
    for name, v, e in (("dx", dx, edx), ("dkernel", dkernel, edk), ("dbias", dbias, edb)):
        out[name] = (v, e + u * (v.abs() + e) + tiny)
    return out


def layer_norm(x, weight, bias, eps, dy, dtype, weights):
    """{name: (value, bound)}; sums over a row are trees of at most 80 + cols / 512 additions, over the rows of 128 + rows / 256."""
    u, uw, uo = half_step(dtype), half_step(wide_of(dtype)), half_step(weights)
    x, weight, bias, dy = map(f64, (x, weight, bias, dy))
    rows, cols = x.shape
    depth, depth_rows = 80 + cols / 512, 128 + rows / 256
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = d * rstd
    emean = depth * uw * x.abs().mean(1, keepdim=True) + 2 * uw * mean.abs()
    ed = uw * d.abs() + emean
    evar = 2 * (ed * d.abs()).mean(1, keepdim=True) + (ed * ed).mean(1, keepdim=True) + (depth + 4) * uw * var
    erstd = rstd * (0.5 * evar / (var + eps).clamp(min=1e-300) + 6 * uw)
    eh = ed * rstd + d.abs() * erstd + ed * erstd + 2 * uw * h.abs()
    w, b = weight if weight is not None else torch.ones(cols, dtype=torch.float64), bias if bias is not None else torch.zeros(cols, dtype=torch.float64)
    y = h * w + b
    ey = eh * w.abs() + 2 * uw * ((h * w).abs() + y.abs())
    out = {"y": (y, ey + u * (y.abs() + ey) + smallest(dtype)), "mean": (mean[:, 0], emean[:, 0] * 1.01 + smallest(wide_of(dtype))), "rstd": (rstd[:, 0], erstd[:, 0] * 1.01)}
    if dy is None:
        return out
    g = dy * w
    c1, c2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    ec1 = (depth + 4) * uw * g.abs().mean(1, keepdim=True)
    ec2 = (g.abs() * eh).mean(1, keepdim=True) + (depth + 6) * uw * (g * h).abs().mean(1, keepdim=True)
    inner = g - c1 - h * c2
    einner = uw * g.abs() + ec1 + h.abs() * ec2 + eh * c2.abs() + eh * ec2 + 4 * uw * (g.abs() + c1.abs() + (h * c2).abs())
    dx = rstd * inner
    edx = rstd * einner + erstd * (inner.abs() + einner) + 2 * uw * dx.abs()
    out["dx"] = (dx, edx + u * (dx.abs() + edx) + smallest(dtype))
    dweight, dbias = (dy * h).sum(0), dy.sum(0)
    edw = (dy.abs() * eh).sum(0) + (depth_rows + 4) * uw * (dy * h).abs().sum(0)
    edb = depth_rows * uw * dy.abs().sum(0)
    for name, v, e in (("dweight", dweight, edw), ("dbias", dbias, edb)):
        out[name] = (v, e + uo * (v.abs() + e) + smallest(weights))
    return out


def agrees(got, want, name):
    value, bound = want
    got = f64(got).reshape(value.shape)
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    excess = (got - value).abs() - bound
    worst = int(excess.argmax()) if excess.numel() else 0
    assert excess.numel() == 0 or float(excess.max()) <= 0, \
        f"{name}: {float(got.reshape(-1)[worst])!r} for {float(value.reshape(-1)[worst])!r}, {float(bound.reshape(-1)[worst]):.3g} allowed"


def near(got, want, steps, dtype, name):
    """The 2-norm of the error within `steps` half steps of the result's: independent roundings of random data add up like that, a term left out of a
    sum of fewer than 1 / (steps u)^2 terms does not."""
    value = want[0]
    got = f64(got).reshape(value.shape)
    size = float(torch.linalg.norm(value))
    if size > 0:
        off = float(torch.linalg.norm(got - value)) / size
        assert off <= steps * half_step(dtype), f"{name}: off by {off:.3g}, {steps * half_step(dtype):.3g} allowed"
