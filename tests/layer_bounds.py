"""What linear layers, layer normalisation and the AdamW step give in 64 bits on the CPU, and how far results may be from it: bounds
that follow from the roundings, element by element.

u = 2^-24 is what rounding to a float changes a value by at most, relative to it, v = 2^-8 what rounding to a bfloat16 does (eight
significant bits).  A sum of n terms t_i in some order is off by at most n u sum |t_i|; rounding errors that do not conspire give about sqrt(n) of them, and (2 sqrt(n) + 8) u sum |t_i| is allowed.
"""
import math

import torch

U, V = 2.0 ** -24, 2.0 ** -8
CURVATURE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}   # of the activations at most: 2 phi(0) = 0.798 and 1 / 2


def terms(n):
    return (2 * math.sqrt(n) + 8) * U


def activation(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        p = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def linear(x, w, b, r, dy, act):
    """{name: (value, how far off it may be)} for y, gx, gw and gb, from tensors of the type that the layer runs in."""
    half = x.dtype == torch.bfloat16
    x, w, b, r, dy = (None if t is None else t.detach().double().cpu() for t in (x, w, b, r, dy))
    n, k = w.shape
    rows = x.shape[0]
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b, size + b.abs()
    y, slope = activation(z, act)
    off_z = terms(k) * size
    # |act'| <= 1.13; the activation's own arithmetic is a few units
    off_y = 1.13 * off_z + 16 * U * (y.abs() + z.abs())
    if r is not None:
        y, off_y = y + r, off_y + U * (y + r).abs()
    out = {"y": (y, off_y + (V if half else U) * y.abs())}
    if dy is None:
        return out
    dz = dy * slope
    # in bfloat16 z is kept rounded, and dz is rounded for the products but not for the bias
    off = dy.abs() * (CURVATURE[act] * (off_z + (V * z.abs() if half else 0)) + 24 * U * (1 + z.abs()))
    off_dz = off + (V * dz.abs() * 1.01 if half else 0)
    if act == "none":
        off = off_dz = torch.zeros_like(dz)
    last = V if half else U
    gx, gw, gb = dz @ w, dz.t() @ x, dz.sum(0)
    out["gx"] = gx, off_dz @ w.abs() + terms(n) * (dz.abs() @ w.abs()) + last * gx.abs()
    out["gw"] = gw, off_dz.t() @ x.abs() + terms(rows) * (dz.abs().t() @ x.abs()) + last * gw.abs()
    out["gb"] = gb, off.sum(0) + terms(rows) * dz.abs().sum(0) + last * gb.abs()
    return out


def layer_norm(x, w, b, dy, eps):
    half = x.dtype == torch.bfloat16
    last = V if half else U
    of = w if w is not None else b
    last_w = V if of is not None and of.dtype == torch.bfloat16 else U
    x, w, b, dy = (None if t is None else t.detach().double().cpu() for t in (x, w, b, dy))
    rows, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if w is None else w
    b = torch.zeros(d, dtype=torch.float64) if b is None else b
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h * w + b
    # a lane adds 16 values (or every 1024th of a long row), then the lanes add theirs in pairs
    c = (max(16, d / 1024) + 8 + math.log2(d + 1)) * U
    off_h = c * (rstd * x.abs().mean(1, keepdim=True) + 2 * h.abs())
    out = {"y": (y, w.abs() * off_h + 2 * U * ((h * w).abs() + b.abs()) + last * y.abs())}
    if dy is None:
        return out
    g = dy * w
    m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    gx = rstd * (g - m1 - h * m2)
    off = (4 * U * g.abs() + c * g.abs().mean(1, keepdim=True) + h.abs() * (c * (g * h).abs().mean(1, keepdim=True))
           + off_h * m2.abs() + h.abs() * (g.abs() * off_h).mean(1, keepdim=True))
    out["gx"] = gx, rstd * (off + 2 * c * (m1.abs() + (h * m2).abs())) + (last + 2 * c) * gx.abs()
    gw, gb = (dy * h).sum(0), dy.sum(0)
    out["gw"] = gw, (dy.abs() * off_h).sum(0) + terms(rows) * (dy * h).abs().sum(0) + last_w * gw.abs()
    out["gb"] = gb, terms(rows) * dy.abs().sum(0) + last_w * gb.abs()
    return out


def within(actual, expected, what):
    value, off = expected
    a = actual.detach().double().cpu()
    assert a.shape == value.shape, f"{what}: shape {tuple(a.shape)}, expected {tuple(value.shape)}"
    far = (a - value).abs()
    beyond = value.abs() > torch.finfo(actual.dtype).max   # (what the type cannot hold is infinite)
    far = torch.where(beyond & (a == value.sign() * float("inf")), torch.zeros_like(far), far)
    bad = ~(far <= off + 1e-30)
    if bad.any():
        at = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {a.numel()} are further off than the roundings allow; first at {at}: "
                             f"{a[at].item()} instead of {value[at].item()}, {far[at].item():.3e} off, {off[at].item():.3e} allowed")
