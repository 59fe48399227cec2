"""What the operators of gated blocks, their 8-bit form and the loss against a teacher give in 64 bits on the CPU, and how far results may be from
it: bounds that follow from the roundings, element by element (U, V and ``terms`` as in tests/layer_bounds.py)."""
import math

import torch

from tests.layer_bounds import CURVATURE, U, V, activation, terms

BLOCK, TOP, LEAST = 128, 448.0, 2.0 ** -100


def rms_norm(x, w, r, dy, ds, eps):
    """{name: (value, how far off)} for y, sum, gx and gw."""
    half = x.dtype == torch.bfloat16
    last, last_w = V if half else U, V if w is not None and w.dtype == torch.bfloat16 else U
    kept = last if r is not None and half else 0.0   # the backward reads the sum as it was rounded
    x, w, r, dy, ds = (None if t is None else t.detach().double().cpu() for t in (x, w, r, dy, ds))
    rows, d = x.shape
    w = torch.ones(d, dtype=torch.float64) if w is None else w
    s = x if r is None else x + r
    rstd = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + eps)
    h = s * rstd
    c = (max(16, d / 1024) + 8 + math.log2(d + 1)) * U   # a lane adds 16 values (or every 1024th of a long row), then the lanes add theirs in pairs
    off_h = h.abs() * (c / 2 + 5 * U)
    out = {"y": (h * w, w.abs() * off_h + 2 * U * (h * w).abs() + last * (h * w).abs())}
    if r is not None:
        out["sum"] = s, last * s.abs() + U * s.abs()
    if dy is None:
        return out
    off_h = off_h + kept * h.abs()
    g = dy * w
    m = (g * h).mean(1, keepdim=True)
    off_m = (g.abs() * off_h).mean(1, keepdim=True) + 2 * c * (g * h).abs().mean(1, keepdim=True)
    gx = rstd * (g - h * m)
    off = rstd * (4 * U * (g.abs() + (h * m).abs()) + off_h * m.abs() + h.abs() * off_m) + (c / 2 + 5 * U) * gx.abs()
    if ds is not None:
        gx, off = gx + ds, off + 2 * U * ds.abs()
    out["gx"] = gx, off + last * gx.abs()
    gw = (dy * h).sum(0)
    out["gw"] = gw, (dy.abs() * off_h).sum(0) + terms(rows) * (dy * h).abs().sum(0) + last_w * gw.abs()
    return out


def _kept(z, halves):
    """What is kept of z for the backward is off by: halves (half an ulp of 2^-10, or of 2^-24, and the last bit of the first of four) where the largest of four neighbouring columns allows it,
    else bfloat16 whose first of four may lose its last bit."""
    n = z.shape[1]
    top = torch.nn.functional.pad(z.abs(), (0, -n % 4)).unflatten(1, (-1, 4)).amax(2).repeat_interleave(4, 1)[:, :n]
    fits = (top > 2.0 ** -11.9) & (top < 65000) & halves
    return torch.where(fits, 1.5 * 2.0 ** -10 * z.abs() + 2.0 ** -24, 3 * V * z.abs() + 1e-40)


def gated_linear(x, w, b, dy, act):
    """{name: (value, how far off)} for y, gx, gw and gb."""
    half = x.dtype == torch.bfloat16
    last = V if half else U
    x, w, b, dy = (None if t is None else t.detach().double().cpu() for t in (x, w, b, dy))
    n, k = w.shape[0] // 2, w.shape[1]
    rows = x.shape[0]
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b, size + b.abs()
    off_g, off_u = (terms(k) * size).split(n, 1)
    g, u = z.split(n, 1)
    a, slope = activation(g, act)

    def off_a(off):   # |act'| <= 1.13; the activation's own arithmetic is a few units
        return 1.13 * off + 16 * U * (a.abs() + g.abs())

    y = a * u
    out = {"y": (y, off_a(off_g) * (u.abs() + off_u) + a.abs() * off_u + (2 * U + last) * y.abs())}
    if dy is None:
        return out
    if half:
        off_g, off_u = off_g + _kept(g, act != "relu"), off_u + _kept(u, True)
    off_s = CURVATURE[act] * off_g + (24 * U * (1 + g.abs()) if act in ("gelu", "silu") else 0)
    dg, du = dy * u * slope, dy * a
    dz = torch.cat([dg, du], 1)
    off = torch.cat([dy.abs() * (slope.abs() * off_u + (u.abs() + off_u) * off_s), dy.abs() * off_a(off_g)], 1) + 3 * U * dz.abs()
    off_dz = off + (V * dz.abs() * 1.01 if half else 0)
    gx, gw, gb = dz @ w, dz.t() @ x, dz.sum(0)
    out["gx"] = gx, off_dz @ w.abs() + terms(2 * n) * (dz.abs() @ w.abs()) + last * gx.abs()
    out["gw"] = gw, off_dz.t() @ x.abs() + terms(rows) * (dz.abs().t() @ x.abs()) + last * gw.abs()
    out["gb"] = gb, off.sum(0) + terms(rows) * dz.abs().sum(0) + last * gb.abs()
    return out


def spread(scale, n):
    return scale.repeat_interleave(BLOCK, -1)[..., :n]


def check_codes(codes, scale, value, off, weight=False):
    """Codes and scales of ``value`` (64 bits; itself off by up to ``off``): the scale is a block's largest magnitude / 448, and no code is further from its value
    than half its step -- an eighth of the value's power of two, 2^-9 below 2^-6 -- and what the arithmetic adds."""
    codes, scale = codes.cpu(), scale.double().cpu()
    assert codes.dtype == torch.float8_e4m3fn
    rows, n = value.shape
    v, o = value, off
    if weight:
        v, o = (torch.nn.functional.pad(t, (0, 0, 0, -rows % BLOCK)).unflatten(0, (-1, BLOCK)).amax(1) for t in (v.abs(), o))
    top = torch.stack([t.abs().amax(1) for t in v.split(BLOCK, 1)], 1).clamp(min=LEAST)
    off_top = torch.stack([t.amax(1) for t in o.split(BLOCK, 1)], 1)
    assert scale.shape == top.shape
    assert bool(((scale * TOP - top).abs() <= off_top + 4 * U * top).all())
    by = scale.repeat_interleave(BLOCK, 0)[:rows] if weight else scale
    by = spread(by, n)
    far = (codes.double() * by - value).abs()
    in_codes = value.abs() / by
    step = torch.exp2(torch.floor(torch.log2(in_codes.clamp(min=2.0 ** -6)))) / 8
    assert bool((far <= (step / 2 + 8 * U * in_codes) * by + off * 1.01 + step * by * (off > 0) * 0).all()), float((far / (step * by)).max())


def linear_codes(x, xs, w, ws, b, r, act, dtype):
    """(value, how far off) of the product of codes."""
    x, xs, w, ws = x.cpu().double(), xs.double().cpu(), w.cpu().double(), ws.double().cpu()
    n, k = w.shape
    x = x * spread(xs, k)
    w = w * spread(ws.repeat_interleave(BLOCK, 0)[:n], k)
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.double().cpu(), size + b.double().cpu().abs()
    # float32: sums of 32 bits.  bfloat16: the products of a block are lined up with the largest of them; 14 bits of it are kept
    off = (terms(k) + (2.0 ** -14 if dtype == torch.bfloat16 else 0)) * size
    y = activation(z, act)[0]
    off = 1.13 * off + (16 * U * (y.abs() + z.abs()) if act != "none" else 0)
    if r is not None:
        y = y + r.double().cpu()
        off = off + U * y.abs()
    return y, off + (V if dtype == torch.bfloat16 else U) * y.abs()


def distillation(l, t, i, y, T, alpha, ignore):
    """{"loss", "grad": (value, how far off)}."""
    last = V if l.dtype == torch.bfloat16 else U
    l, t, i = l.detach().double().cpu(), t.double().cpu(), i.cpu()
    rows, c = l.shape
    keep = torch.ones(rows, dtype=torch.bool) if y is None else y.cpu() != ignore
    a = 1.0 if y is None else alpha
    taught = (t > -math.inf).any(1)
    t = torch.where(taught[:, None], t, torch.zeros_like(t))
    log_p = torch.log_softmax(t / T, 1)
    p = log_p.exp() * taught[:, None]
    log_q = torch.log_softmax(l / T, 1)
    at = log_q.gather(1, i)
    kd = torch.where(p > 0, p * (log_p - at), torch.zeros_like(p)).sum(1)
    loss = a * T * T * kd if a else torch.zeros(rows, dtype=torch.float64)
    # an exponential of x is off by its argument's rounding, |x| U, and a few units; so is the logarithm of their sum
    far = lambda v: torch.where(v > -math.inf, v.abs(), torch.zeros_like(v)).amax(1, keepdim=True)
    off_q = (far(l - l.amax(1, keepdim=True)) / T * 3 + 8) * U + terms(c)
    off_p = (far(t - t.amax(1, keepdim=True)) / T * 3 + 8) * U + terms(t.shape[1])
    fine = torch.where(p > 0, (log_p - at).abs(), torch.zeros_like(p))
    off = a * T * T * ((p * (off_q + off_p + off_p * fine)).sum(1) + terms(t.shape[1]) * (p * fine).sum(1))
    q = log_q.exp()
    grad = a * T * taught[:, None] * q
    off_g = grad * off_q
    grad = grad.scatter_add(1, i, -a * T * p)
    off_g = off_g.scatter_add(1, i, a * T * p * (off_p + 4 * U))
    if y is not None and a != 1:
        of = torch.where(keep, y.cpu(), torch.zeros_like(y.cpu()))[:, None]
        log_o = torch.log_softmax(l, 1)
        off_o = (far(l - l.amax(1, keepdim=True)) * 3 + 8) * U + terms(c)
        loss = loss - (1 - a) * log_o.gather(1, of).squeeze(1)
        off = off + (1 - a) * (off_o.squeeze(1) + 4 * U * log_o.gather(1, of).squeeze(1).abs())
        grad = (grad + (1 - a) * log_o.exp()).scatter_add(1, of, torch.full_like(of, -(1 - a), dtype=torch.float64))
        off_g = (off_g + (1 - a) * log_o.exp() * off_o).scatter_add(1, of, torch.full_like(of, 4 * U, dtype=torch.float64))
    n = max(1, int(keep.sum()))
    loss, off = torch.where(keep, loss, torch.zeros_like(loss)), torch.where(keep, off, torch.zeros_like(off))
    zero = torch.zeros_like(grad)
    grad, off_g = torch.where(keep[:, None], grad / n, zero), torch.where(keep[:, None], off_g / n, zero)
    return {"loss": (loss.sum() / n, off.sum() / n + terms(rows) * loss.abs().sum() / n), "grad": (grad, off_g + (last + 4 * U) * grad.abs())}
