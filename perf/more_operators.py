"""The operators of a gated block that is trained from a teacher and then served in 8 bits, as cases that can be timed: the
root-mean-square norm with the shortcut's addition (and its form that gives 8-bit codes), the gated linear layer, the product of
8-bit operands with a scale for each block of 128 values, and the loss against a teacher's top logits.

    listed()          the named cases            draw(rng)         one more case of the same ranges
    prepare(case, s)  inputs of seed ``s`` on the GPU
    run(state)        one pass: the framework's operators where ``own``, else the same formulas in elementary operations
    exact(case, s)    what the pass returns, from the definition in 64 bits
    work(case)        bytes and operations that a pass cannot do without
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6
BLOCK = 128                # neighbouring values that share a scale; of a weight BLOCK x BLOCK
TOP = 448.0                # the largest e4m3 value
LEAST = 2.0 ** -100        # a block's largest magnitude counts as at least this
TEMPERATURE, ALPHA, IGNORED = 2.0, 0.7, -100


def listed():
    return [
        # serving, one token: the shortcut's addition and the norm in front of a block; nothing but latency
        {"name": "norm_row_bf16", "op": "norm", "dtype": "bfloat16", "rows": 1, "d": 4096, "residual": True, "out": "same", "train": False},
        # the same on a training batch, forward and backward
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bfloat16", "rows": 16384, "d": 2048, "residual": True, "out": "same", "train": True},
        # an odd width and number of rows, in float32, without a shortcut
        {"name": "norm_odd_train_f32", "op": "norm", "dtype": "float32", "rows": 3001, "d": 777, "residual": False, "out": "same", "train": True},
        # serving a long batch in 8 bits: the norm's result as codes for the product behind it
        {"name": "norm_codes_bf16", "op": "norm", "dtype": "bfloat16", "rows": 8192, "d": 4096, "residual": True, "out": "fp8", "train": False},
        # serving a few tokens: the time is that of reading the weight
        {"name": "gated_rows_bf16", "op": "gated", "dtype": "bfloat16", "rows": 4, "k": 4096, "hidden": 8192, "act": "silu", "bias": False, "train": False},
        # a training step's share of a gated block's first half: the largest products here
        {"name": "gated_train_bf16", "op": "gated", "dtype": "bfloat16", "rows": 8192, "k": 1024, "hidden": 4096, "act": "silu", "bias": False, "train": True},
        # sizes that are multiples of nothing, in float32, with biases
        {"name": "gated_odd_train_f32", "op": "gated", "dtype": "float32", "rows": 1531, "k": 515, "hidden": 1027, "act": "gelu", "bias": True, "train": True},
        # serving one token in 8 bits: the time is that of reading the weight
        {"name": "fp8_row_bf16", "op": "fp8", "dtype": "bfloat16", "rows": 1, "k": 4096, "n": 8192, "residual": False},
        # a long batch in 8 bits, with the block's shortcut
        {"name": "fp8_long_bf16", "op": "fp8", "dtype": "bfloat16", "rows": 8192, "k": 4096, "n": 4096, "residual": True},
        # sizes that no block and no tile divides, a float32 result
        {"name": "fp8_odd_f32", "op": "fp8", "dtype": "float32", "rows": 1531, "k": 1000, "n": 1027, "residual": False},
        # a classifier of a thousand classes taught at batch 256, in this framework's own float32
        {"name": "distill_classes_f32", "op": "distill", "dtype": "float32", "rows": 256, "classes": 1000, "top": 20, "labels": True},
        # many classes, as a teacher of tokens has them; a twentieth of the rows is padding
        {"name": "distill_long_bf16", "op": "distill", "dtype": "bfloat16", "rows": 4096, "classes": 32000, "top": 64, "labels": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo, hi, of):
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.4 else -(-n // of) * of


def draw(rng):
    op = rng.choice(["norm", "norm", "gated", "gated", "fp8", "fp8", "distill"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "norm":
        d, out = _width(rng, 16, 16384, 8), rng.choice(["same", "same", "fp8"])
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(32768, (1 << 24) // d)), "d": d, "residual": rng.random() < 0.6, "out": out,
                "train": out == "same" and rng.random() < 0.7}
    if op == "gated":
        k, h = _width(rng, 48, 4096, 8), _width(rng, 16, 4096, 8)
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(16384, (1 << (33 if dtype == "float32" else 35)) // (k * h))), "k": k, "hidden": h,
                "act": rng.choice(["gelu", "silu"]), "bias": rng.random() < 0.5, "train": rng.random() < 0.6}
    if op == "fp8":
        k, n = _width(rng, 128, 8192, 128), _width(rng, 64, 8192, 128)
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(16384, (1 << 36) // (k * n))), "k": k, "n": n, "residual": rng.random() < 0.5}
    classes = _log_int(rng, 10, 128000)
    return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(8192, (1 << 26) // classes)), "classes": classes,
            "top": _log_int(rng, 1, min(classes, 128)), "labels": rng.random() < 0.7}


def _blocks(v, of=BLOCK):
    """The last dimension in blocks of ``of`` values, the last one filled with zeros."""
    return torch.nn.functional.pad(v, (0, -v.shape[-1] % of)).unflatten(-1, (-1, of))


def _codes(v, largest, spread):
    """e4m3 codes of blocks, and the scales that give their values back; ``spread`` lays one number a block over its values."""
    top = largest.clamp(min=LEAST)
    return (v * (TOP / spread(top))).to(torch.float8_e4m3fn), top / TOP


def _codes_rows(v):
    """e4m3 codes of ``v`` (rows, d) and a scale for each BLOCK values of a row."""
    b = _blocks(v)
    q, s = _codes(b, b.abs().amax(-1), lambda t: t.unsqueeze(-1))
    return q.flatten(-2)[..., :v.shape[-1]].contiguous(), s


def _codes_weight(w):
    """e4m3 codes of ``w`` (n, k) and a scale for each BLOCK x BLOCK of it."""
    n, k = w.shape
    b = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).unflatten(0, (-1, BLOCK)).unflatten(2, (-1, BLOCK))
    q, s = _codes(b, b.abs().amax((1, 3)), lambda t: t[:, None, :, None])
    return q.flatten(2).flatten(0, 1)[:n, :k].contiguous(), s


def _inputs(case, seed):
    """The numbers of a case on the GPU, by name."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale).add_(mean).to(dtype)

    def rows_of(m, n):   # what layers hand on: a few channels of large values, as trained networks have
        x = torch.randn(m, n, generator=g, device=DEV)
        x[:, torch.randint(0, n, (max(1, n // 256),), generator=g, device=DEV)] *= 8
        return x

    if case["op"] == "norm":
        m, n = case["rows"], case["d"]
        d = {"x": rows_of(m, n).to(dtype), "w": normal(n, scale=0.1, mean=1.0)}
        if case["residual"]:
            d["r"] = normal(m, n, scale=2.0)
        if case["train"]:
            d["dy"] = normal(m, n, scale=m ** -0.5)
            if case["residual"]:
                d["ds"] = normal(m, n, scale=m ** -0.5)
        return d
    if case["op"] == "gated":
        m, k, h = case["rows"], case["k"], case["hidden"]
        d = {"x": normal(m, k), "w": normal(2 * h, k, scale=k ** -0.5)}   # (the gate's rows first)
        if case["bias"]:
            d["b"] = normal(2 * h, scale=0.1)
        if case["train"]:
            d["dy"] = normal(m, h, scale=m ** -0.5)
        return d
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        d = {}
        d["x"], d["xs"] = _codes_rows(rows_of(m, k))
        d["w"], d["ws"] = _codes_weight(torch.randn(n, k, generator=g, device=DEV) * k ** -0.5)
        if case["residual"]:
            d["r"] = normal(m, n)
        return d
    m, c, k = case["rows"], case["classes"], case["top"]
    teacher = torch.randn(m, c, generator=g, device=DEV) * 2
    l = (0.6 * teacher + 1.2 * torch.randn(m, c, generator=g, device=DEV)).to(dtype)   # a student on its way
    t, i = teacher.topk(k, dim=1)
    d = {"l": l, "t": t.to(dtype), "i": i}
    if case["labels"]:
        y = torch.where(torch.rand(m, generator=g, device=DEV) < 0.8, i[:, 0], torch.randint(0, c, (m,), generator=g, device=DEV))
        d["y"] = torch.where((torch.rand(m, generator=g, device=DEV) < 0.05) & (torch.arange(m, device=DEV) > 0), torch.full_like(y, IGNORED), y)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if own:
        for name in ("x", "w", "b", "r") if case.get("train") else ("l",) if case["op"] == "distill" else ():
            if name in d:
                d[name].requires_grad_(True)
    return {"case": case, **d}


def _act(z, name):
    """The activation and its derivative."""
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _norm(x, w, r, dy, ds):
    """s = x + r, y = s / sqrt(mean(s^2) + eps) w, and the gradients of x, w and r."""
    s = x if r is None else x + r
    rho = 1 / torch.sqrt(s.square().mean(1, keepdim=True) + EPS)
    h = s * rho
    out = {"y": h * w}
    if r is not None:
        out["s"] = s
    if dy is None:
        return out
    g = dy * w
    gx = rho * (g - h * (g * h).mean(1, keepdim=True))
    out["gx"], out["gw"] = gx if ds is None else gx + ds, (dy * h).sum(0)
    if r is not None:
        out["gr"] = out["gx"]
    return out


def _gated(x, w, b, dy, act):
    """act(x wg' + bg) (x wu' + bu), and the gradients of x, w and b."""
    z = x @ w.t()
    if b is not None:
        z = z + b
    g, u = z.chunk(2, 1)
    a, slope = _act(g, act)
    out = {"y": a * u}
    if dy is None:
        return out
    dz = torch.cat([dy * u * slope, dy * a], 1)
    out.update(gx=dz @ w, gw=dz.t() @ x)
    return out if b is None else {**out, "gb": dz.sum(0)}


def _spread(s, n):
    """Scales of blocks as one for each of ``n`` values."""
    return s.repeat_interleave(BLOCK, -1)[..., :n]


def _product(x, xs, w, ws, r):
    n, k = w.shape
    y = (x.float() * _spread(xs, k)) @ (w.float() * _spread(_spread(ws, k).t(), n).t()).t()
    return y if r is None else y + r.float()


def _distill(l, t, i, y):
    """The loss and the logits' gradient."""
    keep = torch.ones(l.shape[0], dtype=torch.bool, device=l.device) if y is None else y != IGNORED
    count = keep.sum().clamp(min=1).to(l.dtype)
    a = 1.0 if y is None else ALPHA
    z = l / TEMPERATURE
    z = z - z.amax(1, keepdim=True)
    log_q = z - torch.log(torch.exp(z).sum(1, keepdim=True))
    v = t / TEMPERATURE
    v = v - v.amax(1, keepdim=True)
    log_p = v - torch.log(torch.exp(v).sum(1, keepdim=True))
    p = torch.exp(log_p)
    row = a * TEMPERATURE ** 2 * (p * (log_p - log_q.gather(1, i))).sum(1)
    grad = (a * TEMPERATURE * torch.exp(log_q)).scatter_add(1, i, -a * TEMPERATURE * p)
    if y is not None:
        of = torch.where(keep, y, torch.zeros_like(y)).unsqueeze(1)
        o = l - l.amax(1, keepdim=True)
        log_o = o - torch.log(torch.exp(o).sum(1, keepdim=True))
        row = row - (1 - a) * log_o.gather(1, of).squeeze(1)
        grad = (grad + (1 - a) * torch.exp(log_o)).scatter_add(1, of, torch.full_like(of, -(1 - a), dtype=l.dtype))
    zero = torch.zeros((), dtype=l.dtype, device=l.device)
    return torch.where(keep, row, zero).sum() / count, torch.where(keep.unsqueeze(1), grad / count, zero)


def _rounded(out, dtype):
    return {name: t.to(dtype) for name, t in out.items()}


def _float(state, *names):
    return [state[n].float() if n in state else None for n in names]


def run(state):
    case = state["case"]
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "norm":
        if own:
            x, w, r = state["x"], state["w"], state.get("r")
            if case["out"] == "fp8":
                from addernetcuda_amd.fp8 import rms_norm_fp8
                got = rms_norm_fp8(x, w, EPS, residual=r)
                return dict(zip(("q", "scale", "s"), got))
            from addernetcuda_amd.rms_norm import rms_norm
            if not case["train"]:
                with torch.no_grad():
                    got = rms_norm(x, w, EPS, residual=r)
                return {"y": got} if r is None else dict(zip(("y", "s"), got))
            got = rms_norm(x, w, EPS, residual=r)
            if r is None:
                return {"y": got, **dict(zip(("gx", "gw"), torch.autograd.grad(got, (x, w), state["dy"])))}
            return {"y": got[0], "s": got[1], **dict(zip(("gx", "gw", "gr"), torch.autograd.grad(got, (x, w, r), (state["dy"], state["ds"]))))}
        out = _norm(*_float(state, "x", "w", "r", "dy", "ds"))
        if case["out"] == "fp8":
            q, scale = _codes_rows(out["y"])
            return {"q": q, "scale": scale, **({"s": out["s"].to(dtype)} if "s" in out else {})}
        return _rounded(out, dtype)
    if case["op"] == "gated":
        if own:
            from addernetcuda_amd.gated import gated_linear
            x, w, b = state["x"], state["w"], state.get("b")
            if not case["train"]:
                with torch.no_grad():
                    return {"y": gated_linear(x, w, b, act=case["act"])}
            y = gated_linear(x, w, b, act=case["act"])
            names, of = (("gx", "gw"), (x, w)) if b is None else (("gx", "gw", "gb"), (x, w, b))
            return {"y": y, **dict(zip(names, torch.autograd.grad(y, of, state["dy"])))}
        return _rounded(_gated(*_float(state, "x", "w", "b", "dy"), case["act"]), dtype)
    if case["op"] == "fp8":
        if own:
            from addernetcuda_amd.fp8 import linear_fp8
            return {"y": linear_fp8(state["x"], state["xs"], state["w"], state["ws"], residual=state.get("r"), dtype=dtype)}
        return {"y": _product(state["x"], state["xs"], state["w"], state["ws"], state.get("r")).to(dtype)}
    if own:
        from addernetcuda_amd.distill import distillation_loss
        loss = distillation_loss(state["l"], state["t"], state["i"], state.get("y"), temperature=TEMPERATURE, alpha=ALPHA, ignore_index=IGNORED)
        return {"loss": loss, "gl": torch.autograd.grad(loss, state["l"])[0]}
    loss, grad = _distill(state["l"].float(), state["t"].float(), state["i"], state.get("y"))
    return {"loss": loss, "gl": grad.to(dtype)}


def _exact_norm(d, out_kind):
    s = d["x"].double()
    if "r" in d:
        s = s + d["r"].double()
    w, n = d["w"].double(), s.shape[1]
    sigma = torch.sqrt((s * s).sum(1, keepdim=True) / n + EPS)
    h = s / sigma
    y = w * h
    out = {"s": s} if "r" in d else {}
    if out_kind == "fp8":
        top = torch.stack([t.abs().amax(1) for t in y.split(BLOCK, 1)], 1).clamp(min=LEAST)
        out["q"] = (y / (top / TOP).repeat_interleave(BLOCK, 1)[:, :n]).float().to(torch.float8_e4m3fn).double()
        out["scale"] = top / TOP
        return out
    out["y"] = y
    if "dy" in d:
        dy = d["dy"].double()
        a = dy * w
        gx = (n * a - h * torch.sum(a * h, 1, keepdim=True)) / (n * sigma)
        out["gx"] = torch.add(gx, d["ds"].double()) if "ds" in d else gx
        out["gw"] = torch.sum(dy * h, 0)
        if "r" in d:
            out["gr"] = out["gx"]
    return out


def _exact_gated(d, act):
    x, w = d["x"].double(), d["w"].double()
    h = w.shape[0] // 2
    b = d["b"].double() if "b" in d else torch.zeros(2 * h, dtype=torch.float64, device=DEV)
    g, u = torch.addmm(b[:h], x, w[:h].t()), torch.addmm(b[h:], x, w[h:].t())
    if act == "gelu":
        below = 0.5 * torch.special.erfc(-g / 2 ** 0.5)
        a, slope = g * below, below + g * torch.exp(-g.square() / 2) * (0.5 / math.pi) ** 0.5
    else:
        e = torch.special.expit(g)
        a, slope = g * e, e + g * e * (1 - e)
    out = {"y": a * u}
    if "dy" in d:
        dy = d["dy"].double()
        dg, du = dy * slope * u, dy * a
        out["gx"] = torch.addmm(dg @ w[:h], du, w[h:])
        out["gw"] = torch.cat([dg.t().contiguous() @ x, du.t().contiguous() @ x])
        if "b" in d:
            out["gb"] = torch.cat([dg.sum(0), du.sum(0)])
    return out


def _exact_product(d):
    x, w, xs, ws = (d[n].double() for n in ("x", "w", "xs", "ws"))
    y = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    of = torch.arange(w.shape[0], device=DEV) // BLOCK
    for b, at in enumerate(range(0, x.shape[1], BLOCK)):
        y += (x[:, at:at + BLOCK] @ w[:, at:at + BLOCK].t()) * xs[:, b:b + 1] * ws[of, b]
    return {"y": y + d["r"].double() if "r" in d else y}


def _exact_distill(d):
    l, t, i, y = d["l"].double(), d["t"].double(), d["i"], d.get("y")
    rows = torch.arange(l.shape[0], device=DEV) if y is None else torch.nonzero(y != IGNORED).squeeze(1)
    a, n = (1.0 if y is None else ALPHA), max(1, rows.numel())
    lk, tk, ik = l[rows], t[rows], i[rows]
    lse = torch.logsumexp(lk / TEMPERATURE, 1, keepdim=True)
    p = torch.softmax(tk / TEMPERATURE, 1)
    log_p = tk / TEMPERATURE - torch.logsumexp(tk / TEMPERATURE, 1, keepdim=True)
    loss = a * TEMPERATURE ** 2 * torch.sum(p * (log_p + lse - torch.gather(lk, 1, ik) / TEMPERATURE))
    part = a * TEMPERATURE * torch.softmax(lk / TEMPERATURE, 1)
    part.scatter_add_(1, ik, -a * TEMPERATURE * p)
    if y is not None:
        at = torch.arange(rows.numel(), device=DEV)
        loss = loss + (1 - a) * torch.sum(torch.logsumexp(lk, 1) - lk[at, y[rows]])
        part += (1 - a) * torch.softmax(lk, 1)
        part[at, y[rows]] -= 1 - a
    grad = torch.zeros_like(l)
    grad[rows] = part / n
    return {"loss": loss / n, "gl": grad}


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "norm":
        return _exact_norm(d, case["out"])
    if case["op"] == "gated":
        return _exact_gated(d, case["act"])
    return _exact_product(d) if case["op"] == "fp8" else _exact_distill(d)


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        m, n = case["rows"], case["d"]
        r, t = (1 if case["residual"] else 0), case["train"]
        rows = e * (1 + 2 * r + (0 if case["out"] == "fp8" else 1))                     # x, r, the sum, y
        rows += (1 + 4 / BLOCK) if case["out"] == "fp8" else 0
        rows += e * (2 + r) if t else 0                                                # dy, the sum's gradient, gx (r's is the same one)
        return {"bytes": rows * m * n + e * n * (2 if t else 1), "flops": (14 if t else 5) * m * n}
    if case["op"] == "gated":
        m, k, h = case["rows"], case["k"], case["hidden"]
        b = 2 * h if case["bias"] else 0
        if not case["train"]:
            return {"bytes": e * (m * k + 2 * h * k + b + m * h), "flops": 4 * m * k * h}
        return {"bytes": e * (2 * m * k + 4 * h * k + 2 * b + 2 * m * h), "flops": 12 * m * k * h}
    if case["op"] == "fp8":
        m, k, n = case["rows"], case["k"], case["n"]
        blocks = -(-k // BLOCK)
        return {"bytes": m * k + n * k + 4 * blocks * (m + -(-n // BLOCK)) + e * m * n * (2 if case["residual"] else 1), "flops": 2 * m * n * k}
    m, c, k = case["rows"], case["classes"], case["top"]
    return {"bytes": 2 * e * m * c + (8 + e) * m * k + (8 * m if case["labels"] else 0), "flops": 16 * m * c}
