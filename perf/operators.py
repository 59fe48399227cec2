"""The operators of a network of linear layers that trains beside the adder layers, as cases that can be timed: a linear layer
with bias, activation and residual in one call, layer normalisation, and the AdamW step over many tensors; forward and
backward, in float32 and bfloat16.

    listed()          the named cases            draw(rng)         one more case of the same ranges
    prepare(case, s)  inputs of seed ``s`` on the GPU, and the optimizer where there is one
    run(state)        one pass: the framework's operators where ``own``, else the same formulas in elementary operations
    exact(case, s)    what the pass returns, from the definition in 64 bits
    work(case)        bytes and operations that a pass cannot do without
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 256          # values that share a scale where the optimizer's state is held in 8 bits
MIN_8BIT = 4096      # smaller tensors keep their state in 32 bits
EPS_NORM = 1e-5
LR, BETA1, BETA2, EPS_ADAM, DECAY, STEPS_DONE = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100

# Tensors of the optimizer's cases.  "resnet20": the parameters of the network that this framework's benchmark trains.
# "mlp": `layers` residual MLP blocks of `width` channels (norm, width -> 4 width, 4 width -> width, with biases).
# "odd": `layers` pairs of a matrix whose sides are multiples of nothing, and its bias.


def _resnet20_sizes():
    sizes, wide = [16 * 3 * 9, 16, 16], [16, 16, 32, 64]
    for stage in (1, 2, 3):
        for block in range(3):
            into = wide[stage - 1] if block == 0 else wide[stage]
            out = wide[stage]
            sizes += [out * into * 9, out, out, out * out * 9, out, out]
            if block == 0 and stage > 1:
                sizes += [out * into, out, out]
    return sizes + [10 * 64, 10, 10]


def _sizes(case):
    n, w = case["layers"], case["width"]
    if case["net"] == "resnet20":
        return _resnet20_sizes()
    if case["net"] == "mlp":
        return [w, w, 4 * w * w, 4 * w, 4 * w * w, w] * n
    return [(w + 3) * (2 * w + 1), 2 * w + 1] * n


def listed():
    return [
        # serving, one token: a square layer with bias and residual; the time is that of reading the weight
        {"name": "linear_row_bf16", "op": "linear", "dtype": "bfloat16", "rows": 1, "k": 4096, "n": 4096, "act": "none",
         "residual": True, "train": False},
        # the classifier of ResNet-50 (2048 features, a thousand classes) on a small batch, in this framework's own float32
        {"name": "linear_classes_f32", "op": "linear", "dtype": "float32", "rows": 32, "k": 2048, "n": 1000, "act": "none",
         "residual": False, "train": False},
        # a long batch through the second layer of an MLP block, with the block's residual, without gradients
        {"name": "linear_long_bf16", "op": "linear", "dtype": "bfloat16", "rows": 8192, "k": 4096, "n": 1024, "act": "none",
         "residual": True, "train": False},
        # a training step's share of the first layer of an MLP block: the largest products here
        {"name": "linear_train_bf16", "op": "linear", "dtype": "bfloat16", "rows": 8192, "k": 1024, "n": 4096, "act": "gelu",
         "residual": False, "train": True},
        # the 512 -> 512 layer with ReLU of the VGG classifiers, training at batch 128: latency counts
        {"name": "linear_vgg_train_f32", "op": "linear", "dtype": "float32", "rows": 128, "k": 512, "n": 512, "act": "relu",
         "residual": False, "train": True},
        # sizes that are multiples of nothing, in float32, with everything in the epilogue
        {"name": "linear_odd_train_f32", "op": "linear", "dtype": "float32", "rows": 1531, "k": 515, "n": 1027, "act": "gelu",
         "residual": True, "train": True},
        # serving, a few tokens: nothing but latency
        {"name": "norm_rows_f32", "op": "norm", "dtype": "float32", "rows": 8, "d": 512, "train": False},
        # the norm in front of the block above, forward and backward, over a long batch
        {"name": "norm_train_bf16", "op": "norm", "dtype": "bfloat16", "rows": 16384, "d": 1024, "train": True},
        # an odd width and number of rows, in float32
        {"name": "norm_odd_train_f32", "op": "norm", "dtype": "float32", "rows": 3001, "d": 777, "train": True},
        # the network of this framework's benchmark: 65 small tensors, 272 000 values in all
        {"name": "adamw_resnet20_f32", "op": "adamw", "dtype": "float32", "bits": 32, "net": "resnet20", "layers": 1, "width": 16},
        # eight MLP blocks of 1024 channels, 67 million values, the optimizer's state in 32 bits
        {"name": "adamw_large_f32", "op": "adamw", "dtype": "float32", "bits": 32, "net": "mlp", "layers": 8, "width": 1024},
        # the same with the state in 8 bits
        {"name": "adamw_large_8bit", "op": "adamw", "dtype": "float32", "bits": 8, "net": "mlp", "layers": 8, "width": 1024},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "adamw"])
    dtype = rng.choice(["float32", "bfloat16"])
    if op == "adamw":
        net = rng.choice(["mlp", "odd"])
        return {"op": op, "dtype": dtype, "bits": rng.choice([8, 32]), "net": net, "layers": rng.randint(1, 7),
                "width": _log_int(rng, 16, 1024) if net == "odd" else 8 * _log_int(rng, 2, 128)}
    train = rng.random() < 0.6
    if op == "norm":
        d = _log_int(rng, 16, 8192)
        if rng.random() < 0.6:
            d = -(-d // 8) * 8
        return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(32768, (1 << 24) // d)), "d": d, "train": train}
    k, n = _log_int(rng, 48, 4096), _log_int(rng, 10, 4096)
    if rng.random() < 0.6:
        k, n = -(-k // 8) * 8, -(-n // 8) * 8
    # (ReLU's gradient jumps where a sum cancels to nothing, and float32 gradients are compared closely: not drawn together)
    acts = ["none", "gelu", "silu"] if train and dtype == "float32" else ["none", "relu", "gelu", "silu"]
    return {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, min(16384, (1 << 35) // (k * n))), "k": k, "n": n,
            "act": rng.choice(acts), "residual": rng.random() < 0.5, "train": train}


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def _inputs(case, seed):
    """The numbers of a case on the GPU, by name."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dtype = getattr(torch, case["dtype"])

    def normal(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(scale).add_(mean).to(dtype)

    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        d = {"x": normal(m, k), "w": normal(n, k, scale=k ** -0.5), "b": normal(n, scale=0.1)}
        if case["residual"]:
            d["r"] = normal(m, n)
        if case["train"]:
            d["dy"] = normal(m, n, scale=m ** -0.5)
        return d
    if case["op"] == "norm":
        m, n = case["rows"], case["d"]
        x = torch.randn(m, n, generator=g, device=DEV) + 0.3 * torch.randn(m, 1, generator=g, device=DEV)
        x[:, torch.randint(0, n, (max(1, n // 256),), generator=g, device=DEV)] *= 8   # a few channels of large values, as trained networks have
        d = {"x": x.to(dtype), "w": normal(n, scale=0.1, mean=1.0), "b": normal(n, scale=0.1)}
        if case["train"]:
            d["dy"] = normal(m, n, scale=m ** -0.5)
        return d
    # The tensors lie one after the other, each from a multiple of BLOCK values on, with zeros between them.  Those whose
    # state is in 8 bits come first.
    small = MIN_8BIT if case["bits"] == 8 else 0
    sizes = _sizes(case)
    sizes = [n for n in sizes if n >= small] + [n for n in sizes if n < small]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + _padded(n))
    total, coded = starts[-1], sum(_padded(n) for n in sizes if n >= small) if case["bits"] == 8 else 0
    live = torch.zeros(total, device=DEV)
    for a, n in zip(starts, sizes):
        live[a:a + n] = 1
    # a gradient's size varies over the channels by orders of magnitude; the state is what such gradients leave
    spread = torch.exp(2 * torch.randn(total // 16, generator=g, device=DEV)).repeat_interleave(16).mul_(1e-3 * live)
    grad = (torch.randn(total, generator=g, device=DEV) * spread).to(dtype)
    first = torch.randn(total, generator=g, device=DEV).mul_(0.25) * spread
    second = (torch.rand(total, generator=g, device=DEV) + 0.05) * spread * spread
    d = {"p": (torch.randn(total, generator=g, device=DEV) * 0.05 * live).to(dtype), "g": grad, "coded": coded,
         "sizes": sizes, "starts": starts[:-1], "m": first[coded:].clone(), "v": second[coded:].clone()}
    if coded:
        d["qm"], d["sm"] = _encode_first(first[:coded])
        d["qv"], d["sv"] = _encode_second(second[:coded])
    return d


# The 8-bit state: BLOCK neighbouring values share the largest magnitude among them as their scale s.  A first moment is
# sign(q) s (q / 127)^2 for a code q of -127 .. 127, a second moment s (q / 255)^4 for a code of 0 .. 255; codes go to the
# nearest in that root's scale, and a second moment that is not zero keeps a code that is not zero.
def _encode_first(m):
    b = m.view(-1, BLOCK)
    s = b.abs().amax(1, keepdim=True)
    q = torch.round(127 * torch.sqrt(b.abs() / torch.where(s > 0, s, torch.ones_like(s)))) * torch.sign(b)
    return q.to(torch.int8).view(-1), s.view(-1)


def _encode_second(v):
    b = v.view(-1, BLOCK)
    s = b.amax(1, keepdim=True)
    q = torch.round(255 * torch.sqrt(torch.sqrt(b / torch.where(s > 0, s, torch.ones_like(s)))))
    return torch.where(b > 0, torch.clamp(q, min=1), q).to(torch.uint8).view(-1), s.view(-1)


def _decode_first(q, s):
    q = q.view(-1, BLOCK).to(s.dtype)
    return (s.view(-1, 1) * torch.sign(q) * (q / 127) ** 2).view(-1)


def _decode_second(q, s):
    return (s.view(-1, 1) * (q.view(-1, BLOCK).to(s.dtype) / 255) ** 4).view(-1)


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["op"] != "adamw":
        if own and case["train"]:
            for name in ("x", "w", "b", "r"):
                if name in d:
                    d[name].requires_grad_(True)
        return {"case": case, **d}
    d["step"] = STEPS_DONE
    if own:
        from addernetcuda_amd.optim import AdamW
        params = []
        for a, n in zip(d["starts"], d["sizes"]):
            p = torch.nn.Parameter(d["p"][a:a + n])
            p.grad = d["g"][a:a + n]
            params.append(p)
        d["opt"] = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS_ADAM, weight_decay=DECAY, state_bits=case["bits"])
        for p, a, n in zip(params, d["starts"], d["sizes"]):   # as a checkpoint restores it
            if a < d["coded"]:
                c, k = a // BLOCK, _padded(n) // BLOCK
                d["opt"].state[p] = {"step": STEPS_DONE, "exp_avg": d["qm"][a:a + n], "exp_avg_scale": d["sm"][c:c + k],
                                     "exp_avg_sq": d["qv"][a:a + n], "exp_avg_sq_scale": d["sv"][c:c + k]}
            else:
                a -= d["coded"]
                d["opt"].state[p] = {"step": STEPS_DONE, "exp_avg": d["m"][a:a + n], "exp_avg_sq": d["v"][a:a + n]}
    return {"case": case, **d}


def _act(z, name):
    """The activation and its derivative."""
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    return z, None


def _linear(x, w, b, r, dy, act):
    """y = act(x w' + b) + r, and the gradients of x, w, b and r, in the type of the arguments."""
    z = x @ w.t() + b
    y, slope = _act(z, act)
    y = y if r is None else y + r
    if dy is None:
        return {"y": y}
    dz = dy if slope is None else dy * slope
    out = {"y": y, "gx": dz @ w, "gw": dz.t() @ x, "gb": dz.sum(0)}
    return out if r is None else {**out, "gr": dy}


def _norm(x, w, b, dy):
    """y = (x - mean) / sqrt(var + eps) w + b over the last dimension, and the gradients of x, w and b."""
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + EPS_NORM)
    h = (x - mean) * rstd
    y = h * w + b
    if dy is None:
        return {"y": y}
    g = dy * w
    gx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return {"y": y, "gx": gx, "gw": (dy * h).sum(0), "gb": dy.sum(0)}


def _adamw(p, g, m, v, step):
    """The new parameters and moments, in the type of the arguments."""
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    root = torch.sqrt(v) / math.sqrt(1 - BETA2 ** step) + EPS_ADAM
    return p * (1 - LR * DECAY) - LR / (1 - BETA1 ** step) * (m / root), m, v


def _rounded(out, dtype):
    return {name: t.to(dtype) for name, t in out.items()}


def run(state):
    case = state["case"]
    if case["op"] == "linear":
        x, w, b, r, dy = state["x"], state["w"], state["b"], state.get("r"), state.get("dy")
        if own:
            from addernetcuda_amd.linear import linear_act
            if dy is None:
                with torch.no_grad():
                    return {"y": linear_act(x, w, b, residual=r, act=case["act"])}
            y = linear_act(x, w, b, residual=r, act=case["act"])
            names, of = (("gx", "gw", "gb"), (x, w, b)) if r is None else (("gx", "gw", "gb", "gr"), (x, w, b, r))
            return {"y": y, **dict(zip(names, torch.autograd.grad(y, of, dy)))}
        return _rounded(_linear(x.float(), w.float(), b.float(), None if r is None else r.float(),
                                None if dy is None else dy.float(), case["act"]), x.dtype)
    if case["op"] == "norm":
        x, w, b, dy = state["x"], state["w"], state["b"], state.get("dy")
        if own:
            from addernetcuda_amd.layer_norm import layer_norm
            if dy is None:
                with torch.no_grad():
                    return {"y": layer_norm(x, w, b, EPS_NORM)}
            y = layer_norm(x, w, b, EPS_NORM)
            return {"y": y, **dict(zip(("gx", "gw", "gb"), torch.autograd.grad(y, (x, w, b), dy)))}
        return _rounded(_norm(x.float(), w.float(), b.float(), None if dy is None else dy.float()), x.dtype)
    # A state of 8 bits is returned as the values that it stands for, which have the digits of a bfloat16.
    c, out = state["coded"], {"p": state["p"], "m": state["m"], "v": state["v"]}
    if own:
        state["opt"].step()
        if c:
            from addernetcuda_amd.optim import state_values
            out["m8"] = state_values(state["qm"], state["sm"], torch.bfloat16)
            out["v8"] = state_values(state["qv"], state["sv"], torch.bfloat16)
        return out
    state["step"] += 1
    m, v = state["m"], state["v"]
    if c:
        m = torch.cat([_decode_first(state["qm"], state["sm"]), m])
        v = torch.cat([_decode_second(state["qv"], state["sv"]), v])
    p, m, v = _adamw(state["p"].float(), state["g"].float(), m, v, state["step"])
    state["p"].copy_(p)
    state["m"].copy_(m[c:])
    state["v"].copy_(v[c:])
    if c:
        state["qm"], state["sm"] = _encode_first(m[:c])
        state["qv"], state["sv"] = _encode_second(v[:c])
        out["m8"] = _decode_first(state["qm"], state["sm"]).to(torch.bfloat16)
        out["v8"] = _decode_second(state["qv"], state["sv"]).to(torch.bfloat16)
    return out


def _exact_linear(d, act):
    x, w = d["x"].double(), d["w"].double()
    z = torch.addmm(d["b"].double(), x, w.t())
    if act == "gelu":
        below = 0.5 * torch.special.erfc(-z / 2 ** 0.5)
        y, slope = z * below, below + z * torch.exp(-z.square() / 2) * (0.5 / math.pi) ** 0.5
    elif act == "silu":
        s = torch.special.expit(z)
        y, slope = z * s, s + z * s * (1 - s)
    elif act == "relu":
        y, slope = z.clamp(min=0), torch.heaviside(z, torch.zeros_like(z))
    else:
        y, slope = z, torch.ones_like(z)
    if "r" in d:
        y = y + d["r"].double()
    out = {"y": y}
    if "dy" in d:
        dz = d["dy"].double() * slope
        out.update(gx=torch.mm(dz, w), gw=torch.mm(dz.t().contiguous(), x), gb=dz.sum(dim=0))
        if "r" in d:
            out["gr"] = d["dy"].double()
    return out


def _exact_norm(d):
    x, w = d["x"].double(), d["w"].double()
    n = x.shape[1]
    centred = x - x.sum(1, keepdim=True) / n
    sigma = torch.sqrt((centred * centred).sum(1, keepdim=True) / n + EPS_NORM)
    h = centred / sigma
    out = {"y": torch.addcmul(d["b"].double(), h, w)}
    if "dy" in d:
        dy = d["dy"].double()
        a = dy * w
        gx = (n * a - a.sum(1, keepdim=True) - h * torch.sum(a * h, 1, keepdim=True)) / (n * sigma)
        out.update(gx=gx, gw=torch.sum(dy * h, 0), gb=torch.sum(dy, 0))
    return out


def _exact_adamw(d):
    c, t = d["coded"], STEPS_DONE + 1
    g, m, v = d["g"].double(), d["m"].double(), d["v"].double()
    if c:
        qm, qv = d["qm"].double().view(-1, BLOCK), d["qv"].double().view(-1, BLOCK)
        m = torch.cat([(d["sm"].double()[:, None] * qm * qm.abs() / 127 ** 2).flatten(), m])
        v = torch.cat([(d["sv"].double()[:, None] * (qv / 255).pow(4)).flatten(), v])
    m = torch.lerp(m, g, 1 - BETA1)
    v = v * BETA2 + (1 - BETA2) * g.square()
    mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = d["p"].double()
    p = p - LR * DECAY * p - LR * mhat / (vhat.sqrt() + EPS_ADAM)
    out = {"p": p, "m": m[c:], "v": v[c:]}
    if c:
        m8, v8 = m[:c].view(-1, BLOCK), v[:c].view(-1, BLOCK)
        tiny = torch.finfo(torch.float64).tiny
        sm, sv = m8.abs().amax(1, keepdim=True), v8.amax(1, keepdim=True)
        qm = torch.round(127 * (m8.abs() / sm.clamp(min=tiny)).sqrt())
        qv = torch.maximum(torch.round(255 * (v8 / sv.clamp(min=tiny)).pow(0.25)), (v8 > 0).double())
        out["m8"] = (torch.copysign(qm * qm, m8) / 127 ** 2 * sm).flatten()
        out["v8"] = ((qv / 255).pow(4) * sv).flatten()
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["op"] == "linear":
        return _exact_linear(d, case["act"])
    return _exact_norm(d) if case["op"] == "norm" else _exact_adamw(d)


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        r = m * n if case["residual"] else 0
        if not case["train"]:
            return {"bytes": e * (m * k + n * k + n + r + m * n), "flops": 2 * m * n * k}
        return {"bytes": e * (2 * m * k + 2 * n * k + 2 * n + r + 2 * m * n), "flops": 6 * m * n * k}   # (the residual's gradient is dy itself)
    if case["op"] == "norm":
        m, n = case["rows"], case["d"]
        return {"bytes": e * ((4 if case["train"] else 2) * m * n + (4 if case["train"] else 2) * n),
                "flops": (20 if case["train"] else 8) * m * n}
    sizes = _sizes(case)
    coded = sum(n for n in sizes if n >= MIN_8BIT) if case["bits"] == 8 else 0
    rest = sum(sizes) - coded
    # p, g read, p written; moments of 32 bits read and written; moments of 8 bits read, written, and returned as bfloat16
    return {"bytes": 3 * e * (coded + rest) + 16 * rest + (4 + 4) * coded + 16 * coded / BLOCK, "flops": 14 * (coded + rest)}
