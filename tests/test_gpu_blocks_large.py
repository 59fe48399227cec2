"""Tensors of more than 2^31 values through the RMS norm, gated linear layers, 8-bit products and the loss against a teacher: the first rows and the last, whose
offsets pass 32 bits, against the formulas in 64 bits."""
import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import within

pytestmark = pytest.mark.gpu


def normal(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(*shape, device="cuda", dtype=torch.bfloat16)
    for i in range(0, shape[0], 1 << 14):   # (no float32 copy of it all)
        t[i:i + (1 << 14)] = torch.randn(min(1 << 14, shape[0] - i), *shape[1:], generator=g, device="cuda").bfloat16()
    return t


def ends(rows):
    return slice(0, 3), slice(rows - 3, rows)


def test_rms_norm(gpu):
    from addernetcuda_amd.fp8 import rms_norm_fp8
    from addernetcuda_amd.rms_norm import rms_norm
    rows, d = 300000, 8000
    x, w = normal(rows, d), normal(d, seed=1)
    dy = x.roll(1, 0)
    x.requires_grad_(True)
    y = rms_norm(x, w, 1e-6)
    gx, = torch.autograd.grad(y, x, dy)
    q, scale = rms_norm_fp8(x.detach(), w, 1e-6)
    for at in ends(rows):
        want = B.rms_norm(x[at], w, None, dy[at], None, 1e-6)
        within(y[at], want["y"], "y"), within(gx[at], want["gx"], "gx")
        B.check_codes(q[at], scale[at], want["y"][0], want["y"][1] - B.V * want["y"][0].abs())


def test_gated_linear(gpu):
    from addernetcuda_amd.gated import gated_linear
    rows, k, h = 1100000, 64, 1000   # 2.2e9 values are kept for the backward
    x, w, dy = normal(rows, k), normal(2 * h, k, seed=1), normal(rows, h, seed=2)
    x.requires_grad_(True)
    y = gated_linear(x, w * k ** -0.5)
    gx, = torch.autograd.grad(y, x, dy)
    for at in ends(rows):
        want = B.gated_linear(x[at], w * k ** -0.5, None, dy[at], "silu")
        within(y[at], want["y"], "y"), within(gx[at], want["gx"], "gx")


def test_products_of_codes(gpu):
    from addernetcuda_amd.fp8 import linear_fp8, quantize, quantize_weight
    rows, k, n = 560000, 4096, 16
    x = normal(rows // 8, k)
    q, s = quantize(x)
    q = q.view(torch.uint8).repeat(8, 1).view(torch.float8_e4m3fn)
    s = s.repeat(8, 1)
    w, ws = quantize_weight(normal(n, k, seed=1))
    y = linear_fp8(q, s, w, ws)
    for at in ends(rows):
        within(y[at], B.linear_codes(q[at], s[at], w, ws, None, None, "none", torch.bfloat16), "product")


def test_distillation(gpu):
    from addernetcuda_amd.distill import distillation_loss
    rows, c = 36000, 60001
    l = normal(rows, c)
    t, i = torch.randn(rows, 4, device="cuda"), torch.randint(0, c, (rows, 4), device="cuda")
    labels = torch.randint(0, c, (rows,), device="cuda")
    l.requires_grad_(True)
    for scale in (1.0, 2.0):
        loss = distillation_loss(l, t, i, labels, 2.0, 0.5)
        g, = torch.autograd.grad(loss * scale, l)
        for at in ends(rows):
            want = B.distillation(l[at], t[at], i[at], labels[at], 2.0, 0.5, -100)["grad"]
            within(g[at], (want[0] * 3 / rows * scale, want[1] * 3 / rows * scale), "grad")
        del g
