"""Every compiled shape of the linear layers' product kernels (tests/linear_shapes.py) against products in 64 bits: operands as rows with NaN between
them, results with the epilogue and, for what keeps values for the backward, the second output's gradients.  A sum of K products in some order is off
by (2 sqrt(K) + 8) 2^-24 of the sum of their sizes, and rounded once more to its type (tests/layer_bounds.py)."""

import pytest
import torch

from tests.layer_bounds import U, V, activation, terms
from tests.linear_shapes import BF16, FWD, GX, GW, SHAPES, STREAM, linear_kernel

pytestmark = pytest.mark.gpu


def near(actual, value, off, what):
    far = (actual.double() - value).abs()
    bad = ~(far <= off + 1e-30)
    if bad.any():
        at = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} further off than the roundings allow; first at {at}: "
                             f"{actual[at].item()} instead of {value[at].item()}, {off[at].item():.3e} allowed")


def with_gaps(t, aligned):
    """The values of t in longer rows with NaN behind them: whole multiples of 16 bytes, or one element beside any."""
    more = -t.shape[1] % 8 + 8 if aligned else 3
    big = torch.full((t.shape[0] * (t.shape[1] + more) + 1,), float("nan"), dtype=t.dtype, device="cuda")[0 if aligned else 1:]
    v = big[:t.shape[0] * (t.shape[1] + more)].view(t.shape[0], -1)[:, :t.shape[1]]
    return v.copy_(t)


def aligned(t):
    return t.data_ptr() % 16 == 0 and t.stride(0) * t.element_size() % 16 == 0


@pytest.mark.parametrize("key", SHAPES, ids=str)
def test_products(key, gpu):
    from addernetcuda_amd.linear import linear_act
    kind, product, family, shape, shared = key
    rows, k, n = SHAPES[key]
    dtype, last = (torch.bfloat16, V) if kind == BF16 else (torch.float32, U)
    g = torch.Generator(device="cuda").manual_seed(rows + k + n)
    t = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)
    x, w, dy = t(rows, k), t(n, k, scale=k ** -0.5), t(rows, n)
    stream = family == STREAM
    x, dy = with_gaps(x, stream), with_gaps(dy, stream)
    b, r = t(n, scale=0.3), with_gaps(t(rows, n), stream)
    a, c, K = {FWD: (x, w, k), GX: (dy, w, n), GW: (dy, x, rows)}[product]
    got = linear_kernel(rows, k, n, product, kind, aligned(a) and aligned(c))
    assert got[:2] == (family, shape) and (got[2] > 1) == shared
    x64, w64, dy64 = x.double(), w.double(), dy.double()
    if product == FWD:
        z, size = x64 @ w64.t() + b.double(), x64.abs() @ w64.abs().t() + b.double().abs()
        for act in ("none", "gelu"):
            y, _ = activation(z, act)
            off = 1.13 * terms(k) * size + 16 * U * (y.abs() + z.abs())
            y = y + r.double()
            off += (U + last) * y.abs()
            with torch.no_grad():
                near(linear_act(x, w, b, r, act), y, off, act)
            if act != "none":   # (with a second output)
                near(linear_act(x, w, b.clone().requires_grad_(True), r, act).detach(), y, off, act + " with its second output")
    elif product == GX:
        leaf = x.detach().requires_grad_(True)
        got, = torch.autograd.grad(linear_act(leaf, w), leaf, dy)
        value = dy64 @ w64
        near(got, value, terms(K) * (dy64.abs() @ w64.abs()) + last * value.abs(), "gx")
    else:
        leaf = w.detach().requires_grad_(True)
        got, = torch.autograd.grad(linear_act(x, leaf), leaf, dy)
        value = dy64.t().contiguous() @ x64
        near(got, value, terms(K) * (dy64.t().abs().contiguous() @ x64.abs()) + last * value.abs(), "gw")
