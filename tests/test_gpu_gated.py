"""``addernetcuda_amd.gated`` against the formula in 64 bits, with bounds that follow from the roundings (tests/block_bounds.py)."""
import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
ACTS = ["none", "relu", "gelu", "silu"]


def make(rows, k, h, dtype, seed=0, bias=True, scale=1.0):
    g = torch.Generator().manual_seed(seed + 31 * rows + 7 * k + h)
    t = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()
    return t(rows, k, scale=scale), t(2 * h, k, scale=k ** -0.5), t(2 * h, scale=0.3 * scale) if bias else None, t(rows, h)


def check(rows, k, h, dtype, act, **kw):
    from addernetcuda_amd.gated import gated_linear
    x, w, b, dy = make(rows, k, h, dtype, **kw)
    want = B.gated_linear(x, w, b, dy, act)
    with torch.no_grad():
        within(gated_linear(x, w, b, act), want["y"], "y without gradients")
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    y = gated_linear(x, w, b, act)
    within(y, want["y"], "y")
    for name, t in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, dy)):
        assert t.dtype == dtype
        within(t, want[name], name)


# one row up to many, widths below, at and beside the tiles' and chunks' sides, products split over k
SIZES = [(1, 1, 1), (1, 8, 8), (1, 64, 16), (2, 7, 5), (3, 65, 33), (1, 4096, 256), (5, 1000, 130), (16, 512, 512), (17, 129, 100), (33, 96, 1), (64, 64, 64), (65, 72, 80),
         (100, 1, 70), (128, 512, 272), (129, 520, 264), (130, 63, 257), (200, 2048, 40), (256, 128, 384), (300, 515, 127), (1031, 33, 129), (2000, 264, 520), (4099, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,h", SIZES)
def test_sizes(rows, k, h, dtype, gpu):
    check(rows, k, h, dtype, ACTS[(rows + k + h) % 4], bias=bool((rows + h) % 2))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ACTS)
def test_activations(act, dtype, gpu):
    for bias in (False, True):
        check(37, 130, 75, dtype, act, bias=bias)
        check(260, 264, 136, dtype, act, bias=bias)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_large(dtype, gpu):
    check(1024, 1024, 2048, dtype, "silu", bias=False)
    check(2500, 1032, 1000, dtype, "gelu")


@pytest.mark.parametrize("scale", [1e-6, 3e5])
def test_values_outside_a_halfs_range(scale, gpu):
    """What is kept for the backward in 16 bits holds for sums that are all small, or too large for a half."""
    for act in ("relu", "silu", "none"):
        check(70, 64, 72, torch.bfloat16, act, scale=scale)


# Each kernel that the forward's product can take -- type, family (1 for few rows, 2 streamed, 3 staged), shape, with shares of k or without, as
# adder_gated_kernel numbers them for a call that keeps what the backward needs -- and a size that takes it
F32, BF16 = DTYPES
KERNELS = {(F32, 1, 1, False): (7, 130, 70), (F32, 1, 2, False): (19, 133, 40), (F32, 1, 4, False): (40, 40, 70), (F32, 3, 0, False): (194, 16, 12304),
           (F32, 3, 0, True): (69, 850, 8194), (F32, 3, 1, False): (17, 16, 14), (F32, 3, 1, True): (33, 544, 16), (F32, 3, 2, False): (67, 33, 13218),
           (F32, 3, 2, True): (68, 715, 4227), (F32, 3, 3, False): (18, 544, 6160), (F32, 3, 3, True): (7, 6681, 516), (BF16, 1, 1, False): (2, 270, 13),
           (BF16, 1, 2, False): (19, 65, 10), (BF16, 1, 4, False): (33, 65, 9), (BF16, 2, 0, False): (265, 16, 13232), (BF16, 2, 0, True): (17309, 5888, 124),
           (BF16, 2, 1, False): (132, 16, 11648), (BF16, 2, 1, True): (65, 3320, 4421), (BF16, 2, 2, False): (17384, 16, 132), (BF16, 2, 2, True): (8936, 4600, 38),
           (BF16, 2, 3, False): (20, 16, 8), (BF16, 2, 3, True): (33, 1104, 9), (BF16, 3, 0, False): (196, 73, 14883), (BF16, 3, 0, True): (65, 4485, 4169),
           (BF16, 3, 1, False): (20, 14, 17), (BF16, 3, 1, True): (33, 1027, 14)}


def gated_kernel(rows, k, h, dtype, aligned, outputs=2):
    import ctypes
    from addernetcuda_amd._lib import lib
    got = ctypes.c_int()
    assert lib.adder_gated_kernel(rows, k, h, int(dtype == BF16), int(aligned), outputs, ctypes.byref(got)) == 0
    return got.value // 10000, got.value // 100 % 100, got.value % 100 > 1


@pytest.mark.parametrize("key", KERNELS, ids=str)
def test_kernels(key, gpu):
    check(*KERNELS[key], key[0], "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layouts(dtype, gpu):
    """Rows with gaps that hold NaN, bases off any alignment, transposed operands, leading dimensions, an expanded gradient."""
    from addernetcuda_amd.gated import GatedLinear, gated_linear
    x, w, b, dy = make(60, 72, 40, dtype)

    def gap(t, more=5):
        big = torch.full((t.shape[0] * (t.shape[1] + more) + 1,), float("nan"), dtype=dtype, device="cuda")
        v = big[1:].view(t.shape[0], t.shape[1] + more)[:, :t.shape[1]]
        v.copy_(t)
        return v

    want = B.gated_linear(x, w, b, dy, "gelu")
    for lay in (gap, lambda t: t.t().contiguous().t()):
        leaves = [lay(x).detach().requires_grad_(True), lay(w).detach().requires_grad_(True), gap(b[None])[0].detach().requires_grad_(True)]
        y = gated_linear(*leaves, "gelu")
        within(y, want["y"], "y")
        for name, t in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, lay(dy))):
            within(t, want[name], name)
    xs = x.view(3, 20, 72).detach().requires_grad_(True)
    y = gated_linear(xs, w, None, "silu")
    want = B.gated_linear(x, w, None, torch.ones_like(dy), "silu")
    within(y.view(60, 40), want["y"], "y")
    within(torch.autograd.grad(y.sum(), xs)[0].view(60, 72), want["gx"], "gx alone")
    none = x[:0].requires_grad_(True)
    y = gated_linear(none, w.requires_grad_(True), b)
    gx, gw = torch.autograd.grad(y.sum(), (none, w))
    assert y.shape == (0, 40) and gx.shape == (0, 72) and not gw.any()
    layer = GatedLinear(72, 40, bias=True).cuda()
    y = layer(x)
    y.float().square().sum().backward()
    assert y.dtype == dtype and layer.weight.grad.dtype == torch.float32 and layer.bias.grad.shape == (80,)
    torch.nn.Linear(72, 80).load_state_dict(layer.state_dict())   # the same names
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert layer(x).dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,h", [(3, 72, 40), (70, 130, 65), (300, 264, 264)])
def test_infinite_and_nan_stay_where_they_are(rows, k, h, dtype, gpu):
    from addernetcuda_amd.gated import gated_linear
    x, w, b, _ = make(rows, k, h, dtype)
    x, w = x.abs() + 0.5, w.abs() + 0.01
    clean = gated_linear(x, w, b)
    x[1, k - 1], x[2, 0], w[3, k // 2] = float("inf"), float("nan"), float("nan")
    y = gated_linear(x, w, b)
    assert torch.isnan(y[2]).all() and torch.isnan(y[:, 3]).all()
    keep = torch.ones(h, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert (y[1][keep] == float("inf")).all() and torch.equal(y[0][keep], clean[0][keep])


def test_graph_and_gradients_of_gradients(gpu):
    from addernetcuda_amd.gated import gated_linear
    x, w, b, dy = make(300, 264, 136, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def run():
        y = gated_linear(*leaves, "gelu")
        return (y, *torch.autograd.grad(y, leaves, dy))

    with torch.cuda.stream(side):
        eager = [t.detach().clone() for t in run()]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
    for _ in range(3):
        for t in out:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, out))
    g = torch.autograd.grad(gated_linear(x, w).float().square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.float().sum().backward()


def test_refusals(gpu):
    from addernetcuda_amd.gated import GatedLinear, gated_linear
    x, w, b, _ = make(4, 24, 16, torch.float32)
    for bad in ((x, w[:31], None), (x, w[:, :5], None), (x, w, b[:5]), (x, w.bfloat16(), None), (x, w, b.bfloat16()), (x, w.cpu(), None), (x, w[0], None)):
        with pytest.raises(RuntimeError):
            gated_linear(*bad)
    with pytest.raises(ValueError):
        gated_linear(x, w, act="tanh")
    with pytest.raises(ValueError):
        GatedLinear(4, 4, act="tanh")


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradient_against_differences(act, gpu):
    """The kernels' gradients beside the differences of the formula in 64 bits."""
    from addernetcuda_amd.gated import gated_linear
    x, w, b, dy = make(5, 12, 9, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(gated_linear(*leaves, act), leaves, dy)
    values = [t.detach().double().cpu() for t in leaves]
    of = lambda v: float((B.gated_linear(*v, None, act)["y"][0] * dy.double().cpu()).sum())
    for k, at in ((0, (2, 3)), (1, (4, 5)), (1, (13, 2)), (2, (3,)), (2, (15,))):
        lo, hi = ([t.clone() for t in values] for _ in range(2))
        lo[k][at] -= 1e-5
        hi[k][at] += 1e-5
        assert abs((of(hi) - of(lo)) / 2e-5 - float(grads[k][at])) < 1e-5 * (1 + abs(float(grads[k][at])))
