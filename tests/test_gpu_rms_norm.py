"""``addernetcuda_amd.rms_norm`` and its 8-bit form against the formula in 64 bits, with bounds that follow from the roundings (tests/block_bounds.py)."""
import pytest
import torch
import torch.nn.functional as F

from tests import block_bounds as B
from tests.layer_bounds import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
EPS = 1e-6
# a value, lanes' and waves' borders, widths that no chunk divides, rows that are read again; few and many rows
SIZES = [(1, 1), (3, 7), (1, 128), (5, 129), (9, 136), (70, 256), (33, 515), (1030, 64), (257, 1024), (1, 4096), (300, 2048), (40, 4100), (7, 8192), (3, 16384), (2, 16385),
         (5, 20001), (3001, 24)]


def make(rows, d, dtype, weight=None, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * rows + d)
    t = lambda *s, scale=1.0, mean=0.0: (torch.randn(*s, generator=g) * scale + mean).cuda()
    return t(rows, d).to(dtype), t(d, scale=0.2, mean=1.0).to(weight or dtype), t(rows, d, scale=2.0).to(dtype), t(rows, d).to(dtype), t(rows, d).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,d", SIZES)
def test_sizes(rows, d, dtype, gpu):
    from addernetcuda_amd.rms_norm import rms_norm
    x, w, r, dy, ds = make(rows, d, dtype)
    want = B.rms_norm(x, w, r, dy, ds, EPS)
    with torch.no_grad():
        y, s = rms_norm(x, w, EPS, residual=r)
        within(y, want["y"], "y"), within(s, want["sum"], "sum")
        within(rms_norm(x, w, EPS), B.rms_norm(x, w, None, None, None, EPS)["y"], "y alone")
        within(rms_norm(x, None, EPS), B.rms_norm(x, None, None, None, None, EPS)["y"], "y without weight")
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    y, s = rms_norm(*leaves[:2], EPS, residual=r)
    within(y, want["y"], "y"), within(s, want["sum"], "sum")
    gx, gw, gr = torch.autograd.grad((y, s), leaves, (dy, ds))
    within(gx, want["gx"], "gx"), within(gw, want["gw"], "gw")
    assert torch.equal(gx, gr) and gx.dtype == dtype
    want = B.rms_norm(x, w, None, dy, None, EPS)
    gx, gw = torch.autograd.grad(rms_norm(x, w, EPS), (x, w), dy)
    within(gx, want["gx"], "gx alone"), within(gw, want["gw"], "gw alone")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,d", SIZES)
def test_codes(rows, d, dtype, gpu):
    from addernetcuda_amd.fp8 import rms_norm_fp8
    x, w, r, _, _ = make(rows, d, dtype)
    for residual in (None, r):
        want = B.rms_norm(x, w, residual, None, None, EPS)
        value, off = want["y"]
        off = off - (2.0 ** -8 if dtype == torch.bfloat16 else 0) * value.abs()   # (not rounded to the type)
        got = rms_norm_fp8(x, w, EPS, residual=residual)
        B.check_codes(got[0], got[1], value, off)
        if residual is not None:
            within(got[2], want["sum"], "sum")


def test_layouts_and_broadcast(gpu):
    """Rows with gaps, bases off any alignment, leading dimensions, an expanded gradient, a shortcut that is broadcast, a float32 weight beside bfloat16."""
    from addernetcuda_amd.rms_norm import RMSNorm, rms_norm
    for dtype in DTYPES:
        x, w, r, dy, ds = make(30, 100, dtype, weight=torch.float32)

        def gap(t):
            big = torch.full((t.shape[0] * (t.shape[1] + 5) + 1,), float("nan"), dtype=dtype, device="cuda")
            v = big[1:].view(t.shape[0], t.shape[1] + 5)[:, :t.shape[1]]
            v.copy_(t)
            return v

        want = B.rms_norm(x, w, r, dy, ds, EPS)
        for lay in (gap, lambda t: t.t().contiguous().t()):
            a, b, c = lay(x).detach().requires_grad_(True), w.clone().requires_grad_(True), lay(r).detach().requires_grad_(True)
            y, s = rms_norm(a, b, EPS, residual=c)
            within(y, want["y"], "y"), within(s, want["sum"], "sum")
            gx, gw, gr = torch.autograd.grad((y, s), (a, b, c), (lay(dy), lay(ds)))
            within(gx, want["gx"], "gx"), within(gw, want["gw"], "gw")
            assert gw.dtype == torch.float32
        row = r[0].clone().requires_grad_(True)
        a = x.view(5, 6, 100).detach().requires_grad_(True)
        y, s = rms_norm(a, w, EPS, residual=row)
        gx, gr = torch.autograd.grad(y.float().sum(), (a, row))
        want = B.rms_norm(x, w, row.detach().expand(30, 100), torch.ones_like(dy), None, EPS)
        within(y.view(30, 100), want["y"], "y"), within(gx.view(30, 100), want["gx"], "gx")
        value, off = want["gx"]
        last = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
        within(gr, (value.sum(0), off.sum(0) + 32 * last * value.abs().sum(0)), "the broadcast shortcut's gradient")
        only = torch.autograd.grad(rms_norm(a, w, EPS, residual=row)[1].float().sum(), row)[0]   # (the sum alone)
        assert torch.equal(only, torch.full_like(row, 30))
    norm = RMSNorm(100).cuda()
    torch.nn.RMSNorm(100, eps=1e-6).load_state_dict(norm.state_dict())   # the same names
    assert torch.equal(norm(x.float()), rms_norm(x.float(), norm.weight, 1e-6))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_empty_rows_of_zeros_and_what_is_no_number(dtype, gpu):
    from addernetcuda_amd.fp8 import rms_norm_fp8, values
    from addernetcuda_amd.rms_norm import rms_norm
    x, w, r, dy, _ = make(6, 300, dtype)
    none = x[:0].requires_grad_(True)
    y, s = rms_norm(none, w, EPS, residual=none)
    assert y.shape == s.shape == (0, 300)
    gx, gw = torch.autograd.grad(rms_norm(none, w.requires_grad_(True), EPS).sum(), (none, w))
    assert gx.shape == (0, 300) and not gw.any()
    q, scale = rms_norm_fp8(none.detach(), None)
    assert q.shape == (0, 300) and scale.shape == (0, 3)
    x = x.detach().clone()
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    with torch.no_grad():
        y = rms_norm(x, None, EPS)
        assert not y[1].any() and torch.isnan(y[2]).all() and not y[3, :7].any() and torch.isnan(y[3, 7])
        within(y[4:], B.rms_norm(x[4:], None, None, None, None, EPS)["y"], "the rows beside them")
        q, scale = rms_norm_fp8(x, None)
        assert not q[1].float().any() and float(scale[1].max()) == float(torch.tensor(2.0 ** -100) / 448)
        assert torch.isnan(values(q, scale)[2]).all() and torch.isfinite(values(q, scale)[4:]).all()


def test_streams_graphs_autocast_and_gradients_of_gradients(gpu):
    from addernetcuda_amd.rms_norm import rms_norm
    x, w, r, dy, ds = make(64, 512, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a, b, c = (t.clone().requires_grad_(True) for t in (x, w, r))

    def run():
        y, s = rms_norm(a, b, EPS, residual=c)
        return (y, s, *torch.autograd.grad((y, s), (a, b, c), (dy, ds)))

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
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert rms_norm(x, w).dtype == F.rms_norm(x, (512,), w).dtype == torch.bfloat16
        assert rms_norm(x, w.float()).dtype == rms_norm(x, w).dtype
        y, s = rms_norm(x, w, residual=r.float())   # (types that meet in the wider)
        assert torch.equal(s, x.float() + r.float()) and y.dtype == torch.float32
        assert all(torch.equal(p, q) for p, q in zip((y, s), rms_norm(x.float(), w.float(), residual=r.float())))
    y = rms_norm(a, b)
    g = torch.autograd.grad(y.float().square().sum(), a, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.float().sum().backward()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_the_module_without_eps(gpu, dtype):
    """``eps=None`` is nn.RMSNorm's: of the type that the norm computes in.  Values of 2^-10 or so, whose mean square is some eight of it."""
    from addernetcuda_amd.fp8 import RMSNormFp8, values
    from addernetcuda_amd.rms_norm import RMSNorm
    x = (make(16, 256, torch.float32)[0] * 2.0 ** -10).to(dtype)
    norm = RMSNorm(256, eps=None, device=x.device, dtype=dtype)
    want = B.rms_norm(x, None, None, None, None, torch.finfo(torch.float32).eps)["y"]
    half = torch.finfo(dtype).eps / 2   # (float16 goes through torch's operators, which round the root and the product, and the weight's)
    y = norm(x).detach().double()
    assert ((y - want[0].to(y.device)).abs() <= (4 * half + 1e-5) * want[0].to(y.device).abs() + 1e-7).all()
    if dtype != torch.float16:
        q, scale = RMSNormFp8(norm)(x)
        v = values(q, scale).double()
        assert ((v - want[0].to(v.device)).abs() <= want[0].to(v.device).abs() * (2.0 ** -4 + 2 * half + 1e-5) + scale.max() * 2.0 ** -10).all()


def test_refusals(gpu):
    from addernetcuda_amd.fp8 import rms_norm_fp8
    from addernetcuda_amd.rms_norm import RMSNorm, rms_norm
    x, w, r, _, _ = make(4, 24, torch.float32)
    for bad in (dict(weight=w[:5]), dict(weight=w.bfloat16()), dict(eps=-1.0), dict(residual=r[:, :5]), dict(residual=r.bfloat16()), dict(weight=w.cpu()), dict(residual=r.cpu())):
        with pytest.raises(RuntimeError):
            rms_norm(x, **bad)
        with pytest.raises(RuntimeError):
            rms_norm_fp8(x, **bad)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_fp8(x.requires_grad_(True))
    with pytest.raises(RuntimeError):
        RMSNorm(25).cuda()(x)


def test_gradient_against_differences(gpu):
    """The kernels' gradients beside the differences of the formula in 64 bits."""
    from addernetcuda_amd.rms_norm import rms_norm
    x, w, r, dy, ds = make(4, 30, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, r)]
    grads = torch.autograd.grad(rms_norm(*leaves[:2], EPS, residual=r), leaves, (dy, ds))
    values = [t.detach().double().cpu() for t in leaves]

    def of(v):
        out = B.rms_norm(*v, None, None, EPS)
        return float((out["y"][0] * dy.double().cpu()).sum() + (out["sum"][0] * ds.double().cpu()).sum())

    for k, at in ((0, (2, 3)), (0, (0, 29)), (1, (4,)), (2, (3, 7))):
        lo, hi = ([t.clone() for t in values] for _ in range(2))
        lo[k][at] -= 1e-5
        hi[k][at] += 1e-5
        assert abs((of(hi) - of(lo)) / 2e-5 - float(grads[k][at])) < 1e-5 * (1 + abs(float(grads[k][at])))
