"""``addernetcuda_amd.fp8``: codes, their products and the layers made of them, against the formulas in 64 bits (tests/block_bounds.py)."""
import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import activation, within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]


def normal(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))) * scale


def codes(rows, k, seed=0):
    """Random codes with scales of many sizes, as a quantised tensor has them."""
    from addernetcuda_amd.fp8 import quantize
    x = normal(rows, k, seed=seed) * torch.exp(normal(rows, 1, seed=seed + 1))
    return tuple(t.cuda() for t in quantize(x))


def weight(n, k, seed=5):
    from addernetcuda_amd.fp8 import quantize_weight
    return tuple(t.cuda() for t in quantize_weight(normal(n, k, seed=seed, scale=k ** -0.5) * torch.exp(normal(n, 1, seed=seed + 1) * 0.3)))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 127), (5, 128), (17, 129), (130, 300), (1, 4096), (260, 1000), (1000, 136)])
def test_quantize(rows, d, dtype, gpu):
    from addernetcuda_amd.fp8 import quantize, quantize_weight
    x = (normal(rows, d) * torch.exp(2 * normal(rows, 1, seed=3))).to(dtype).cuda()
    x[rows // 2, : d // 2] = 0
    zero = torch.zeros(rows, d, dtype=torch.float64)
    B.check_codes(*quantize(x), x.double().cpu(), zero)
    B.check_codes(*quantize_weight(x), x.double().cpu(), zero, weight=True)
    q, s = quantize(x)
    cpu = quantize(x.cpu())   # the same arithmetic in float32
    assert torch.equal(q.cpu().view(torch.uint8), cpu[0].view(torch.uint8)) and torch.equal(s.cpu(), cpu[1])
    z = (normal(rows, 2 * d, seed=9)).to(dtype).cuda()
    for act in ("none", "relu", "gelu", "silu"):
        g, u = z.double().cpu().split(d, 1)
        a = activation(g, act)[0]
        B.check_codes(*quantize(z, gate=act), a * u, 16 * B.U * (a.abs() + g.abs()) * u.abs())


def test_quantize_of_what_is_no_number(gpu):
    from addernetcuda_amd.fp8 import quantize, values
    x = normal(4, 300).cuda()
    x[0, 5], x[1, 130], x[2, 299] = float("nan"), float("inf"), float("-inf")
    q, s = quantize(x)
    v = values(q, s)
    assert torch.isnan(v[0, 5]) and torch.isfinite(v[0, :5]).all() and torch.isfinite(v[0, 6:]).all()
    assert torch.isnan(v[1, 128:256]).all() and torch.isfinite(v[1, :128]).all() and torch.isfinite(v[1, 256:]).all()
    assert torch.isnan(v[2, 256:]).all() and torch.isfinite(v[2, :256]).all() and torch.isfinite(v[3]).all()
    tiny = torch.full((1, 128), 1e-38, device="cuda")
    q, s = quantize(tiny)
    assert not q.float().any() and float(s) == float(torch.tensor(2.0 ** -100) / 448)
    assert quantize(x[:0])[0].shape == (0, 300)


# few rows, tiles' borders, widths that no block and no load divides, shares of k
SIZES = [(1, 1, 1), (1, 128, 16), (2, 127, 130), (16, 4096, 100), (17, 1000, 33), (30, 515, 77), (33, 96, 300), (64, 2048, 129), (20, 8192, 8192),  (65, 128, 64), (70, 144, 200), (100, 1000, 257), (128, 4096, 128),
         (130, 16, 1000), (200, 333, 77), (300, 640, 640), (513, 272, 1030), (1100, 528, 2000), (2048, 1024, 1024), (2300, 512, 4200)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_products(rows, k, n, dtype, gpu):
    from addernetcuda_amd.fp8 import linear_fp8
    (x, xs), (w, ws) = codes(rows, k), weight(n, k)
    b, r = normal(n, seed=2).to(dtype).cuda(), normal(rows, n, seed=3).to(dtype).cuda()
    within(linear_fp8(x, xs, w, ws, dtype=dtype), B.linear_codes(x, xs, w, ws, None, None, "none", dtype), "product")
    act = ("relu", "gelu", "silu")[(rows + n) % 3]
    within(linear_fp8(x, xs, w, ws, b, r, act, dtype), B.linear_codes(x, xs, w, ws, b, r, act, dtype), "with everything")


# sizes of the large shapes, whose results are looked at in part
LARGE = [(4096, 1024, 4096), (8200, 300, 4100)]


def test_each_kernel_is_reached():
    """The sizes take each shape of the kernels, the streamed ones with and without shares of k."""
    import ctypes
    from addernetcuda_amd._lib import lib
    for dtype in DTYPES:
        got = set()
        for rows, k, n in SIZES + LARGE:
            v = ctypes.c_int()
            assert lib.adder_linear_codes_kernel(rows, k, n, int(dtype == torch.bfloat16), ctypes.byref(v)) == 0
            got.add((v.value // 100, v.value % 100 > 1))
        want = {101, 102, 200, 201} | ({202} if dtype == torch.bfloat16 else set())
        assert {g[0] for g in got} == want and {(201, True), (201, False), (200, False)} <= got, got


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_large(dtype, gpu):
    from addernetcuda_amd.fp8 import linear_fp8
    for rows, k, n in LARGE:
        (x, xs), (w, ws) = codes(rows, k), weight(n, k)
        r = normal(300, n, seed=3).to(dtype).cuda()
        r = torch.cat([r, r.new_zeros(rows - 600, n), r])
        got = linear_fp8(x, xs, w, ws, residual=r, dtype=dtype)
        for at in (slice(0, 300), slice(rows - 300, rows)):
            within(got[at], B.linear_codes(x[at], xs[at], w, ws, None, r[at], "none", dtype), f"rows {at}")


def test_layouts(gpu):
    """Codes in rows with gaps that are no numbers, off any alignment, one row for all; leading dimensions; a shortcut that is broadcast."""
    from addernetcuda_amd.fp8 import linear_fp8
    nan = torch.tensor(float("nan")).to(torch.float8_e4m3fn)

    def gap(t, more, off):
        big = nan.cuda().view(torch.uint8).expand(t.shape[0] * (t.shape[1] + more) + off).clone().view(torch.float8_e4m3fn)
        v = big[off:].view(t.shape[0], t.shape[1] + more)[:, :t.shape[1]]
        v.view(torch.uint8).copy_(t.view(torch.uint8))
        return v

    for rows, k, n in ((3, 200, 40), (150, 200, 70), (150, 208, 70)):
        (x, xs), (w, ws) = codes(rows, k), weight(n, k)
        want = B.linear_codes(x, xs, w, ws, None, None, "none", torch.float32)
        for more, off in ((5, 1), (8, 0), (16 - k % 16, 0), (24, 16)):
            within(linear_fp8(gap(x, more, off), xs, gap(w, more, off), ws, dtype=torch.float32), want, f"gaps of {more}")
        lead = linear_fp8(x.view(torch.uint8).view(rows // 3, 3, k).view(torch.float8_e4m3fn), xs.view(rows // 3, 3, -1), w, ws, residual=torch.ones(n, device="cuda"),
                          dtype=torch.float32)
        within(lead.reshape(rows, n) - 1, (want[0], want[1] + 2.0 ** -23 * (1 + want[0].abs())), "leading dimensions")
        one = x[:1].expand(rows, k)
        got = linear_fp8(one, xs[:1].expand(rows, -1), w, ws, dtype=torch.float32)
        assert torch.equal(got, got[:1].expand(rows, n))
    assert linear_fp8(x[:0], xs[:0], w, ws).shape == (0, n)


def test_nan_stays_in_its_row_and_column(gpu):
    from addernetcuda_amd.fp8 import linear_fp8
    for rows in (3, 300):
        (x, xs), (w, ws) = codes(rows, 272), weight(264, 272)
        clean = linear_fp8(x, xs, w, ws)
        xs = xs.clone()
        xs[1, 2] = float("nan")
        w = w.clone()
        w.view(torch.uint8)[5, 7] = 0x7F
        y = linear_fp8(x, xs, w, ws)
        assert torch.isnan(y[1]).all() and torch.isnan(y[:, 5]).all()
        keep = [c for c in range(264) if c != 5]
        assert torch.equal(y[0][keep], clean[0][keep]) and torch.equal(y[2:][:, keep], clean[2:][:, keep])


def test_graph_and_side_stream(gpu):
    from addernetcuda_amd.fp8 import linear_fp8, quantize, rms_norm_fp8
    (w, ws), x = weight(200, 300), normal(150, 300).bfloat16().cuda()
    run = lambda: (linear_fp8(*quantize(x), w, ws), linear_fp8(*rms_norm_fp8(x), w, ws))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [t.clone() for t in run()]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, out))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer(dtype, gpu):
    """A layer made from one of linear layers: its call is the product of the input's codes with the weight's."""
    from addernetcuda_amd.fp8 import LinearFp8, linear_fp8, quantize, quantize_weight
    from addernetcuda_amd.linear import LinearAct
    torch.manual_seed(3)
    layer = LinearAct(200, 130, act="gelu").cuda()
    made = LinearFp8.of(layer)
    x, r = normal(40, 200).to(dtype).cuda(), normal(40, 130, seed=1).to(dtype).cuda()
    with torch.no_grad():
        y = made(x, residual=r)
        assert y.dtype == dtype and torch.equal(y, made(quantize(x), residual=r))
        w, ws = quantize_weight(layer.weight)
        assert torch.equal(y, linear_fp8(*quantize(x), w, ws, layer.bias.to(dtype), r, "gelu", dtype))
        full = layer(x, residual=r).float()
        assert float((y.float() - full).norm() / full.norm()) < 0.06   # (codes of three bits of mantissa: each is off by a sixteenth at most)
    again = LinearFp8(200, 130, act="gelu").cuda()
    again.load_state_dict(made.state_dict())
    with torch.no_grad():
        assert torch.equal(again(x, residual=r), y)


def test_refusals(gpu):
    from addernetcuda_amd.fp8 import LinearFp8, linear_fp8, quantize, quantize_weight
    (x, xs), (w, ws) = codes(4, 200), weight(40, 200)
    b = torch.zeros(40, device="cuda", dtype=torch.bfloat16)
    for bad in ((x.float(), xs, w, ws), (x, xs[:, :1], w, ws), (x, xs, w[:, :100], ws), (x, xs, w, ws.t()), (x, xs.bfloat16(), w, ws), (x, xs, w, ws, b[:3]), (x, xs, w, ws, b.float()),
                (x, xs, w, ws, None, b[:3]), (x, xs, w.cpu(), ws), (x.cpu(), xs, w, ws), (x[0, 0], xs, w, ws)):
        with pytest.raises(RuntimeError):
            linear_fp8(*bad)
    for bad in (dict(act="tanh"), dict(dtype=torch.float16)):
        with pytest.raises(ValueError):
            linear_fp8(x, xs, w, ws, **bad)
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_fp8(x, xs, w, ws, b.clone().requires_grad_(True))
    v = torch.zeros(3, 5, device="cuda")
    with pytest.raises(RuntimeError):
        quantize(v, gate="silu")
    with pytest.raises(ValueError):
        quantize(v, gate="tanh")
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize(v.requires_grad_(True))
    with pytest.raises(RuntimeError):
        quantize_weight(v.detach()[0])
    with pytest.raises(ValueError):
        LinearFp8(4, 4, gate="tanh")
