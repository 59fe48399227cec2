"""``addernetcuda_amd.linear`` against the formula in 64 bits: every type, activation, layout and size where the kernels can go wrong,
with bounds that follow from the roundings (tests/layer_bounds.py)."""
import pytest
import torch

from tests import layer_bounds as B

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
ACTS = ["none", "relu", "gelu", "silu"]


def make(rows, k, n, dtype, seed=0, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed + 31 * rows + 7 * k + n)
    t = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).cuda()
    return (t(rows, k), t(n, k, scale=k ** -0.5), t(n, scale=0.3) if bias else None, t(rows, n) if residual else None, t(rows, n))


def check(rows, k, n, dtype, act, seed=0, bias=True, residual=True):
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = make(rows, k, n, dtype, seed, bias, residual)
    want = B.linear(x, w, b, r, dy, act)
    with torch.no_grad():
        B.within(linear_act(x, w, b, r, act), want["y"], "y without gradients")
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = linear_act(x, w, b, r, act)
    B.within(y, want["y"], "y")
    got = torch.autograd.grad(y, leaves, dy)
    names = ["gx", "gw"] + (["gb"] if bias else [])
    for name, t in zip(names, got):
        assert t.dtype == dtype
        B.within(t, want[name], name)
    if residual:
        assert torch.equal(got[-1], dy)


# one row up to many, widths below, at and beside the tiles' and chunks' sides, products that are split over k and that are not
SIZES = [(1, 1, 1), (1, 8, 8), (1, 64, 16), (2, 7, 5), (3, 65, 33), (1, 4096, 256), (5, 1000, 130), (16, 512, 512), (17, 129, 100),
         (33, 96, 1), (64, 64, 64), (65, 72, 80), (100, 1, 70), (128, 512, 512), (129, 520, 264), (130, 63, 257), (200, 2048, 40),
         (256, 128, 384), (300, 515, 127), (512, 256, 256), (1031, 33, 129), (2000, 264, 520), (4099, 40, 24)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", SIZES)
def test_sizes(rows, k, n, dtype, gpu):
    check(rows, k, n, dtype, ACTS[(rows + k + n) % 4])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_epilogues(act, bias, residual, dtype, gpu):
    check(37, 130, 75, dtype, act, bias=bias, residual=residual)
    check(2, 264, 72, dtype, act, bias=bias, residual=residual)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_large(dtype, gpu):
    check(1024, 1024, 2048, dtype, "gelu", residual=False)
    check(2500, 1032, 1000, dtype, "silu")


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(3, 40, 24), (130, 72, 136), (300, 100, 50)])
def test_layouts(rows, k, n, dtype, gpu):
    """Rows with gaps that hold NaN, bases off any alignment, transposed inputs, leading dimensions, expanded gradients and residuals."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = make(rows, k, n, dtype)
    nan = float("nan")

    def gap(t, more=5):   # the same values in rows that are `more` longer, one element off the allocation's start
        big = torch.full((t.shape[0] * (t.shape[1] + more) + 1,), nan, dtype=dtype, device="cuda")
        v = big[1:].view(t.shape[0], t.shape[1] + more)[:, :t.shape[1]]
        v.copy_(t)
        return v

    want = B.linear(x, w, b, r, dy, "gelu")
    across = lambda t: t.t().contiguous().t()
    for lay_x, lay_r, lay_dy, lay_w in [(gap, gap, gap, gap), (across, across, across, across), (gap, across, gap, across)]:
        leaves = [lay_x(x).detach().requires_grad_(True), lay_w(w).detach().requires_grad_(True), gap(b[None])[0].detach().requires_grad_(True)]
        y = linear_act(leaves[0], leaves[1], leaves[2], lay_r(r), "gelu")
        B.within(y, want["y"], "y")
        for name, t in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, lay_dy(dy))):
            B.within(t, want[name], name)
    # three leading dimensions, a residual that is broadcast, a gradient that is one number expanded
    xs = x[: rows // 3 * 3].view(3, rows // 3, k).requires_grad_(True)
    row = r[0].clone().requires_grad_(True)
    y = linear_act(xs, w, b, row, "silu")
    assert y.shape == (3, rows // 3, n)
    used = rows // 3 * 3
    want = B.linear(xs.detach().view(used, k), w, b, row.detach().expand(used, n), torch.ones(used, n, dtype=dtype), "silu")
    B.within(y.view(used, n), want["y"], "y")
    gx, gr = torch.autograd.grad(y.sum(), (xs, row))
    B.within(gx.view(used, k), want["gx"], "gx")
    assert torch.equal(gr, torch.full_like(row, used))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_rows_that_do_not_exist_and_single_gradients(dtype, gpu):
    from addernetcuda_amd.linear import linear_act, LinearAct
    x, w, b, _, _ = make(4, 24, 16, dtype)
    none = x[:0].requires_grad_(True)
    for t in (w, b):
        t.requires_grad_(True)
    y = linear_act(none, w, b, act="relu")
    assert y.shape == (0, 16)
    gx, gw, gb = torch.autograd.grad(y.sum(), (none, w, b))
    assert gx.shape == (0, 24) and not gw.any() and not gb.any()
    dy = torch.randn(4, 16, device="cuda").to(dtype)
    want = B.linear(x, w, b, None, dy, "gelu")
    for name, leaf in (("gw", w), ("gb", b)):
        y = linear_act(x, w, b, act="gelu")
        B.within(torch.autograd.grad(y, leaf, dy)[0], want[name], name)
    xr = x.clone().requires_grad_(True)
    y = linear_act(xr, w.detach(), None, act="gelu")
    B.within(torch.autograd.grad(y, xr, dy)[0], B.linear(x, w, None, None, dy, "gelu")["gx"], "gx alone")
    layer = LinearAct(24, 16, act="silu").cuda()   # float32 parameters; their gradients come back float32
    y = layer(x, residual=dy)
    y.float().square().sum().backward()
    assert layer.weight.grad.dtype == torch.float32 and layer.bias.grad.dtype == torch.float32
    ref = torch.nn.Linear(24, 16)
    ref.load_state_dict(layer.state_dict())   # the same names


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(3, 72, 40), (70, 130, 65), (300, 264, 264)])
def test_infinite_and_nan_stay_where_they_are(rows, k, n, dtype, gpu):
    """An infinite or not-a-number input reaches its own row only, and as the formula has it; so does one in the weights its column."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, _ = make(rows, k, n, dtype)
    x, w = x.abs() + 0.5, w.abs() + 0.01
    clean = linear_act(x, w, b, r)
    x[1, k - 1] = float("inf")
    x[2, 0] = float("nan")
    w[3, k // 2] = float("-inf")
    y = linear_act(x, w, b, r).float()
    assert torch.isnan(y[2]).all() and torch.isnan(y[1, 3])
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[3] = False
    assert (y[1][keep] == float("inf")).all()
    rest = [i for i in range(rows) if i not in (1, 2)]
    assert (y[rest][:, 3] == float("-inf")).all()
    assert torch.equal(y[rest][:, keep], clean.float()[rest][:, keep])


@pytest.mark.parametrize("rows,k,n", [(2, 40, 33), (200, 72, 64), (300, 300, 300)])
def test_float32_over_its_whole_range(rows, k, n, gpu):
    """Values that round up to infinity in bfloat16, products of the largest with the smallest, values whose parts lie below the smallest
    normal number: as good as in the middle of the range."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, _, dy = make(rows, k, n, torch.float32)
    for sx, sw in ((2.0 ** 100, 2.0 ** -100), (2.0 ** -60, 2.0 ** 50), (2.0 ** -115, 2.0 ** 110)):
        xs, ws, bs = x * sx, w * sw, b * (sx * sw)
        if sx > 1:
            xs[0, 0], ws[:, 0] = 3.4e38, 2.0 ** -130
        want = B.linear(xs, ws, bs, None, dy, "none")
        leaves = [t.requires_grad_(True) for t in (xs, ws, bs)]
        y = linear_act(*leaves)
        names = ("gx", "gw", "gb")
        # (what is lost below the smallest normal float, 2^-126 a term at most)
        for name, t, terms in zip(("y",) + names, (y,) + torch.autograd.grad(y, leaves, dy), (k, n, rows, rows)):
            value, off = want[name]
            size = {"y": 1, "gx": float(dy.abs().max()), "gw": float(dy.abs().max()), "gb": 1}[name]
            big = {"y": max(sx, sw), "gx": 1, "gw": 1, "gb": 1}[name]
            B.within(t, (value, off + terms * 2.0 ** -126 * max(1.0, size) * max(1.0, big) * 4), name)


def test_what_torch_does_with_calls_it_does_with_these(gpu):
    """A gradient of a gradient is an error, vmap and autocast work, a parameter that changes between forward and backward is noticed."""
    from addernetcuda_amd.linear import linear_act, LinearAct
    x, w, b, r, dy = make(6, 24, 16, torch.float32)
    x.requires_grad_(True)
    gx, = torch.autograd.grad(linear_act(x, w, b, act="gelu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gx.sum().backward()
    each = torch.func.vmap(lambda t: linear_act(t, w, b, act="silu"))(x.detach().view(3, 2, 24))
    assert torch.allclose(each.view(6, 16), linear_act(x.detach(), w, b, act="silu"), atol=1e-5)
    layer = LinearAct(24, 16, act="relu").cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert layer(x.detach().bfloat16()).dtype == torch.bfloat16
    y = layer(x)
    with torch.no_grad():
        layer.weight.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_against_differences(gpu):
    """f(t + e d) - f(t - e d) = 2 e |grad f|^2 / |grad f| along d = grad f / |grad f|; float32 sums of 2^15 outputs carry 1e-5 of
    their size at most, the step's third-order term less."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = (t.requires_grad_(True) for t in make(128, 96, 256, torch.float32))
    f = lambda *t: (linear_act(*t, act="gelu").double() * dy.double()).sum().item()
    args = [x, w, b, r]
    grads = torch.autograd.grad(linear_act(*args, act="gelu"), args, dy)
    with torch.no_grad():
        for i, g in enumerate(grads):
            size = g.norm().item()
            d = g / size
            e = 0.02 * args[i].norm().item() / args[i].numel() ** 0.5
            up, down = ([a + s * e * d if j == i else a for j, a in enumerate(args)] for s in (1, -1))
            assert abs((f(*up) - f(*down)) / (2 * e) - size) <= 5e-3 * size


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n", [(4, 512, 512), (128, 1024, 128), (1500, 264, 264)])
def test_same_bits_every_time_and_on_other_streams(rows, k, n, dtype, gpu):
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = make(rows, k, n, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        y = linear_act(x, w, b, r, "gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for a, b_ in zip(first, second):
        assert torch.equal(a, b_)


def test_more_than_two_to_the_31_values(gpu):
    from addernetcuda_amd.linear import linear_act
    rows, k, n = (1 << 22) + 3, 520, 8
    _, w, b, _, _ = make(1, k, n, torch.bfloat16)
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[-5:] = torch.randn(5, k, device="cuda").to(torch.bfloat16)
    y = linear_act(x, w, b)
    B.within(y[-5:], B.linear(x[-5:], w, b, None, None, "none")["y"], "last rows")
    assert torch.equal(y[: rows - 5], b.expand(rows - 5, n))


def test_refusals(gpu):
    from addernetcuda_amd.linear import linear_act, LinearAct
    x, w, b, r, _ = make(4, 24, 16, torch.float32)
    with pytest.raises(ValueError, match="act must be one of"):
        linear_act(x, w, act="tanh")
    with pytest.raises(ValueError, match="act must be one of"):
        LinearAct(4, 4, act="tanh")
    with pytest.raises(RuntimeError, match="expects 24 features"):
        linear_act(x[:, :23], w)
    with pytest.raises(RuntimeError, match="two dimensions"):
        linear_act(x, w[0])
    with pytest.raises(RuntimeError, match="bias must have shape"):
        linear_act(x, w, b[:3])
    with pytest.raises(RuntimeError, match="the type of x"):
        linear_act(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="same device"):
        linear_act(x, w.cpu())
    with pytest.raises(RuntimeError, match="does not broadcast"):
        linear_act(x, w, b, r[:, :5])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k,n", [(1, 5, 3), (33, 24, 17), (256, 128, 64)])
def test_relu_reads_its_own_result(gpu, rows, k, n, dtype):
    """Its gradients are those of the plain product for dy where the result is not zero: the same launches of the same numbers
    (where the result is no number, dy's; torch's does the same).  An edit of the result is noticed."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, _, dy = make(rows, k, n, dtype)
    x[0, 0] = float("nan")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    own, product = linear_act(*leaves, act="relu"), linear_act(*leaves)
    dz = torch.where(own.detach() == 0, torch.zeros_like(dy), dy)
    for g, h in zip(torch.autograd.grad(own, leaves, dy, retain_graph=True), torch.autograd.grad(product, leaves, dz)):
        assert torch.equal(g.nan_to_num(7), h.nan_to_num(7))
    own.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        own.sum().backward()


def test_autocast_as_torch_linear(gpu):
    """The product in autocast's type, a residual of another type added in the wider one, gradients of the leaves' own type; a type that
    has no kernel goes through torch."""
    from addernetcuda_amd.linear import linear_act, LinearAct
    x, w, b, r, dy = make(40, 72, 56, torch.float32)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear_act(x.requires_grad_(True), w.requires_grad_(True), b, act="gelu")
        wide = linear_act(x, w, b, r, act="gelu")
        with pytest.raises(RuntimeError, match="does not broadcast"):
            linear_act(x, w, b, r[:, :3], act="gelu")
    half = [t.detach().bfloat16() for t in (x, w, b)]
    assert y.dtype == torch.bfloat16 and torch.equal(y, linear_act(*half, act="gelu"))
    assert wide.dtype == torch.float32 and torch.equal(wide, y.float() + r)
    own = [t.requires_grad_(True) for t in half[:2]]
    want = torch.autograd.grad(linear_act(*own, half[2], act="gelu"), own, dy.bfloat16())
    for g, h in zip(torch.autograd.grad(y, (x, w), dy.bfloat16()), want):
        assert g.dtype == torch.float32 and torch.equal(g, h.float())
    layer = LinearAct(72, 56, act="silu").cuda()
    with torch.autocast("cuda", dtype=torch.float16):
        assert layer(x).dtype == torch.float16
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert layer(x).dtype == torch.bfloat16 and linear_act(x.double().detach(), w.double().detach()).dtype == torch.float64


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("rows,k,n", [(3, 24, 10), (200, 64, 136), (256, 128, 128)])
def test_derivative_far_from_zero(gpu, rows, k, n, act, dtype):
    """|z| far beyond 65504: the derivative is one or zero, and the gradients are the plain product's for dy in the rows of positive z,
    by the same launches."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, _, dy = make(rows, k, n, dtype)
    sign = torch.where(torch.arange(rows, device="cuda") % 3 == 0, -1.0, 1.0)[:, None]
    x, w = (x.float().abs().add(1) * sign * 2.0 ** 20).to(dtype), w.float().abs().add(2.0 ** -4).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(linear_act(*leaves, act=act), leaves, dy)
    want = torch.autograd.grad(linear_act(*leaves), leaves, torch.where(sign > 0, dy, torch.zeros_like(dy)))
    for g, h in zip(got, want):
        assert torch.equal(g, h)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,k,n,more", [(300, 515, 264, 5), (1000, 1027, 130, 5), (2050, 71, 72, 1), (201, 72, 136, 8), (130, 264, 257, 8)])
def test_aligned_rows_with_gaps_and_expanded_rows(rows, k, n, more, dtype, gpu):
    """Views whose rows begin at multiples of 16 bytes, of odd and even widths, with NaN between them (the last value of an odd width shares its
    word with nothing that exists); x, the gradient and the residual as one row expanded."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = make(rows, k, n, dtype)

    def gap(t):
        wide = -(-(t.shape[1] + more) // 8) * 8
        big = torch.full((t.shape[0], wide), float("nan"), dtype=dtype, device="cuda")
        big[:, :t.shape[1]] = t
        return big[:, :t.shape[1]]

    row = lambda t: t[:1].expand(t.shape[0], t.shape[1])
    for lay_x, lay_r, lay_dy in [(gap, gap, gap), (row, row, gap), (gap, gap, row), (row, gap, row)]:
        for act in ("none", "gelu"):
            xs, rs, ds = lay_x(x), lay_r(r), lay_dy(dy)
            want = B.linear(xs, w, b, rs, ds, act)
            leaves = [xs.detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)]
            y = linear_act(leaves[0], leaves[1], leaves[2], rs, act)
            B.within(y, want["y"], "y")
            for name, t in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, ds)):
                B.within(t, want[name], name)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,k,n", [(1, 24, 17), (40, 24, 16), (300, 72, 130)])
def test_relu_lets_nothing_through_where_it_is_off(rows, k, n, residual, dtype, gpu):
    """Infinite gradients, and ones that are no numbers, at zeros of the result: as if they were zero there."""
    from addernetcuda_amd.linear import linear_act
    x, w, b, r, dy = make(rows, k, n, dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear_act(*leaves, r if residual else None, "relu")
    off = linear_act(x, w, b, None, "relu").detach() == 0
    assert off.any()
    kinds = torch.tensor([float("inf"), float("-inf"), float("nan"), 3.0], device="cuda").to(dtype)
    broken = torch.where(off, kinds[torch.arange(rows * n, device="cuda").view(rows, n) % 4], dy)
    for g, h in zip(torch.autograd.grad(y, leaves, broken, retain_graph=True), torch.autograd.grad(y, leaves, torch.where(off, torch.zeros_like(dy), dy))):
        assert torch.isfinite(g).all() and torch.equal(g, h)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("n", [512, 515])
def test_values_before_the_activation_keep_eleven_bits(act, n, gpu):
    """bfloat16: the bias's gradient of two rows with opposite gradients and nearly the same z is a difference that rounding to its type hardly
    touches.  z as a half, rounded toward zero, is 2^-10 |z| + 2^-24 off, which moves the derivative by its own derivative times that (a
    tenth more for the next term); z as a bfloat16 would not stay within that.  And what the forward hands on is that half."""
    from addernetcuda_amd._lib import lib, check, ptr, stream_ptr
    from addernetcuda_amd.linear import ACTS, linear_act
    g = torch.Generator().manual_seed(n)
    x = torch.randn(1, 64, generator=g).bfloat16().repeat(2, 1)
    x[1, :4] += 0.03
    w, b = (torch.randn(n, 64, generator=g) / 16).bfloat16(), (torch.randn(n, generator=g)).bfloat16()
    dy = torch.tensor([[1.0], [-1.0]]).expand(2, n).bfloat16()
    z = (x.double() @ w.double().t() + b.double()).requires_grad_(True)
    _, slope = B.activation(z, act)
    bend, = torch.autograd.grad(slope.sum(), z)
    z, slope = z.detach(), slope.detach()
    off_z = B.terms(64) * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    moved = 1.1 * bend.abs() * (2.0 ** -10 * z.abs() + 2.0 ** -24 + off_z) + 24 * B.U * (1 + z.abs())
    value = slope[0] - slope[1]
    expected = value, moved.sum(0) + 4 * B.U + B.V * value.abs()
    leaf = b.cuda().requires_grad_(True)
    gb, = torch.autograd.grad(linear_act(x.cuda(), w.cuda(), leaf, act=act), leaf, dy.cuda())
    B.within(gb, expected, "gb")
    short = B.activation(z.bfloat16().double(), act)[1]
    with pytest.raises(AssertionError, match="further off"):
        B.within((short[0] - short[1]).float(), expected, "gb from z in bfloat16")
    xs, ws, bs = x.cuda(), w.cuda(), b.cuda()
    y, pre = torch.empty(2, n, dtype=torch.bfloat16, device="cuda"), torch.empty(2, n, dtype=torch.float16, device="cuda")
    check(lib.adder_linear_fwd(ptr(xs), 64, ptr(ws), ptr(bs), None, 0, ptr(y), ptr(pre), ACTS[act], 2, 64, n, 1, None, 0, stream_ptr(xs.device)), "adder_linear_fwd")
    assert ((pre.double().cpu() - z).abs() <= 2.0 ** -10 * z.abs() + 2.0 ** -24 + off_z).all()
