"""``addernetcuda_amd.layer_norm`` against the formula in 64 bits, with bounds that follow from the roundings (tests/layer_bounds.py)."""
import pytest
import torch

from tests import layer_bounds as B

pytestmark = pytest.mark.gpu
KINDS = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)]
IDS = ["f32", "bf16", "bf16_f32"]
EPS = 1e-5


def make(rows, d, kind, mean=0.5):
    g = torch.Generator().manual_seed(13 * rows + d)
    t = lambda dtype, *s, scale=1.0, off=0.0: (torch.randn(*s, generator=g) * scale + off).to(dtype).cuda()
    return t(kind[0], rows, d, off=mean), t(kind[1], d, scale=0.2, off=1.0), t(kind[1], d, scale=0.2), t(kind[0], rows, d)


def check(x, w, b, dy, eps=EPS, want=None):
    from addernetcuda_amd.layer_norm import layer_norm
    want = want or B.layer_norm(x, w, b, dy, eps)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b) if t is not None]
    full = iter(leaves)
    args = [next(full) if t is not None else None for t in (x, w, b)]
    with torch.no_grad():
        B.within(layer_norm(*args, eps), want["y"], "y without gradients")
    y = layer_norm(*args, eps)
    B.within(y, want["y"], "y")
    names = ["gx"] + (["gw"] if w is not None else []) + (["gb"] if b is not None else [])
    for name, leaf, t in zip(names, leaves, torch.autograd.grad(y, leaves, dy)):
        assert t.dtype == leaf.dtype
        B.within(t, want[name], name)


# widths at and beside what 8, 16, ... 1024 lanes of 16 values hold, and wider; rows that fill no workgroup, and many
@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 512), (2, 3), (3, 8), (5, 127), (64, 128), (7, 129), (200, 256), (33, 257), (10, 512),
                                    (9, 777), (100, 1024), (21, 1025), (40, 2048), (3, 2049), (6, 4096), (5, 4100), (4, 8191), (3, 8193),
                                    (2, 16384), (3, 16385), (70, 20000), (5000, 64), (3001, 40), (2100, 777)])
def test_sizes(rows, d, kind, gpu):
    check(*make(rows, d, kind))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("d", [48, 520, 3000])
def test_without_weight_or_bias(d, kind, gpu):
    x, w, b, dy = make(19, d, kind)
    check(x, None, None, dy)
    check(x, w, None, dy)
    check(x, None, b, dy)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("rows,d", [(7, 40), (130, 515), (6, 2500), (3, 17000)])
def test_layouts(rows, d, kind, gpu):
    """Rows with gaps that hold NaN and start off any alignment, columns side by side, leading dimensions, several normalised ones."""
    from addernetcuda_amd.layer_norm import layer_norm, LayerNorm
    x, w, b, dy = make(rows, d, kind)

    def gap(t):
        big = torch.full((t.shape[0] * (t.shape[1] + 3) + 1,), float("nan"), dtype=t.dtype, device="cuda")
        v = big[1:].view(t.shape[0], t.shape[1] + 3)[:, :t.shape[1]]
        v.copy_(t)
        return v

    want = B.layer_norm(x, w, b, dy, EPS)
    check(gap(x), gap(w[None])[0], gap(b[None])[0], gap(dy), want=want)
    check(x.t().contiguous().t(), w, b, dy.t().contiguous().t(), want=want)
    leaf = x.clone().requires_grad_(True)   # a gradient that is one number expanded
    gx = torch.autograd.grad(layer_norm(leaf, w, b, EPS).sum(), leaf)[0]
    B.within(gx, B.layer_norm(x, w, b, torch.ones_like(dy), EPS)["gx"], "gx of a sum")
    x4 = x.view(rows, 1, d).expand(rows, 2, d)
    assert torch.equal(layer_norm(x4, w, b, EPS)[:, 1], layer_norm(x, w, b, EPS))
    if d % 5 == 0:
        m = LayerNorm((5, d // 5)).cuda()
        with torch.no_grad():
            m.weight.copy_(w.view(5, -1))
            m.bias.copy_(b.view(5, -1))
        if kind[1] == torch.float32:
            B.within(m(x.view(rows, 5, d // 5)).view(rows, d), want["y"], "two normalised dimensions")
        torch.nn.LayerNorm((5, d // 5)).load_state_dict(m.state_dict())


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_rows_that_do_not_vary_or_are_not_numbers(kind, gpu):
    """A constant row normalises to the bias; one with an infinite value or one that is none becomes NaN; neither touches its
    neighbours; a mean far larger than the spread loses nothing to it (float32)."""
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, _ = make(12, 264, kind)
    clean = layer_norm(x, w, b, EPS)
    x[2], x[5, 7], x[9, 263] = 3.0, float("inf"), float("nan")
    y = layer_norm(x, w, b, EPS)
    assert torch.equal(y[2], b.to(y.dtype)) and torch.isnan(y[5]).all() and torch.isnan(y[9]).all()
    rest = [0, 1, 3, 4, 6, 7, 8, 10, 11]
    assert torch.equal(y[rest], clean[rest])
    if kind[0] == torch.float32:
        check(*make(20, 1000, kind, mean=1000.0))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_rows_that_do_not_exist_and_single_gradients(kind, gpu):
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, dy = make(30, 72, kind)
    none = x[:0].requires_grad_(True)
    for t in (w, b):
        t.requires_grad_(True)
    gx, gw, gb = torch.autograd.grad(layer_norm(none, w, b).sum(), (none, w, b))
    assert gx.shape == (0, 72) and not gw.any() and not gb.any()
    want = B.layer_norm(x, w, b, dy, EPS)
    leaf = x.clone().requires_grad_(True)
    for name, t in (("gx", leaf), ("gw", w), ("gb", b)):
        B.within(torch.autograd.grad(layer_norm(leaf, w, b, EPS), t, dy)[0], want[name], name)
    B.within(torch.autograd.grad(layer_norm(leaf, w.detach(), b.detach(), EPS), leaf, dy)[0], want["gx"], "gx alone")


def test_gradients_against_differences(gpu):
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, dy = make(64, 200, KINDS[0])
    args = [t.requires_grad_(True) for t in (x, w, b)]
    f = lambda *t: (layer_norm(*t).double() * dy.double()).sum().item()
    grads = torch.autograd.grad(layer_norm(*args), args, dy)
    with torch.no_grad():
        for i, g in enumerate(grads):
            size = g.norm().item()
            d = g / size
            e = 0.02 * args[i].norm().item() / args[i].numel() ** 0.5
            up, down = ([a + s * e * d if j == i else a for j, a in enumerate(args)] for s in (1, -1))
            assert abs((f(*up) - f(*down)) / (2 * e) - size) <= 5e-3 * size


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_second_derivatives_are_an_error_and_vmap_works(kind, gpu):
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, _ = make(6, 40, kind)
    x.requires_grad_(True)
    gx, = torch.autograd.grad(layer_norm(x, w, b).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        gx.sum().backward()
    if kind[0] == torch.float32:
        assert torch.allclose(torch.func.vmap(lambda t: layer_norm(t, w, b))(x.detach()), layer_norm(x.detach(), w, b), atol=1e-5)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
def test_same_bits_every_time_and_on_other_streams(kind, gpu):
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, dy = make(3000, 264, kind)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def once():
        y = layer_norm(x, w, b)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(first, second):
        assert torch.equal(p, q)


def test_more_than_two_to_the_31_values(gpu):
    from addernetcuda_amd.layer_norm import layer_norm
    rows, d = (1 << 21) + 3, 1032
    x = torch.ones(rows, d, dtype=torch.bfloat16, device="cuda")
    x[-4:] = torch.randn(4, d, device="cuda").to(torch.bfloat16)
    _, w, b, _ = make(1, d, KINDS[1])
    x.requires_grad_(True)
    y = layer_norm(x, w, b)
    want = B.layer_norm(x[-4:], w, b, torch.ones(4, d, dtype=torch.bfloat16), EPS)
    B.within(y[-4:], want["y"], "last rows")
    assert torch.equal(y[:1000], b.expand(1000, d))
    B.within(torch.autograd.grad(y, x, torch.ones_like(y))[0][-4:], want["gx"], "last rows' gradient")


def test_refusals(gpu):
    from addernetcuda_amd.layer_norm import layer_norm, LayerNorm
    x, w, b, _ = make(4, 24, KINDS[0])
    with pytest.raises(RuntimeError, match="the last dimensions are to be"):
        layer_norm(x, w[:20])
    with pytest.raises(RuntimeError, match="bias must have shape"):
        layer_norm(x, w, b[:20])
    with pytest.raises(RuntimeError, match="must have the type of x"):
        layer_norm(x, w.bfloat16())
    with pytest.raises(RuntimeError, match="must have the type of x"):
        layer_norm(x.bfloat16(), w, b.bfloat16())
    with pytest.raises(RuntimeError, match="same device"):
        layer_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="eps must not be negative"):
        layer_norm(x, w, b, -1e-5)
    with pytest.raises(RuntimeError, match="the last dimension"):
        LayerNorm(20, elementwise_affine=False).cuda()(x)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("a,d", [(3, 40), (7, 65), (5, 4000)])
def test_all_dimensions_normalised_of_matrices_with_gaps(a, d, kind, gpu):
    """A matrix that is one row as a whole, where its lines do not follow each other: with gaps of NaN, with columns side by side, one line
    expanded; as input and as gradient."""
    from addernetcuda_amd.layer_norm import layer_norm, LayerNorm
    x, w, b, dy = make(1, a * d, kind)
    want = B.layer_norm(x, w, b, dy, EPS)
    w, b = w.view(a, d), b.view(a, d)

    def gap(t):
        big = torch.full((a, d + 3), float("nan"), dtype=t.dtype, device="cuda")
        big[:, :d] = t
        return big[:, :d]

    for lay in (gap, lambda t: t.t().contiguous().t()):
        leaves = [lay(x.view(a, d)).detach().requires_grad_(True), w.detach().requires_grad_(True), b.detach().requires_grad_(True)]
        y = layer_norm(*leaves, EPS)
        B.within(y.reshape(1, -1), want["y"], "y")
        for name, t in zip(("gx", "gw", "gb"), torch.autograd.grad(y, leaves, lay(dy.view(a, d)))):
            B.within(t.reshape(want[name][0].shape), want[name], name)
    line = x[:, :d].expand(a, d)
    assert torch.equal(layer_norm(line, w, b, EPS), layer_norm(line.contiguous(), w, b, EPS))
    leaf = x.view(a, d).clone().requires_grad_(True)   # a gradient that is one number expanded
    gx, = torch.autograd.grad(layer_norm(leaf, w, b, EPS).sum(), leaf)
    B.within(gx.view(1, -1), B.layer_norm(x, w.flatten(), b.flatten(), torch.ones_like(dy), EPS)["gx"], "gx of a sum")
    plain = LayerNorm((a, d), elementwise_affine=False)
    assert torch.equal(plain(gap(x.view(a, d))), plain(x.view(a, d)))


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("d", [8, 264, 1032, 4100, 17000])
def test_over_the_whole_range(d, kind, gpu):
    """Where the squares of the differences leave a float's range the variance is infinite: the row is its bias, its gradient zero (and what the
    others' are without it).  Below that, and where the differences' squares vanish beside eps, as the formula has it.  One value that is not
    finite makes a row not a number, at any size."""
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b, dy = make(16, d, kind)
    far = torch.tensor([3e20, 1e24, 1e28, 1e29, 1e30, 1e32, 1e33, 2e33], device="cuda")[:, None]
    x[:8] = ((x[:8].float() + 3) * far).to(x.dtype)
    x[8:10] = (x[8:10].float() * 2.0 ** 48).to(x.dtype)   # squares of 2^96 and their sums
    x[10:12] = (x[10:12].float() * 2.0 ** -80).to(x.dtype)
    x[12], x[13] = 1e33, -3e28   # constant
    x[14], x[14, 1], x[15], x[15, d - 1] = 1e30, float("inf"), -1e33, float("nan")
    leaf = x.detach().requires_grad_(True)
    y = layer_norm(leaf, w, b, EPS)
    gx, = torch.autograd.grad(y, leaf, dy)
    assert torch.equal(y[:8], b.to(y.dtype).expand(8, d)) and not gx[:8].any()
    assert torch.equal(y[12:14], b.to(y.dtype).expand(2, d))
    assert torch.isnan(y[14:]).all()
    want = B.layer_norm(x[8:12], w, b, dy[8:12], EPS)
    B.within(y[8:12], want["y"], "y")
    B.within(gx[8:12], want["gx"], "gx")


@pytest.mark.parametrize("affine", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("within_type", [torch.bfloat16, torch.float16])
def test_autocast_as_torchs(within_type, dtype, affine, gpu):
    """In place of nn.LayerNorm: float32 out of whatever goes in, gradients of the inputs' own types."""
    from addernetcuda_amd.layer_norm import LayerNorm
    x, w, b, dy = make(33, 264, KINDS[0])
    x = x.to(dtype)
    mine, theirs = (kind(264, elementwise_affine=affine).cuda() for kind in (LayerNorm, torch.nn.LayerNorm))
    if affine:
        for m in (mine, theirs):
            m.weight.data.copy_(w)
            m.bias.data.copy_(b)
    outs = []
    for m in (mine, theirs):
        leaf = x.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=within_type):
            y = m(leaf)
        outs.append([y, *torch.autograd.grad(y, [leaf, *m.parameters()], dy)])
    for p, q in zip(*outs):
        assert p.dtype == q.dtype
    want = B.layer_norm(x.float(), w if affine else None, b if affine else None, dy, EPS)
    assert outs[0][0].dtype == torch.float32
    B.within(outs[0][0], want["y"], "y")
    value, off = want["gx"]
    B.within(outs[0][1], (value, off + (value.abs() * B.V + 2.0 ** -25 if dtype != torch.float32 else 0)), "gx")
    for name, t in zip(("gw", "gb"), outs[0][2:]):
        B.within(t, want[name], name)
