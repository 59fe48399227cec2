"""``addernetcuda_amd.distill`` against the formula in 64 bits, with bounds that follow from the roundings (tests/block_bounds.py)."""
import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import within

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]
IDS = ["f32", "bf16"]
INF = float("inf")


def make(rows, c, k, dtype, seed=0, labels=True, spread=2.0):
    g = torch.Generator().manual_seed(seed + 31 * rows + 7 * c + k)
    teacher = torch.randn(rows, c, generator=g) * spread
    t, i = teacher.topk(k, 1)
    l = 0.5 * teacher + torch.randn(rows, c, generator=g) * spread / 2
    y = torch.randint(0, c, (rows,), generator=g)
    y[1::7] = -100
    return l.to(dtype).cuda(), t.to(dtype).cuda(), i.cuda(), y.cuda() if labels else None


def check(l, t, i, y, T=2.0, alpha=0.7, scale=1.0):
    from addernetcuda_amd.distill import distillation_loss
    want = B.distillation(l, t, i, y, T, alpha, -100)
    with torch.no_grad():
        within(distillation_loss(l, t, i, y, T, alpha), want["loss"], "loss without gradient")
    l = l.detach().requires_grad_(True)
    loss = distillation_loss(l, t, i, y, T, alpha)
    assert loss.dtype == torch.float32 and loss.shape == ()
    within(loss, want["loss"], "loss")
    (loss * scale).backward()
    value, off = want["grad"]
    within(l.grad, (value * scale, off * abs(scale)), "grad")
    return l.grad


# classes at the borders of a wave's, a workgroup's and a piece's; rows few and many, so that a row is one workgroup's or several's
SIZES = [(1, 1, 1), (2, 2, 1), (5, 10, 3), (64, 100, 100), (3, 257, 64), (300, 256, 5), (33, 1000, 20), (9, 1025, 7), (17, 2049, 65), (300, 3001, 16), (7, 4096, 33), (256, 4097, 8),
         (260, 8200, 70), (2, 8193, 3), (4, 20000, 64), (257, 16500, 10), (1, 50000, 200), (256, 33000, 4), (300, 66000, 2), (3, 100003, 1000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,c,k", SIZES)
def test_sizes(rows, c, k, dtype, gpu):
    check(*make(rows, c, k, dtype, labels=(rows + k) % 3 != 0))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,alpha", [(1.0, 0.5), (1.0, 1.0), (4.0, 0.0), (4.0, 1.0), (0.5, 0.9), (20.0, 0.3)])
def test_temperature_and_alpha(T, alpha, dtype, gpu):
    for size in ((12, 300, 9), (3, 20000, 9)):
        check(*make(*size, dtype), T=T, alpha=alpha)
        check(*make(*size, dtype, labels=False), T=T, alpha=alpha)


@pytest.mark.parametrize("size", [(20, 700, 12), (4, 20000, 12), (300, 5000, 12)])
def test_other_gradients_of_the_loss(size, gpu):
    """A loss that is scaled, negated, added up, or passed through twice: every pass has its own gradient."""
    from addernetcuda_amd.distill import distillation_loss
    l, t, i, y = make(*size, torch.float32)
    for scale in (1.0, 0.25, -3.0, 0.0, 1024.0):
        check(l, t, i, y, scale=scale)
    a = l.clone().requires_grad_(True)
    loss = distillation_loss(a, t, i, y, 2.0, 0.7)
    first = torch.autograd.grad(loss, a, retain_graph=True)[0]
    kept = first.clone()
    second = torch.autograd.grad(loss, a, retain_graph=True)[0]
    third = torch.autograd.grad(loss * 2, a)[0]
    assert first.data_ptr() != second.data_ptr() and torch.equal(first, kept)
    within(second, (kept.double().cpu(), 64 * B.U * kept.double().cpu().abs() + 1e-12), "the second pass")
    within(third, (2 * kept.double().cpu(), 128 * B.U * kept.double().cpu().abs() + 1e-12), "the third")
    g = torch.autograd.grad(distillation_loss(a, t, i, y) ** 2, a, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.parametrize("size", [(14, 300, 8), (14, 20000, 8), (280, 3000, 8)])
def test_rows_that_leave_nothing(size, gpu):
    l, t, i, y = make(*size, torch.float32)
    t[0, 3:] = -INF                      # fewer top logits
    t[2] = -INF                          # none
    t[3] = torch.finfo(torch.float32).min
    y[4] = -100
    g = check(l, t, i, y)
    assert not g[4].any() and not g[1].any()
    g = check(l, t, i, None)
    assert not g[2].any()
    from addernetcuda_amd.distill import distillation_loss
    a, anywhere = l.clone().requires_grad_(True), i.clone()
    anywhere[0, 3:], anywhere[2] = -1, size[1] + 7   # (beside -infinity)
    assert torch.equal(torch.autograd.grad(distillation_loss(a, t, anywhere, None, 2.0), a)[0], g)
    everything = torch.full_like(y, -100)
    g = check(l, t, i, everything)
    assert not g.any()
    l[5, 17:40] = -INF                   # masked classes, of which the teacher and the label know none
    i[5] = torch.arange(8, device="cuda")
    y[5] = 12
    check(l, t, i, y)
    l[6] = torch.where(torch.arange(size[1], device="cuda") < 20, l[6], torch.full_like(l[6], torch.finfo(torch.float32).min))
    i[6] = torch.arange(8, device="cuda")
    y[6] = 3
    check(l, t, i, y)


@pytest.mark.parametrize("T,alpha", [(1.0, 0.5), (2.0, 0.5), (4.0, 0.7), (3.0, 0.5), (2.0, 0.0), (2.0, 1.0)])
@pytest.mark.parametrize("size", [(6, 300, 8), (3, 20000, 8), (260, 5000, 8)])
def test_logits_far_from_zero(size, T, alpha, gpu):
    """A row's logits and its teacher's may all be large: what counts is how far they are from each other."""
    l, t, i, y = make(*size, torch.float32)
    for off in (1000.0, -3e4):
        check(l + off, t - off, i, y, T, alpha)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T,alpha", [(1.0, 0.5), (2.0, 0.5), (0.5, 0.5), (3.0, 1.0), (2.0, 0.0)])
@pytest.mark.parametrize("size", [(6, 300, 8), (3, 20000, 8), (260, 2500, 8)])
def test_rows_masked_by_the_lowest_value(size, T, alpha, dtype, gpu):
    """Of a row that is masked as a whole every class is as likely; of one that is masked but for a few, those are."""
    l, t, i, y = make(*size, dtype)
    lowest = torch.finfo(dtype).min
    l[0] = t[0] = lowest
    l[1] = lowest
    l[2, :9000] = lowest
    i[1], y[:3] = torch.arange(8, device="cuda"), 4
    i[2] = size[1] - 1 - torch.arange(8, device="cuda") if size[1] > 9000 else torch.arange(8, device="cuda")
    y[2] = i[2, 0]
    check(l, t, i, y, T, alpha)


@pytest.mark.parametrize("size", [(6, 300, 8), (3, 20000, 8)])
def test_the_same_class_twice(size, gpu):
    l, t, i, y = make(*size, torch.bfloat16)
    i[0] = i[0, 0]
    i[1, 1::2] = i[1, ::2]
    y[0] = i[0, 0]
    check(l, t, i, y)


@pytest.mark.parametrize("size", [(6, 300, 8), (6, 20000, 8)])
def test_what_is_no_number_stays_in_its_row(size, gpu):
    from addernetcuda_amd.distill import distillation_loss
    l, t, i, y = make(*size, torch.float32)
    y[:] = torch.arange(6, device="cuda")
    l.requires_grad_(True)
    want = torch.autograd.grad(distillation_loss(l, t, i, y), l)[0]

    def rows_of(l, t, i, y):
        a = l.detach().clone().requires_grad_(True)
        loss = distillation_loss(a, t, i, y)
        assert torch.isnan(loss)
        g = torch.autograd.grad(loss, a)[0]
        return torch.isnan(g).all(1), g

    for change in ("class", "below", "label", "teacher", "logit", "infinite"):
        L, T, I, Y = l.detach().clone(), t.clone(), i.clone(), y.clone()
        if change == "class":
            I[2, 3] = size[1]
        if change == "below":
            I[2, 3] = -1
        if change == "label":
            Y[2] = size[1] + 5
        if change == "teacher":
            T[2, 1] = float("nan")
        if change == "logit":
            L[2, 299] = float("nan")
        if change == "infinite":
            L[2, 1] = INF
        bad, g = rows_of(L, T, I, Y)
        assert bad.tolist() == [False, False, True, False, False, False], change
        assert torch.equal(g[[0, 1, 3, 4, 5]], want[[0, 1, 3, 4, 5]]), change


def test_layouts_and_types(gpu):
    from addernetcuda_amd.distill import distillation_loss
    for size in ((30, 301, 9), (5, 20001, 9)):
        l, t, i, y = make(*size, torch.bfloat16)
        big = torch.full((size[0], size[1] + 7), float("nan"), device="cuda", dtype=torch.bfloat16)
        v = big[:, 3:3 + size[1]]
        v.copy_(l)
        for lay in (v, l.t().contiguous().t()):
            check(lay, t.t().contiguous().t(), i.t().contiguous().t(), torch.stack([y, y], 1)[:, 0])
        check(l, t.float() + 0.001, i, y)                  # a teacher in float32
        check(l.float(), t, i, y)                          # and in bfloat16
        one = l[:1].expand(size[0], -1).detach().requires_grad_(True)
        loss = distillation_loss(one, t, i, y)
        within(torch.autograd.grad(loss, one)[0], B.distillation(l[:1].expand(size[0], -1), t, i, y, 1.0, 0.5, -100)["grad"], "one row for all")


@pytest.mark.parametrize("size", [(40, 700, 12), (4, 20000, 12), (300, 3000, 12)])
def test_graph(size, gpu):
    from addernetcuda_amd.distill import distillation_loss
    l, t, i, y = make(*size, torch.bfloat16)
    l.requires_grad_(True)
    up = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def run():
        loss = distillation_loss(l, t, i, y, 2.0, 0.5)
        return loss, torch.autograd.grad(loss, l, up)[0]

    with torch.cuda.stream(side):
        want = {}
        for v in (1.0, 0.5):
            up.fill_(v)
            want[v] = [x.detach().clone() for x in run()]
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
    for v in (1.0, 0.5, 1.0):
        up.fill_(v)
        for x in out:
            x.detach().zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want[v], out))


def test_gradient_against_differences(gpu):
    """The loss's own differences in 64 bits, on the formula of the tests' oracle, beside the kernel's gradient."""
    l, t, i, y = make(4, 30, 5, torch.float32)
    g = check(l, t, i, y).double().cpu()
    for r, c in ((0, 3), (2, 17), (3, 0)):
        step = torch.zeros(4, 30, dtype=torch.float64)
        step[r, c] = 1e-4
        lo, hi = (B.distillation(l.double().cpu() + s * step, t.double().cpu(), i.cpu(), y.cpu(), 2.0, 0.7, -100)["loss"][0] for s in (-1, 1))
        assert abs(float((hi - lo) / 2e-4 - g[r, c])) < 1e-6


def test_refusals(gpu):
    from addernetcuda_amd.distill import distillation_loss
    l, t, i, y = make(4, 30, 5, torch.float32)
    for bad in ((l, t[:3], i, y), (l, t, i[:, :2], y), (l, t, i.int(), y), (l, t, i, y[:2]), (l, t, i, y.int()), (l[0], t, i, y), (l, t.cpu(), i, y), (l, t, i, y.cpu()),
                (l[:, :0], t, i, y), (l, t[:, :0], i[:, :0], y)):
        with pytest.raises(RuntimeError):
            distillation_loss(*bad)
    for bad in (dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=INF), dict(alpha=1.5), dict(alpha=-0.1), dict(alpha=float("nan"))):
        with pytest.raises(ValueError):
            distillation_loss(l, t, i, y, **bad)
    assert float(distillation_loss(l[:0], t[:0], i[:0], y[:0])) == 0
    c = 1200   # more top logits than the kernel holds
    l, t, i, y = make(3, c, 1100, torch.float32)
    check(l, t, i, y)
