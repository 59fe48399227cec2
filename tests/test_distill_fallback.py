"""The loss against a teacher where torch's operators compute it (CPU tensors here): what is no number, or names a class that does not exist, does to the loss and
the gradients what it does in the kernels -- nothing in a row that does not count, and in one that counts, no number for the row as a whole."""
import pytest
import torch

from tests import block_bounds as B

INF, NAN = float("inf"), float("nan")


def make(rows=6, c=40, k=5):
    g = torch.Generator().manual_seed(3)
    l = torch.randn(rows, c, generator=g, dtype=torch.float64)
    t, i = torch.randn(rows, c, generator=g, dtype=torch.float64).topk(k, 1)
    y = torch.randint(0, c, (rows,), generator=g)
    y[1] = -100
    return l, t, i, y


def loss_and_gradient(l, t, i, y, T=2.0, alpha=0.6):
    from addernetcuda_amd.distill import distillation_loss
    l = l.clone().requires_grad_(True)
    loss = distillation_loss(l, t, i, y, T, alpha)
    return loss.detach(), torch.autograd.grad(loss, l)[0]


def change(row, what, l, t, i, y):
    l, t, i, y = l.clone(), t.clone(), i.clone(), y.clone()
    if what in ("teacher nan", "teacher inf"):
        t[row, 1] = NAN if what == "teacher nan" else INF
    if what == "class":
        i[row, 2] = 40
    if what == "no class":
        i[row, 2] = -1
    if what == "class of no weight":     # (p is zero there)
        i[row, 4], t[row, 4] = 77, -1e6
    if what in ("logit nan", "logit inf"):
        l[row, 7] = NAN if what == "logit nan" else INF
    if what == "masked":
        l[row] = -INF
    return l, t, i, y


WHATS = ["teacher nan", "teacher inf", "class", "no class", "class of no weight", "logit nan", "logit inf", "masked"]


@pytest.mark.parametrize("what", WHATS)
def test_a_row_that_does_not_count_adds_nothing(what):
    whole = make()
    want_loss, want = loss_and_gradient(*whole)
    loss, grad = loss_and_gradient(*change(1, what, *whole))
    assert torch.equal(loss, want_loss) and torch.equal(grad, want) and not grad[1].any()


@pytest.mark.parametrize("what", WHATS)
@pytest.mark.parametrize("labels", [True, False])
def test_a_row_that_counts_is_no_number_as_a_whole(what, labels):
    whole = make()
    _, want = loss_and_gradient(*whole[:3], whole[3] if labels else None)
    l, t, i, y = change(2, what, *whole)
    loss, grad = loss_and_gradient(l, t, i, y if labels else None)
    assert torch.isnan(loss)
    others = [0, 1, 3, 4, 5]
    assert torch.isnan(grad[2]).all() and torch.equal(grad[others], want[others])


def test_what_is_not_asked_for_does_not_count():
    """The teacher's part where alpha is zero, the label where it is one, a class beside -infinity."""
    l, t, i, y = make()
    want = loss_and_gradient(l, t, i, y, alpha=0.0)
    for what in ("teacher nan", "class", "no class"):
        got = loss_and_gradient(*change(2, what, l, t, i, y), alpha=0.0)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    want = loss_and_gradient(l, t, i, y, alpha=1.0)
    other = y.clone()
    other[2] = 99
    got = loss_and_gradient(l, t, i, other, alpha=1.0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    t[3, 2:] = t[4] = -INF
    want, formula = loss_and_gradient(l, t, i, y), B.distillation(l, t, i, y, 2.0, 0.6, -100)
    i[3, 2:], i[4] = 1000, -7
    got = loss_and_gradient(l, t, i, y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.allclose(got[1], formula["grad"][0], atol=1e-12) and abs(float(got[0] - formula["loss"][0])) < 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("what", WHATS)
@pytest.mark.parametrize("row", [1, 2])
def test_the_kernels_say_the_same(what, row, gpu):
    """Loss and gradients of both ways: finite together, or no numbers in the same rows."""
    args = change(row, what, *make())
    want = loss_and_gradient(*args)
    l, t, i, y = args
    got = loss_and_gradient(l.float().cuda(), t.float().cuda(), i.cuda(), y.cuda())
    assert torch.equal(torch.isnan(got[0]).cpu(), torch.isnan(want[0]))
    assert torch.equal(torch.isnan(got[1]).cpu(), torch.isnan(want[1]))
    assert torch.equal((got[1] == 0).all(1).cpu(), (want[1] == 0).all(1))


@pytest.mark.gpu
def test_more_top_logits_than_the_kernel_holds(gpu):
    whole = make(6, 1200, 1100)
    y = whole[3].cuda()
    for row in (1, 2):
        for what in ("teacher nan", "logit nan", "no class"):
            l, t, i, _ = change(row, what, *whole)
            loss, grad = loss_and_gradient(l.float().cuda(), t.float().cuda(), i.cuda(), y)
            assert bool(torch.isnan(loss)) == (row == 2)
            assert torch.isnan(grad).all(1).tolist() == [r == 2 and row == 2 for r in range(6)] and not torch.isnan(grad[[0, 1, 3, 4, 5]]).any()
            assert not grad[1].any()
