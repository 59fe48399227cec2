"""The loss against a teacher where its forward and its backward are not captured together: a backward that is replayed has no gradient ready but its own."""
import pytest
import torch

from tests.test_gpu_distill import make

pytestmark = pytest.mark.gpu


def passes(size):
    from addernetcuda_amd.distill import distillation_loss
    l, t, i, y = make(*size, torch.float32)
    l.requires_grad_(True)
    up = torch.ones((), device="cuda")
    loss_of = lambda: distillation_loss(l, t, i, y, 2.0, 0.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    return l, up, loss_of, side


def check(replay, out, up, want):
    """Replays with other gradients of the loss, and with a result that was edited in between, against what eager passes gave."""
    for k, v in enumerate((1.0, 0.5, 1.0, -2.0, 1.0)):
        up.fill_(v)
        if k % 2:
            out.detach().fill_(7.0)
        torch.cuda.synchronize()
        replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[v]), (k, v)


@pytest.mark.parametrize("size", [(40, 700, 12), (4, 20000, 12), (300, 3000, 12)])
def test_a_backward_captured_by_itself(size, gpu):
    l, up, loss_of, side = passes(size)
    with torch.cuda.stream(side):
        want = {}
        for v in (1.0, 0.5, -2.0):
            up.fill_(v)
            loss = loss_of()
            torch.autograd.grad(loss, l, retain_graph=True)   # (the second pass computes its own, as the captured one)
            want[v] = torch.autograd.grad(loss, l, up)[0].clone()
        up.fill_(1.0)
        loss = loss_of()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out, = torch.autograd.grad(loss, l, up, retain_graph=True)
    check(graph.replay, out, up, want)


@pytest.mark.parametrize("size", [(40, 700, 12), (4, 20000, 12), (300, 3000, 12)])
def test_forward_and_backward_in_graphs_of_their_own(size, gpu):
    l, up, loss_of, side = passes(size)
    with torch.cuda.stream(side):
        want = {}
        for v in (1.0, 0.5, -2.0):
            up.fill_(v)
            loss = loss_of()
            torch.autograd.grad(loss, l, retain_graph=True)
            want[v] = torch.autograd.grad(loss, l, up)[0].clone()
        side.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=side):
            loss = loss_of()
        with torch.cuda.graph(second, stream=side, pool=first.pool()):
            out, = torch.autograd.grad(loss, l, up, retain_graph=True)
    first.replay()
    check(second.replay, out, up, want)
    first.replay()
    check(second.replay, out, up, want)
