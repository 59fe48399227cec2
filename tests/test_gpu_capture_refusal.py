"""A backward pass that is captured beside a living graph of the same leaves from the default stream is refused by the first of the layers' nodes that it comes to, before
anything is captured for a leaf; without that graph it is captured, and replays what the eager pass gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(which):
    """A pass, and the leaves whose gradients it gives."""
    from addernetcuda_amd.distill import distillation_loss
    from addernetcuda_amd.gated import GatedLinear, gated_linear
    from addernetcuda_amd.layer_norm import layer_norm
    from addernetcuda_amd.linear import linear_act
    from addernetcuda_amd.models import GatedMLP, gated_mlp
    torch.manual_seed(12)
    x = torch.randn(8, 256, device="cuda")
    leaf = lambda *shape: torch.randn(*shape, device="cuda").requires_grad_(True)
    if which == "linear_act":
        w, b = leaf(64, 256), leaf(64)
        return lambda: linear_act(x, w, b, act="gelu").sum(), [w, b]
    if which == "layer_norm":
        w, b = leaf(256), leaf(256)
        return lambda: layer_norm(x, w, b).sum(), [w, b]
    if which == "a strided weight":
        w = leaf(256, 64)
        return lambda: gated_linear(x, w.t()).sum(), [w]
    if which == "parameters that are cast":
        layer = GatedLinear(256, 32, bias=True).cuda()
        return lambda: layer(x.bfloat16()).sum(), list(layer.parameters())
    if which == "autocast":
        layer = GatedLinear(256, 32).cuda()

        def run():
            with torch.autocast("cuda", dtype=torch.bfloat16):
                return layer(x).float().sum()
        return run, list(layer.parameters())
    if which == "a leaf behind torch's operators":
        w = leaf(64, 256)
        return lambda: layer_norm(x @ (w * 2).t()).square().sum(), [w]
    if which == "a gated block":
        block, first = GatedMLP(256, 64).cuda(), leaf(8, 256)
        return lambda: block(first, added=x).square().sum(), [first, *block.parameters()]
    net = gated_mlp(width=64, layers=1).cuda()
    images, labels = torch.randn(8, 3, 32, 32, device="cuda"), torch.randint(10, (8,), device="cuda")
    top, classes = torch.randn(8, 4, device="cuda"), torch.randint(10, (8, 4), device="cuda")
    return lambda: distillation_loss(net(images), top, classes, labels), list(net.parameters())


@pytest.mark.parametrize("which", ["linear_act", "layer_norm", "a strided weight", "parameters that are cast", "autocast", "a leaf behind torch's operators", "a gated block",
                                   "a network"])
def test_refused_beside_a_living_graph(which, gpu):
    run, leaves = make(which)
    run().backward()
    want = [t.grad.clone() for t in leaves]
    for t in leaves:
        t.grad = None
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    held = run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        loss = run()
        with pytest.raises(RuntimeError, match="cannot be captured while"):
            loss.backward()
    assert all(t.grad is None for t in leaves)
    del held, loss, graph
    if which == "a network":   # (its BatchNorm has moved on)
        return
    with torch.cuda.stream(side):
        run().backward()   # (on the way to a capture: nothing that the first pass of a program makes)
        side.synchronize()
        for t in leaves:
            t.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run().backward()
    for _ in range(3):
        for t in leaves:
            t.grad.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, g in zip(leaves, want):
            assert torch.equal(t.grad, g)
