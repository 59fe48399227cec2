"""Which leaves a backward pass comes to from a node on: what the layers' nodes look through before their gradients are captured into a graph.  (The walk is host code
over the graph that torch made, here of its own operators.)"""
import torch


def below(y):
    from addernetcuda_amd._lib import nodes
    return {t.data_ptr() for t in nodes().leaves_below(y)}


def leaf(*shape, dtype=torch.float32):
    return torch.randn(*shape).to(dtype).requires_grad_(True)


def test_leaves_behind_casts_views_and_other_layers():
    from addernetcuda_amd.models import GatedMLP
    x, w, b = leaf(4, 6), leaf(5, 6), leaf(5)
    held = lambda *leaves: {t.data_ptr() for t in leaves}
    y = torch.nn.functional.linear(x.to(torch.bfloat16), w.to(torch.bfloat16), b.to(torch.bfloat16))
    assert below(y) == held(x, w, b)
    assert below(torch.nn.functional.linear(x, w.t().contiguous().t(), b.expand(5))) == held(x, w, b)
    assert below(x.detach() @ w.t()) == held(w) and below((x.view(2, 2, 6).transpose(0, 1) * 2).sum()) == held(x)
    block = GatedMLP(6, 8)
    out = block(x, added=leaf(4, 6))
    assert held(x, *block.parameters()) <= below(out)
    assert len(below(out)) == 2 + len(list(block.parameters()))
    twice = block(block(x))
    assert below(twice) == held(x, *block.parameters())
    assert below(leaf(3)) == set()


def test_a_pass_for_some_inputs_comes_to_those_alone():
    x, w, b = leaf(4, 6), leaf(5, 6), leaf(5)
    got = []
    h = (x * 2).sin()
    y = torch.nn.functional.linear(h, w * 1, b)
    h.register_hook(lambda g: got.append(below(h)))
    y.register_hook(lambda g: got.append(below(y)))
    torch.autograd.grad(y.sum(), x, retain_graph=True)
    assert got == [{x.data_ptr()}] * 2
    got.clear()
    y.sum().backward()
    assert got == [{x.data_ptr(), w.data_ptr(), b.data_ptr()}, {x.data_ptr()}]


def test_many_nodes_and_no_recursion():
    x = leaf(2)
    y = x
    for _ in range(30000):
        y = y + x
    assert below(y) == {x.data_ptr()}
