"""RMS norm, gated linear layers, the loss against a teacher and the 8-bit layers together, as the training script runs them: the network of gated blocks
behind an adder layer against the same network of torch's modules, its captured step against the eager one, trained from a teacher, served in 8 bits."""
import copy
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def networks(gpu, **kw):
    from addernetcuda_amd.models import gated_mlp
    torch.manual_seed(5)
    ours = gated_mlp(width=64, layers=2, **kw).to(gpu)
    theirs = gated_mlp(width=64, layers=2, fused=False, **kw).to(gpu)
    theirs.load_state_dict(ours.state_dict())   # the same names
    return ours, theirs


def teach(logits, labels):
    from addernetcuda_amd.distill import distillation_loss
    g = torch.Generator().manual_seed(9)
    top = torch.randn(logits.shape, generator=g).to(logits.device).topk(4, 1)
    return distillation_loss(logits, *top, labels, temperature=3.0, alpha=0.6), top


def test_the_networks_agree(gpu):
    """float32: outputs and gradients through a dozen layers that each round to 1e-7 of their sums differ by 1e-5 of their size at most."""
    ours, theirs = networks(gpu)
    x = torch.randn(32, 3, 32, 32, device=gpu)
    y = torch.randint(0, 10, (32,), device=gpu)
    outs = []
    for net in (ours, theirs):
        logits = net(x)
        loss, top = teach(logits, y)
        if net is theirs:
            from addernetcuda_amd.distill import _torch_distillation_loss
            loss = _torch_distillation_loss(logits, *top, y, 3.0, 0.6, -100)
        loss.backward()
        outs.append([logits.detach(), loss.detach()] + [p.grad for n, p in net.named_parameters() if not n.startswith("stem")])
    for a, b in zip(*outs):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-7


@pytest.mark.parametrize("bf16", [False, True])
def test_captured_step_is_the_eager_one(bf16, gpu):
    from addernetcuda_amd import train
    eager, _ = networks(gpu)
    graphed = copy.deepcopy(eager)
    teacher = train.Teacher(networks(gpu)[1], top=3, temperature=2.0)
    lr = torch.tensor(1e-3, device=gpu)
    oe, og = (train.build_optimizer("adamw", net.parameters(), lr) for net in (eager, graphed))
    step = train.GraphedStep(graphed, og, warmup=1, bf16=bf16, teacher=teacher)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.Generator().manual_seed(0)
    for t in range(5):
        images, labels = torch.randn(16, 3, 32, 32, generator=g).to(gpu), torch.randint(0, 10, (16,), generator=g).to(gpu)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b = step(images, labels)
            a = train.train_step(eager, oe, images, labels, bf16, teacher, teacher(images))
        torch.cuda.synchronize()
        assert torch.equal(a, b), t
        for p, q in zip(eager.parameters(), graphed.parameters()):
            assert torch.equal(p, q), t


def test_the_script_trains_it_from_a_teacher_and_serves_it(gpu, tmp_path):
    from addernetcuda_amd import train
    common = ["--lr", "0.002", "--synthetic", "600", "--epochs", "2", "--batch-size", "100", "--test-batch-size", "50", "--seed", "4", "--optimizer", "adamw"]
    first, second = str(tmp_path / "teacher"), str(tmp_path / "student")
    train.run(train.parse_args(["--arch", "token_mlp", "--output-dir", first] + common))
    teacher = os.path.join(first, "addernet.pt")
    hist = train.run(train.parse_args(["--arch", "gated_mlp", "--output-dir", second, "--teacher", teacher, "--teacher-arch", "token_mlp"] + common))
    assert all(h["train_loss"] == h["train_loss"] for h in hist)
    state = torch.load(os.path.join(second, "addernet.pt"), map_location="cpu", weights_only=True)
    assert "over_channels.0.gated.weight" in state and "stem.adder" in state
    again = ["--arch", "gated_mlp", "--eval-only", "--resume", os.path.join(second, "addernet.pt")] + common
    full, eight, half = (train.run(train.parse_args(again + extra))[0] for extra in ([], ["--fp8"], ["--fp8", "--bf16-activations"]))
    for got in (eight, half):
        assert got["test_loss"] == got["test_loss"] and abs(got["test_loss"] - full["test_loss"]) < 1
    with pytest.raises(ValueError):
        train.run(train.parse_args(["--arch", "token_mlp", "--eval-only", "--fp8"] + common))
    with pytest.raises(ValueError):
        train.run(train.parse_args(["--arch", "gated_mlp", "--fp8"] + common))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_block_in_8_bits(dtype, gpu):
    """norm -> codes -> product -> gate and codes -> product + shortcut: what the parts give one after the other, and near the block in full."""
    from addernetcuda_amd.fp8 import linear_fp8, quantize, quantize_weight, rms_norm_fp8, serve_fp8
    from addernetcuda_amd.models import GatedMLP
    torch.manual_seed(1)
    block = GatedMLP(200, 150).to(gpu)
    full = copy.deepcopy(block)
    x, added = torch.randn(3, 70, 200, device=gpu, dtype=dtype), torch.randn(3, 70, 200, device=gpu, dtype=dtype)
    serve_fp8(torch.nn.Sequential(block))
    with torch.no_grad():
        got, alone = block(x, added), block(x)
        q, qs, s = rms_norm_fp8(added, full.norm.weight.to(dtype), 1e-6, x)
        z = linear_fp8(q, qs, *quantize_weight(full.gated.weight.detach()), dtype=torch.bfloat16)
        want = linear_fp8(*quantize(z, gate="silu"), *quantize_weight(full.down.weight.detach()), residual=s, dtype=dtype)
        assert got.dtype == dtype and torch.equal(got, want)
        for a, b in ((got, full(x, added)), (alone, full(x))):
            part = b.float() - (x + added if a is got else x).float()
            assert float((a.float() - b.float()).norm()) < 0.15 * float(part.norm()) + 0.01 * float(b.float().norm())   # (three roundings to an e4m3 of a sixteenth at most)


@pytest.mark.parametrize("which", ["rms_norm", "gated_linear", "distillation_loss"])
def test_a_capture_beside_a_living_graph_of_the_same_leaves_is_refused(which, gpu):
    """Leaves that a graph of the default stream holds take their gradients there, where no capture may reach; without it they are captured."""
    from addernetcuda_amd.distill import distillation_loss
    from addernetcuda_amd.gated import gated_linear
    from addernetcuda_amd.rms_norm import rms_norm
    g = torch.Generator().manual_seed(11)
    x, w = (torch.randn(*s, generator=g).cuda().requires_grad_(True) for s in ((8, 256), (64, 256)))
    top, classes = torch.randn(8, 4, generator=g).cuda(), torch.randint(256, (8, 4), generator=g).cuda()
    run = {"rms_norm": lambda: rms_norm(x).sum(), "gated_linear": lambda: gated_linear(x, w).sum(), "distillation_loss": lambda: distillation_loss(x, top, classes)}[which]
    run().backward()
    want, x.grad, w.grad = x.grad.clone(), None, None
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    held = run()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        loss = run()
        with pytest.raises(RuntimeError, match="cannot be captured while"):
            loss.backward()
    del held, loss, graph
    with torch.cuda.stream(side):
        run().backward()   # (on the way to a capture: nothing that the first pass of a program makes)
        side.synchronize()
        x.grad = w.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run().backward()
    for _ in range(3):
        x.grad.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x.grad, want)
