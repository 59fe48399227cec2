"""Linear layers, layer norm and AdamW together, as the training script runs them: the network of residual MLPs behind an adder layer
against the same network of torch's modules, its captured step against the eager one, and training through the script."""
import copy
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def networks(gpu, **kw):
    from addernetcuda_amd.models import token_mlp
    torch.manual_seed(5)
    ours = token_mlp(width=64, layers=2, **kw).to(gpu)
    theirs = token_mlp(width=64, layers=2, fused=False, **kw).to(gpu)
    theirs.load_state_dict(ours.state_dict())   # the same names
    return ours, theirs


def test_the_networks_agree(gpu):
    """float32: outputs and gradients through 17 layers that each round to 1e-7 of their sums differ by 1e-5 of their size at most."""
    ours, theirs = networks(gpu)
    x = torch.randn(32, 3, 32, 32, device=gpu)
    y = torch.randint(0, 10, (32,), device=gpu)
    outs = []
    for net in (ours, theirs):
        logits = net(x)
        torch.nn.functional.cross_entropy(logits, y).backward()
        outs.append([logits.detach()] + [p.grad for n, p in net.named_parameters() if not n.startswith("stem")])
    for a, b in zip(*outs):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm()) + 1e-7
    ours.eval(), theirs.eval()
    with torch.no_grad():
        a, b = ours(x), theirs(x)
    assert float((a - b).norm()) <= 1e-4 * float(b.norm())


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8bit"])
def test_captured_step_is_the_eager_one(optimizer, gpu):
    from addernetcuda_amd import train
    eager, _ = networks(gpu)
    graphed = copy.deepcopy(eager)
    lr = torch.tensor(1e-3, device=gpu)
    oe, og = (train.build_optimizer(optimizer, net.parameters(), lr) for net in (eager, graphed))
    step = train.GraphedStep(graphed, og, warmup=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.Generator().manual_seed(0)
    for t in range(5):
        images, labels = torch.randn(16, 3, 32, 32, generator=g).to(gpu), torch.randint(0, 10, (16,), generator=g).to(gpu)
        lr.fill_(1e-3 / (t + 1))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            b = step(images, labels)
            a = train.train_step(eager, oe, images, labels)
        torch.cuda.synchronize()
        assert torch.equal(a, b), t
        for p, q in zip(eager.parameters(), graphed.parameters()):
            assert torch.equal(p, q), t


@pytest.mark.parametrize("extra", [["--optimizer", "adamw"], ["--optimizer", "adamw8bit"], ["--optimizer", "adamw8bit", "--bf16-activations", "--no-graph"]])
def test_the_script_trains_it(extra, gpu, tmp_path):
    from addernetcuda_amd import train
    hist = train.run(train.parse_args(["--arch", "token_mlp", "--lr", "0.002", "--synthetic", "2000", "--epochs", "5", "--batch-size", "100",
                                       "--test-batch-size", "50", "--output-dir", str(tmp_path), "--seed", "4"] + extra))
    assert all(h["train_loss"] == h["train_loss"] for h in hist)
    assert hist[-1]["train_loss"] < hist[0]["train_loss"] and max(h["accuracy"] for h in hist) > 0.4
    state = torch.load(os.path.join(str(tmp_path), "addernet.pt"), map_location="cpu", weights_only=True)
    assert "over_channels.0.fc1.weight" in state and "stem.adder" in state
