"""The autograd nodes of rms_norm, gated_linear and the loss against a teacher in calls that are not plain ones: hooks on what is saved, anomaly mode, checkpointing, other
threads, and torch's transforms and compiler, which take torch's own operators."""
import copy
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
WHICH = ["rms_norm", "gated_linear", "distillation_loss", "block"]


def make(which, dtype=torch.float32, seed=0):
    """A function of leaves, and the leaves."""
    from addernetcuda_amd.distill import distillation_loss
    from addernetcuda_amd.gated import gated_linear
    from addernetcuda_amd.rms_norm import rms_norm
    g = torch.Generator().manual_seed(seed)
    t = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    x = t(40, 72)
    if which == "rms_norm":
        def of(x, w, r):
            y, s = rms_norm(x, w, 1e-6, residual=r)
            return y * 2 + s
        return of, (x, t(72), t(40, 72))
    if which == "gated_linear":
        return lambda x, w, b: gated_linear(x, w, b, "gelu"), (x, t(48, 72), t(48))
    top, classes, labels = t(40, 5), torch.randint(72, (40, 5), generator=g).cuda(), torch.randint(72, (40,), generator=g).cuda()
    if which == "distillation_loss":
        return lambda x: distillation_loss(x, top, classes, labels, 2.0, 0.5), (x,)

    def of(x, w, r, wide, down):
        y, s = rms_norm(x, w, 1e-6, residual=r)
        return distillation_loss(gated_linear(y, wide) @ down + s, top, classes, labels, 3.0, 0.5)
    return of, (x, t(72), t(40, 72), t(48, 72), t(24, 72))


def leaves_of(tensors):
    return [t.detach().clone().requires_grad_(True) for t in tensors]


def gradients(of, leaves, dy=None):
    y = of(*leaves)
    return y, torch.autograd.grad(y, leaves, torch.ones_like(y) if dy is None else dy)


@pytest.mark.parametrize("which", WHICH)
def test_hooks_on_what_is_saved_and_anomaly_mode(which, gpu):
    of, tensors = make(which)
    leaves = leaves_of(tensors)
    y, want = gradients(of, leaves)
    packed = []

    def pack(t):
        packed.append(t.shape)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        z = of(*leaves)
    assert torch.equal(z, y) and len(packed) >= 3
    for g, h in zip(torch.autograd.grad(z, leaves, torch.ones_like(z)), want):
        assert torch.equal(g, h)
    with torch.autograd.detect_anomaly(check_nan=True):
        with pytest.raises(RuntimeError, match="nan values"):
            torch.autograd.grad(of(*leaves), leaves, torch.full_like(y, float("nan")))
        assert all(torch.equal(g, h) for g, h in zip(gradients(of, leaves)[1], want))


@pytest.mark.parametrize("which", WHICH)
def test_checkpointing(which, gpu):
    from torch.utils.checkpoint import checkpoint
    of, tensors = make(which, torch.bfloat16)
    leaves = leaves_of(tensors)
    y, want = gradients(of, leaves)
    for reentrant in (False, True):
        again = leaves_of(tensors)
        z = checkpoint(of, *again, use_reentrant=reentrant)
        assert torch.equal(z, y)
        z.backward(torch.ones_like(z))
        assert all(torch.equal(t.grad, g) for t, g in zip(again, want))


def test_two_threads_with_a_stream_each(gpu):
    """Passes of all of them at once, over leaves that the threads share; each thread's gradients are those of a pass alone."""
    cases = [(of, leaves_of(tensors)) for of, tensors in (make(which, seed=k) for k, which in enumerate(WHICH))]
    want = [gradients(of, leaves)[1] for of, leaves in cases]
    torch.cuda.synchronize()
    wrong, begin = [], threading.Barrier(2)

    def work():
        try:
            stream = torch.cuda.Stream()
            begin.wait(30)
            with torch.cuda.stream(stream):
                for _ in range(20):
                    for (of, leaves), w in zip(cases, want):
                        got = gradients(of, leaves)[1]
                        stream.synchronize()
                        if not all(torch.equal(g, h) for g, h in zip(got, w)):
                            wrong.append("gradients differ")
        except Exception as e:   # (said by the test, not by a thread)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(90)
    assert not wrong and not any(t.is_alive() for t in threads)


def near(a, b):
    a, b = a.detach(), b.detach()
    return float((a - b).abs().max()) <= 1e-5 * (1 + float(b.abs().max()))


@pytest.mark.parametrize("which", WHICH)
def test_transforms(which, gpu):
    """float32 sums of 72 terms at most, in another order."""
    of, tensors = make(which)
    y, want = gradients(of, leaves_of(tensors))
    got = torch.func.grad(lambda *a: of(*a).sum(), argnums=tuple(range(len(tensors))))(*tensors)
    assert all(near(g, h) for g, h in zip(got, want))
    tangent = torch.randn_like(tensors[0])
    value, along = torch.func.jvp(lambda x: of(x, *tensors[1:]).sum(), (tensors[0],), (tangent,))
    assert near(value, y.sum()) and abs(float(along - (want[0] * tangent).sum())) <= 1e-4 * (1 + float((want[0] * tangent).abs().sum()))
    both = torch.stack([tensors[0], tensors[0] * 0.5])
    each = torch.vmap(lambda x: of(x, *tensors[1:]))(both)
    assert near(each[0], y) and near(each[1], of(both[1], *tensors[1:]))


@pytest.mark.parametrize("which", WHICH)
def test_the_compiler(which, gpu):
    of, tensors = make(which)
    leaves = leaves_of(tensors)
    y, want = gradients(of, leaves)
    torch._dynamo.reset()
    z, got = gradients(torch.compile(of, backend="eager"), leaves)
    assert near(z, y) and all(near(g, h) for g, h in zip(got, want))


def test_8_bit_layers_are_copied_and_saved(gpu, tmp_path):
    from addernetcuda_amd.fp8 import LinearFp8
    torch.manual_seed(1)
    made = LinearFp8.of(torch.nn.Linear(200, 70).cuda(), gate=None)
    x = torch.randn(5, 200, device="cuda")
    with torch.no_grad():
        want = made(x)
        assert torch.equal(copy.deepcopy(made)(x), want)
        torch.save(made.state_dict(), tmp_path / "layer.pt")
        again = LinearFp8(200, 70).cuda()
        again.load_state_dict(torch.load(tmp_path / "layer.pt", weights_only=True))
        assert torch.equal(again(x), want)
