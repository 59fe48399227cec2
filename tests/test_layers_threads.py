"""Other Python threads run while the host module of the linear layers, layer norm and AdamW is inside the library."""
import ctypes
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture
def slow_library(gpu):
    """The host module bound to the library with usleep in place of some entry points (it sleeps for as many microseconds as their first argument
    says, and returns 0); bound to the library itself again behind the test."""
    from addernetcuda_amd import _lib
    real = {name: ctypes.cast(getattr(_lib.lib, name), ctypes.c_void_p).value for name in _lib.EXPORTED}
    sleep = ctypes.cast(ctypes.CDLL(None).usleep, ctypes.c_void_p).value
    yield lambda *names: _lib.nodes().bind({**real, **dict.fromkeys(names, sleep)})
    _lib.nodes().bind(real)


def others_run_during(call):
    stop, times = threading.Event(), []

    def count():
        while not stop.is_set():
            times.append(time.perf_counter())
            time.sleep(0.0002)

    thread = threading.Thread(target=count)
    thread.start()
    begin = time.perf_counter()
    result = call()
    end = time.perf_counter()
    stop.set()
    thread.join()
    edge = 0.25 * (end - begin)
    assert end - begin > 0.02
    return result, sum(begin + edge < t < end - edge for t in times) >= 3


def test_linear_act(slow_library):
    from addernetcuda_amd.linear import linear_act
    rows = 200000
    x, w = torch.randn(rows, 1, device="cuda"), torch.ones(1, 1, device="cuda")
    linear_act(x, w)
    slow_library("adder_linear_fwd_workspace_bytes")   # (none is needed)
    for leaf in (x, x.clone().requires_grad_(True)):
        y, ran = others_run_during(lambda: linear_act(leaf, w))
        assert ran and torch.equal(y, x)


def test_adamw_step(slow_library):
    from addernetcuda_amd import _lib
    p = torch.nn.Parameter(torch.ones(1 << 22, device="cuda"))
    p.grad = torch.ones_like(p)
    state = {"step": 0, "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p)}
    slow_library("adder_adamw_step")   # (96 entries, 96 microseconds)
    done, ran = others_run_during(lambda: _lib.nodes().adamw_step([p], [state], False, 0.1, 0, 0.9, 0.99, 1e-8, 0.0, 256, 1 << 20))
    assert done and ran and state["step"] == 1 and p.detach().eq(1).all()


@pytest.mark.parametrize("layer", ["linear", "norm"])
def test_python_hooks_run_inside_the_nodes(layer, gpu):
    """Hooks on what is saved for the backward are Python, called from inside the module; so is what anomaly mode records."""
    from addernetcuda_amd.layer_norm import layer_norm
    from addernetcuda_amd.linear import linear_act
    x, w, b = torch.randn(40, 24, device="cuda"), torch.randn(24, 24, device="cuda"), torch.randn(24, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w if layer == "linear" else b)]
    run = (lambda: linear_act(x, w, b, act="gelu")) if layer == "linear" else lambda: layer_norm(x, b)
    want = torch.autograd.grad(run().square().sum(), leaves)
    packed = []

    def pack(t):
        packed.append(t.shape)
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        y = run()
    assert len(packed) >= 3
    for g, h in zip(torch.autograd.grad(y.square().sum(), leaves), want):
        assert torch.equal(g, h)
    with torch.autograd.detect_anomaly(check_nan=True):
        with pytest.raises(RuntimeError, match="nan values"):
            torch.autograd.grad(run(), leaves, torch.full((40, 24), float("nan"), device="cuda"))
