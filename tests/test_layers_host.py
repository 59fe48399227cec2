"""The linear layer, layer normalisation and AdamW without a GPU: the C entry points refuse bad arguments before they touch one, and the
modules run torch's own operators on the CPU."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p
A = [P(k << 32) for k in range(1, 10)]


def size(call, *args):
    n = ctypes.c_size_t(123)
    return call(*args, ctypes.byref(n)), n.value


def test_linear_refuses():
    from addernetcuda_amd._lib import lib
    f, b = lib.adder_linear_fwd, lib.adder_linear_bwd
    fwd = lambda x=A[0], ldx=64, w=A[1], bias=None, r=None, ldr=0, y=A[2], pre=None, act=0, rows=8, k=64, n=32, t=0, ws=A[3], nb=1 << 30: \
        f(x, ldx, w, bias, r, ldr, y, pre, act, rows, k, n, t, ws, nb, None)
    for bad in ({"x": None}, {"w": None}, {"y": None}):
        assert fwd(**bad) == -1
    for bad in ({"rows": 0}, {"k": 0}, {"n": -1}, {"act": 4}, {"act": -1}, {"t": 2}, {"ldx": 63}, {"ldx": -64}, {"r": A[4], "ldr": 31}):
        assert fwd(**bad) == -2
    assert fwd(rows=1 << 40) == -3 and fwd(ldx=1 << 40) == -3 and fwd(rows=1 << 30, k=64, n=1 << 20) == -3 and fwd(n=(1 << 26) + 1) == -3
    for bad in ({"y": A[0]}, {"y": A[1]}, {"pre": A[2]}, {"r": A[2], "ldr": 32}, {"bias": A[2]}):
        assert fwd(**bad) == -6
    bwd = lambda dy=A[0], ldd=32, pre=A[1], x=A[2], ldx=64, w=A[3], gx=A[4], gw=A[5], gb=A[6], act=2, rows=8, k=64, n=32, t=0, ws=A[7], nb=1 << 30: \
        b(dy, ldd, pre, x, ldx, w, gx, gw, gb, act, rows, k, n, t, ws, nb, None)
    for bad in ({"dy": None}, {"pre": None}, {"x": None}, {"w": None}, {"gx": None, "gw": None, "gb": None}):
        assert bwd(**bad) == -1
    for bad in ({"rows": 0}, {"ldd": 31}, {"ldx": 3}, {"act": 7}, {"t": -1}):
        assert bwd(**bad) == -2
    rc, need = size(lib.adder_linear_bwd_workspace_bytes, 8, 64, 32, 2, 0)
    assert rc == 0 and need >= 8 * 32 * 4
    for bad in ({"ws": None}, {"nb": need - 1}, {"ws": P((7 << 32) + 8)}):
        assert bwd(**bad) == -4
    for bad in ({"gx": A[0]}, {"gw": A[2]}, {"gb": A[3]}, {"gw": A[4]}, {"ws": A[1]}):
        assert bwd(**bad) == -6
    assert size(lib.adder_linear_fwd_workspace_bytes, 0, 64, 32, 0)[0] == -2
    assert lib.adder_linear_fwd_workspace_bytes(8, 64, 32, 0, None) == -1
    assert size(lib.adder_linear_bwd_workspace_bytes, 8, 64, 32, 9, 0)[0] == -2


def test_layer_norm_refuses():
    from addernetcuda_amd._lib import lib
    f, b = lib.adder_layer_norm_fwd, lib.adder_layer_norm_bwd
    fwd = lambda x=A[0], ldx=64, w=A[1], bias=A[2], y=A[3], m=A[4], r=A[5], eps=1e-5, rows=8, d=64, t=0, wt=0: f(x, ldx, w, bias, y, m, r, eps, rows, d, t, wt, None)
    for bad in ({"x": None}, {"y": None}, {"m": None}, {"r": None}):
        assert fwd(**bad) == -1
    for bad in ({"rows": 0}, {"d": 0}, {"ldx": 10}, {"eps": -1.0}, {"eps": float("nan")}, {"t": 3}, {"wt": 3}):
        assert fwd(**bad) == -2
    assert fwd(wt=1) == -7 and fwd(rows=1 << 40) == -3
    for bad in ({"y": A[0]}, {"m": A[3]}, {"r": A[4]}, {"w": A[3]}):
        assert fwd(**bad) == -6
    bwd = lambda dy=A[0], ldd=64, x=A[1], ldx=64, w=A[2], m=A[3], r=A[4], gx=A[5], gw=A[6], gb=A[7], rows=8, d=64, t=1, wt=0, ws=A[8], nb=1 << 30: \
        b(dy, ldd, x, ldx, w, m, r, gx, gw, gb, rows, d, t, wt, ws, nb, None)
    for bad in ({"dy": None}, {"x": None}, {"m": None}, {"r": None}, {"gx": None, "gw": None, "gb": None}):
        assert bwd(**bad) == -1
    for bad in ({"rows": -1}, {"ldd": 1}, {"ldx": 1}, {"t": 9}):
        assert bwd(**bad) == -2
    rc, need = size(lib.adder_layer_norm_bwd_workspace_bytes, 8, 64, 1)
    assert rc == 0 and need >= 2 * 64 * 4
    assert bwd(nb=need - 1) == -4 and bwd(ws=None) == -4 and bwd(t=0, wt=1) == -7
    for bad in ({"gx": A[0]}, {"gw": A[1]}, {"gb": A[6]}, {"ws": A[2]}):
        assert bwd(**bad) == -6


def test_adamw_refuses():
    from addernetcuda_amd._lib import lib
    at = lambda *ks: (P * len(ks))(*[k << 32 for k in ks])
    n1 = (ctypes.c_long * 2)(100, 300)

    def step(count=2, p=at(1, 2), g=at(3, 4), m=at(5, 6), v=at(7, 8), n=n1, lr=0.1, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, t=1, kind=0):
        return lib.adder_adamw_step(count, p, g, m, v, n, None, lr, b1, b2, eps, wd, t, None, kind, None)

    def step8(count=2, p=at(1, 2), g=at(3, 4), m=at(5, 6), v=at(7, 8), ms=at(9, 10), vs=at(11, 12), n=n1, t=1):
        return lib.adder_adamw_step_8bit(count, p, g, m, v, ms, vs, n, None, 0.1, 0.9, 0.99, 1e-8, 0.0, t, None, 0, None)

    for name in "pgmvn":
        assert step(**{name: None}) == -1
    assert step(p=(P * 2)(1 << 32, None)) == -1
    nan = float("nan")
    for bad in ({"count": 0}, {"count": 97}, {"lr": -0.1}, {"lr": nan}, {"b1": 1.0}, {"b2": -0.1}, {"b2": nan}, {"eps": -1.0}, {"wd": -1.0}, {"t": 0},
                {"kind": 2}, {"n": (ctypes.c_long * 2)(100, 0)}):
        assert step(**bad) == -2, bad
    assert step(n=(ctypes.c_long * 2)(100, 1 << 31)) == -3
    for bad in ({"g": at(1, 4)}, {"m": at(1, 6)}, {"v": at(5, 8)}):
        assert step(**bad) == -6
    for name in ("ms", "vs"):
        assert step8(**{name: None}) == -1
    assert step8(count=65) == -2 and step8(t=0) == -2
    for bad in ({"ms": at(5, 10)}, {"vs": at(9, 12)}, {"m": at(3, 6)}):
        assert step8(**bad) == -6
    assert lib.adder_adamw_advance(None, 0.9, 0.99, A[0], None) == -1 and lib.adder_adamw_advance(A[0], 1.0, 0.99, A[1], None) == -2
    assert lib.adder_adamw_advance(A[0], 0.9, 0.99, A[0], None) == -6
    assert lib.adder_state_values(A[0], 1, A[1], None, 8, 0, None) == -1 and lib.adder_state_values(A[0], 1, A[1], A[2], 0, 0, None) == -2
    assert lib.adder_state_values(A[0], 1, A[1], A[0], 8, 0, None) == -6


@pytest.mark.parametrize("act,fn", [("none", lambda t: t), ("relu", torch.relu), ("gelu", torch.nn.functional.gelu), ("silu", torch.nn.functional.silu)])
def test_cpu_tensors_take_torchs_operators(act, fn):
    from addernetcuda_amd.linear import LinearAct
    from addernetcuda_amd.layer_norm import LayerNorm
    layer, norm = LinearAct(12, 7, act=act), LayerNorm(12)
    x, r = torch.randn(3, 5, 12), torch.randn(7)
    want = fn(torch.nn.functional.linear(torch.nn.functional.layer_norm(x, (12,), norm.weight, norm.bias), layer.weight, layer.bias)) + r
    assert torch.allclose(layer(norm(x), residual=r), want)


def test_adamw_on_the_cpu_is_torchs():
    from addernetcuda_amd.optim import AdamW
    a, b = (torch.nn.Parameter(torch.ones(5, 4)) for _ in range(2))
    oa, ob = AdamW([a], lr=0.1), torch.optim.AdamW([b], lr=0.1)
    for t in range(3):
        for p in (a, b):
            p.grad = torch.full((5, 4), 0.1 * (t + 1))
        oa.step()
        ob.step()
    assert torch.allclose(a, b)
    with pytest.raises(RuntimeError, match="state_bits=8"):
        o8 = AdamW([a], state_bits=8)
        o8.step()


def test_token_mlp_on_the_cpu_is_the_network_of_torchs_modules():
    from addernetcuda_amd.models import token_mlp
    stem = lambda i, o, kernel_size, stride, padding, bias: torch.nn.Conv2d(i, o, kernel_size, stride, padding, bias=bias)
    a, b = (token_mlp(width=32, layers=1, adder2d_cls=stem, fused=fused) for fused in (True, False))
    b.load_state_dict(a.state_dict())
    x = torch.randn(4, 3, 32, 32)
    assert torch.allclose(a.eval()(x), b.eval()(x), atol=1e-6)


def test_optimizers_of_the_training_script():
    from addernetcuda_amd import optim, train
    p = [torch.nn.Parameter(torch.ones(3))]
    assert isinstance(train.build_optimizer("sgd", p, 0.1), optim.SGD) and train.build_optimizer("sgd", p, 0.1).defaults["weight_decay"] == 5e-4
    assert train.build_optimizer("adamw8bit", p, 0.1, 0.3).state_bits == 8 and train.build_optimizer("adamw", p, 0.1).state_bits == 32
    with pytest.raises(ValueError, match="unknown optimizer"):
        train.build_optimizer("adam", p, 0.1)


def test_wrapped_and_transformed_calls_take_torchs_operators():
    """vmap, forward-mode derivatives, tracing and second derivatives are torch's business (here on the CPU)."""
    from addernetcuda_amd.linear import linear_act
    from addernetcuda_amd.layer_norm import layer_norm
    x, w, b = torch.randn(4, 3, 8, dtype=torch.float64), torch.randn(5, 8, dtype=torch.float64), torch.randn(5, dtype=torch.float64)
    f = lambda t: linear_act(t, w, b, act="silu")
    assert torch.allclose(torch.func.vmap(f)(x), f(x))
    _, tangent = torch.func.jvp(f, (x,), (torch.ones_like(x),))
    assert tangent.shape == (4, 3, 5)
    assert torch.autograd.gradgradcheck(lambda t: layer_norm(t, torch.ones(8, dtype=torch.float64)), (x[0].requires_grad_(True),))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_survives_copy_and_pickle(bits):
    import copy
    import pickle
    from addernetcuda_amd.optim import AdamW
    opt = AdamW([torch.nn.Parameter(torch.ones(5, 4))], lr=0.1, state_bits=bits, min_8bit_size=77)
    for o in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (o.state_bits, o.min_8bit_size) == (bits, 77)
        p = o.param_groups[0]["params"][0]
        p.grad = torch.ones_like(p)
        if bits == 32:
            o.step()
            assert torch.allclose(p, torch.full_like(p, 0.899))
        else:
            with pytest.raises(RuntimeError, match="state_bits=8 needs"):
                o.step()
        o.load_state_dict(o.state_dict())
        assert o.state_bits == bits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize("amsgrad", [False, True])
def test_adamw_on_the_cpu_resumes_as_torchs(amsgrad, dtype):
    """Step, save, load, step: the same numbers and the same types of state as torch.optim.AdamW, whose moments have the parameter's type."""
    from addernetcuda_amd.optim import AdamW
    results = []
    for kind in (AdamW, torch.optim.AdamW):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 30).to(dtype).view(5, 6))
        opt = kind([p], lr=0.03, amsgrad=amsgrad)
        for t in range(4):
            p.grad = (torch.linspace(1, 2, 30).view(5, 6) / (t + 1)).sin().to(dtype)
            opt.step()
            if t == 1:
                saved = opt.state_dict()
                opt = kind([p], lr=0.03, amsgrad=amsgrad)
                opt.load_state_dict(saved)
        results.append((p, opt.state[p]))
    (p, mine), (q, theirs) = results
    assert torch.equal(p, q) and mine.keys() == theirs.keys()
    for name, value in theirs.items():
        assert mine[name].dtype == value.dtype and torch.equal(mine[name], value), name


def test_adamw_refuses_codes_of_parameters_that_the_kernel_does_not_take():
    from addernetcuda_amd.optim import AdamW
    p = torch.nn.Parameter(torch.ones(300))
    opt = AdamW([p])
    opt.load_state_dict({"state": {0: {"step": 3, "exp_avg": torch.ones(300, dtype=torch.int8), "exp_avg_scale": torch.ones(2),
                                       "exp_avg_sq": torch.ones(300, dtype=torch.uint8), "exp_avg_sq_scale": torch.ones(2)}},
                         "param_groups": opt.state_dict()["param_groups"]})
    p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="state_bits=8 needs"):
        opt.step()
    state = opt.state[p]
    assert torch.equal(p, torch.ones(300)) and state["exp_avg"].dtype == torch.int8 and state["exp_avg_sq"].dtype == torch.uint8
    assert state["exp_avg_scale"].dtype == torch.float32


@pytest.mark.parametrize("name,kw", [("AdamW", {}), ("SGD", {"momentum": 0.9})])
@pytest.mark.parametrize("made", [False, True])
def test_hooks_run_once_a_step(made, name, kw):
    """Also where the whole step is torch's, and an optimizer of torch's own class has been made in the process."""
    from addernetcuda_amd import optim
    if made:
        getattr(torch.optim, name)([torch.nn.Parameter(torch.ones(3))], lr=0.1)
    p = torch.nn.Parameter(torch.ones(3))
    opt = getattr(optim, name)([p], lr=0.1, **kw)
    calls = []
    opt.register_step_pre_hook(lambda *a: calls.append("pre"))
    opt.register_step_post_hook(lambda *a: calls.append("post"))
    for t in range(2):
        p.grad = torch.ones(3)
        opt.step()
    assert calls == ["pre", "post"] * 2 and len(opt.param_groups) == 1 and (p < 0.95).all()
    with torch.no_grad():
        before = p.clone()
    assert opt.step(lambda: torch.tensor(5.0)) == 5.0 and not torch.equal(p, before)   # (still without gradients in the update)


def test_adamw_hands_no_launch_more_than_it_takes():
    """The limit that the optimizer cuts its launches at is the entry points' own: one value more is refused (before the pointers are looked at)."""
    from addernetcuda_amd import optim
    from addernetcuda_amd._lib import lib
    piece = optim._PIECE
    most = optim._GROUPS * 1024
    sizes = [piece] * (most // piece) + [most % piece + 1]
    ps = (P * len(sizes))()
    n = (ctypes.c_long * len(sizes))(*sizes)
    call = lambda k: lib.adder_adamw_step(k, ps, ps, ps, ps, n, None, 0.1, 0.9, 0.99, 1e-8, 0.0, 1, None, 0, None)
    assert call(len(sizes)) == -3
    n[len(sizes) - 1] -= 1
    assert call(len(sizes)) == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("within", [torch.float16, torch.bfloat16])
def test_linear_act_inside_autocast_rounds_its_weights_once(within, dtype):
    """To autocast's type, as nn.Linear: not through bfloat16 on the way to float16."""
    from addernetcuda_amd.linear import LinearAct
    mine, theirs = LinearAct(64, 48), torch.nn.Linear(64, 48)
    theirs.load_state_dict(mine.state_dict())
    x = torch.randn(5, 64).to(dtype)
    with torch.autocast("cpu", dtype=within):
        a, b = mine(x), theirs(x)
    assert a.dtype == b.dtype and torch.equal(a, b)
    assert LinearAct(4, 3, device="meta")(torch.empty(2, 4, dtype=torch.bfloat16, device="meta")).shape == (2, 3)


def test_the_adder_layers_do_without_the_host_module():
    """Where csrc/nodes.cpp is not built, or for another torch, everything but the layers that run on it imports and works."""
    import subprocess
    import sys
    from tests.conftest import ROOT
    code = """
import sys
sys.modules["addernetcuda_amd._nodes"] = None   # what an import of it then finds is an ImportError
import torch
from addernetcuda_amd import adder, models, optim, resnet20, train, _lib
from addernetcuda_amd.linear import LinearAct
models.token_mlp(width=16, layers=1)
LinearAct(4, 3)(torch.ones(2, 4))
p = torch.nn.Parameter(torch.ones(3))
for opt in (optim.SGD([p], lr=0.1, momentum=0.9), optim.AdamW([p])):
    for _ in range(2):
        p.grad = torch.ones(3)
        opt.step()
try:
    _lib.nodes()
except ImportError as e:
    assert "build.py" in str(e)
    print("as it should be")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and "as it should be" in r.stdout, r.stderr


def test_the_library_is_linked_before_the_host_module_can_fail(monkeypatch):
    import importlib.util
    import os
    from tests.conftest import ROOT
    spec = importlib.util.spec_from_file_location("a_build", os.path.join(ROOT, "addernetcuda_amd", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    linked = []

    def no_headers(verbose):
        raise RuntimeError("g++ failed on nodes.cpp")

    monkeypatch.setattr(build, "_compile", lambda src, verbose: src)
    monkeypatch.setattr(build, "_build_nodes", no_headers)
    monkeypatch.setattr(build.subprocess, "check_call", linked.append)
    with pytest.raises(RuntimeError, match="nodes.cpp"):
        build.build()
    assert len(linked) == 1 and build.LIB in linked[0]
