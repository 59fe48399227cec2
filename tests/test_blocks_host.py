"""RMS norm, gated linear layers, 8-bit codes and the loss against a teacher without a GPU: the C entry points refuse bad arguments before they
touch one, and the functions run torch's own operators on the CPU."""
import ctypes

import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import within

P = ctypes.c_void_p
A = [P(k << 36) for k in range(1, 14)]


def size(call, *args):
    n = ctypes.c_size_t(123)
    return call(*args, ctypes.byref(n)), n.value


def test_rms_norm_refuses():
    from addernetcuda_amd._lib import lib
    fwd = lambda x=A[0], ldx=64, r=A[1], ldr=64, w=A[2], s=A[3], y=A[4], rstd=A[5], eps=1e-6, rows=8, d=64, t=0, wt=0: \
        lib.adder_rms_norm_fwd(x, ldx, r, ldr, w, s, y, rstd, eps, rows, d, t, wt, None)
    codes = lambda x=A[0], ldx=64, r=A[1], ldr=64, w=A[2], s=A[3], q=A[4], qs=A[5], eps=1e-6, rows=8, d=64, t=0, wt=0: \
        lib.adder_rms_norm_fwd_codes(x, ldx, r, ldr, w, s, q, qs, eps, rows, d, t, wt, None)
    for call in (fwd, codes):
        assert call(x=None) == -1
        for bad in ({"rows": 0}, {"d": 0}, {"ldx": 10}, {"ldr": 63}, {"ldx": -64}, {"eps": -1.0}, {"eps": float("nan")}, {"t": 3}, {"wt": 3}):
            assert call(**bad) == -2, bad
        assert call(wt=1) == -7 and call(rows=1 << 40) == -3 and call(ldr=1 << 40) == -3 and call(d=(1 << 26) + 1, ldx=1 << 27, ldr=1 << 27) == -3
        for bad in ({"s": A[0]}, {"s": A[1]}, {"w": A[3]}, {"r": A[4]}):
            assert call(**bad) == -6, bad
    assert fwd(y=None) == -1 and fwd(y=A[0]) == -6 and fwd(rstd=A[4]) == -6
    assert codes(q=None) == -1 and codes(qs=None) == -1 and codes(qs=A[4]) == -6
    bwd = lambda dy=A[0], ldd=64, ds=A[1], lds=64, x=A[2], ldx=64, w=A[3], rstd=A[4], gx=A[5], gw=A[6], rows=8, d=64, t=1, wt=0, ws=A[7], nb=1 << 30: \
        lib.adder_rms_norm_bwd(dy, ldd, ds, lds, x, ldx, w, rstd, gx, gw, rows, d, t, wt, ws, nb, None)
    for bad in ({"dy": None}, {"x": None}, {"rstd": None}, {"gx": None, "gw": None}):
        assert bwd(**bad) == -1
    for bad in ({"rows": -1}, {"ldd": 1}, {"lds": 1}, {"ldx": 1}, {"t": 9}):
        assert bwd(**bad) == -2
    rc, need = size(lib.adder_rms_norm_bwd_workspace_bytes, 8, 64, 1)
    assert rc == 0 and need >= 64 * 4
    assert bwd(nb=need - 1) == -4 and bwd(ws=None) == -4 and bwd(ws=P((8 << 36) + 8)) == -4 and bwd(t=0, wt=1) == -7
    for bad in ({"gx": A[0]}, {"gx": A[1]}, {"gw": A[2]}, {"ws": A[3]}, {"gw": A[5]}):
        assert bwd(**bad) == -6
    assert lib.adder_rms_norm_bwd_workspace_bytes(8, 64, 1, None) == -1 and size(lib.adder_rms_norm_bwd_workspace_bytes, 0, 64, 1)[0] == -2


def test_codes_refuse():
    from addernetcuda_amd._lib import lib
    q = lambda x=A[0], ld=64, act=-1, c=A[1], s=A[2], rows=8, d=64, t=0: lib.adder_quantize(x, ld, act, c, s, rows, d, t, None)
    w = lambda x=A[0], ld=64, c=A[1], s=A[2], rows=8, d=64, t=0: lib.adder_quantize_weight(x, ld, c, s, rows, d, t, None)
    for call in (q, w):
        for bad in ({"x": None}, {"c": None}, {"s": None}):
            assert call(**bad) == -1
        for bad in ({"rows": 0}, {"d": -1}, {"ld": 63}, {"t": 2}):
            assert call(**bad) == -2
        assert call(rows=1 << 40) == -3 and call(d=(1 << 26) + 1, ld=1 << 27) == -3
        for bad in ({"c": A[0]}, {"s": A[1]}, {"s": A[0]}):
            assert call(**bad) == -6
    assert q(act=4) == -2 and q(act=3) == -2 and q(act=3, ld=128, rows=0) == -2   # (a gated row is twice as long)
    lin = lambda x=A[0], ldx=64, xs=A[1], w=A[2], ldw=64, ws=A[3], b=None, r=None, ldr=0, y=A[4], act=0, rows=8, k=64, n=32, t=0, work=A[5], nb=1 << 30: \
        lib.adder_linear_codes(x, ldx, xs, w, ldw, ws, b, r, ldr, y, act, rows, k, n, t, work, nb, None)
    for bad in ({"x": None}, {"xs": None}, {"w": None}, {"ws": None}, {"y": None}):
        assert lin(**bad) == -1
    for bad in ({"rows": 0}, {"k": 0}, {"n": -1}, {"act": 4}, {"act": -1}, {"t": 2}, {"ldx": 63}, {"ldw": 63}, {"r": A[6], "ldr": 31}):
        assert lin(**bad) == -2
    assert lin(rows=1 << 40) == -3 and lin(ldx=1 << 23) == -3 and lin(ldw=1 << 23) == -3 and lin(k=1 << 23, ldx=1 << 23, ldw=1 << 23) == -3
    for bad in ({"y": A[0]}, {"y": A[1]}, {"y": A[2]}, {"y": A[3]}, {"b": A[4]}, {"r": A[4], "ldr": 32}):
        assert lin(**bad) == -6
    rc, need = size(lib.adder_linear_codes_workspace_bytes, 200, 100, 70, 0, 0, 0)
    assert rc == 0 and need >= (200 + 70) * 100 and size(lib.adder_linear_codes_workspace_bytes, 200, 112, 70, 0, 1, 1)[1] < need
    for bad in ({"work": None}, {"nb": need - 300}, {"work": P((7 << 36) + 8)}):
        assert lin(rows=200, k=100, ldx=100, ldw=100, n=70, **bad) == -4
    assert size(lib.adder_linear_codes_workspace_bytes, 0, 1, 1, 0, 0, 0)[0] == -2 and lib.adder_linear_codes_kernel(1, 1, 1, 0, None) == -1


def test_gated_refuses():
    from addernetcuda_amd._lib import lib
    fwd = lambda x=A[0], ldx=64, w=A[1], b=None, y=A[2], pre=None, act=3, rows=8, k=64, h=32, t=0, ws=A[3], nb=1 << 30: \
        lib.adder_gated_fwd(x, ldx, w, b, y, pre, act, rows, k, h, t, ws, nb, None)
    for bad in ({"x": None}, {"w": None}, {"y": None}):
        assert fwd(**bad) == -1
    for bad in ({"rows": 0}, {"k": 0}, {"h": -1}, {"act": 4}, {"act": -1}, {"t": 2}, {"ldx": 63}):
        assert fwd(**bad) == -2
    assert fwd(rows=1 << 40) == -3 and fwd(ldx=1 << 40) == -3 and fwd(h=1 << 25) == -3 and fwd(h=0x7fffffff) == -3
    for bad in ({"y": A[0]}, {"y": A[1]}, {"pre": A[2]}, {"b": A[2]}):
        assert fwd(**bad) == -6
    bwd = lambda dy=A[0], ldd=32, pre=A[1], x=A[2], ldx=64, w=A[3], gx=A[4], gw=A[5], gb=A[6], act=2, rows=8, k=64, h=32, t=0, ws=A[7], nb=1 << 30: \
        lib.adder_gated_bwd(dy, ldd, pre, x, ldx, w, gx, gw, gb, act, rows, k, h, t, ws, nb, None)
    for bad in ({"dy": None}, {"pre": None}, {"x": None}, {"w": None}, {"gx": None, "gw": None, "gb": None}):
        assert bwd(**bad) == -1
    for bad in ({"rows": 0}, {"ldd": 31}, {"ldx": 3}, {"act": 7}, {"t": -1}):
        assert bwd(**bad) == -2
    rc, need = size(lib.adder_gated_bwd_workspace_bytes, 8, 64, 32, 0)
    assert rc == 0 and need >= 8 * 64 * 4
    for bad in ({"ws": None}, {"nb": need - 1}, {"ws": P((8 << 36) + 8)}):
        assert bwd(**bad) == -4
    for bad in ({"gx": A[0]}, {"gw": A[2]}, {"gb": A[3]}, {"gw": A[4]}, {"ws": A[1]}):
        assert bwd(**bad) == -6
    assert size(lib.adder_gated_fwd_workspace_bytes, 0, 64, 32, 0)[0] == -2 and lib.adder_gated_kernel(8, 8, 8, 0, 1, 3, ctypes.byref(ctypes.c_int())) == -2


def test_distill_refuses():
    from addernetcuda_amd._lib import lib
    fwd = lambda l=A[0], ld=100, t=A[1], i=A[2], y=A[3], loss=A[4], stats=A[5], g=A[6], T=2.0, a=0.5, rows=8, c=100, k=5, ty=0, tt=0, ws=A[7], nb=1 << 20: \
        lib.adder_distill_fwd(l, ld, t, i, y, loss, stats, g, T, a, -100, rows, c, k, ty, tt, ws, nb, None)
    nan, inf = float("nan"), float("inf")
    for bad in ({"l": None}, {"t": None}, {"i": None}, {"loss": None}, {"stats": None}):
        assert fwd(**bad) == -1
    for bad in ({"rows": 0}, {"c": 0}, {"k": 0}, {"ld": 99}, {"ty": 2}, {"tt": -1}, {"T": 0.0}, {"T": nan}, {"T": inf}, {"a": -0.1}, {"a": 1.1}, {"a": nan}):
        assert fwd(**bad) == -2, bad
    assert fwd(k=1025) == -7 and fwd(rows=4, c=100000, ld=100000) == -7   # (no gradient on the way where workgroups share a row)
    assert fwd(rows=1 << 40) == -3 and fwd(c=(1 << 26) + 1, ld=1 << 27, g=None) == -3
    assert fwd(ws=None) == -4 and fwd(nb=8) == -4
    for bad in ({"g": A[0]}, {"loss": A[1]}, {"stats": A[2]}, {"ws": A[3]}, {"g": A[5]}):
        assert fwd(**bad) == -6
    bwd = lambda l=A[0], t=A[1], i=A[2], y=A[3], stats=A[4], up=A[5], g=A[6], T=2.0, rows=8, c=100, k=5: \
        lib.adder_distill_bwd(l, c, t, i, y, stats, up, 0, g, T, 0.5, -100, rows, c, k, 0, 0, None)
    for bad in ({"l": None}, {"t": None}, {"i": None}, {"stats": None}, {"up": None}, {"g": None}):
        assert bwd(**bad) == -1
    assert bwd(rows=0) == -2 and bwd(T=-1.0) == -2 and bwd(k=2000) == -7
    for bad in ({"g": A[0]}, {"g": A[4]}, {"g": A[5]}):
        assert bwd(**bad) == -6
    assert lib.adder_distill_in_rows(8, 100, 0) == 1 and lib.adder_distill_in_rows(4, 100000, 0) == 0 and lib.adder_distill_in_rows(0, 5, 0) == 0
    assert size(lib.adder_distill_workspace_bytes, 0, 5, 0)[0] == -2 and lib.adder_distill_workspace_bytes(1, 5, 0, None) == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_cpu_tensors_take_torchs_operators(dtype):
    from addernetcuda_amd.fp8 import linear_fp8, quantize, quantize_weight, rms_norm_fp8
    from addernetcuda_amd.gated import GatedLinear
    from addernetcuda_amd.rms_norm import RMSNorm, rms_norm
    small = torch.randn(5, 200).to(dtype) * 2.0 ** -10
    assert torch.equal(RMSNorm(200, eps=None, dtype=dtype)(small), torch.nn.RMSNorm(200, eps=None, dtype=dtype)(small))
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(6, 200, generator=g).to(dtype) for _ in range(2))
    norm, gated = RMSNorm(200, dtype=dtype), GatedLinear(200, 30, dtype=dtype)
    with torch.no_grad():
        y, s = norm(x, residual=r)
    assert torch.equal(s, x + r) and y.dtype == dtype
    want = torch.nn.functional.rms_norm(x + r, (200,), norm.weight, 1e-6)
    assert torch.allclose(y, want)
    a, b = torch.nn.functional.linear(y, gated.weight).chunk(2, -1)
    assert torch.allclose(gated(y), torch.nn.functional.silu(a) * b)
    w, ws = quantize_weight(gated.weight.detach())
    q, qs = quantize(x)
    B.check_codes(q, qs, x.double(), torch.zeros(6, 200, dtype=torch.float64))
    B.check_codes(w, ws, gated.weight.detach().double(), torch.zeros(60, 200, dtype=torch.float64), weight=True)
    within(linear_fp8(q, qs, w, ws, torch.ones(60, dtype=dtype), act="gelu", dtype=dtype), B.linear_codes(q, qs, w, ws, torch.ones(60, dtype=dtype), None, "gelu", dtype), "product")
    got = rms_norm_fp8(x, norm.weight.detach(), 1e-6, r)
    assert torch.equal(got[2], s) and torch.equal(got[0].float(), quantize(rms_norm(x, norm.weight.detach(), 1e-6, r)[0])[0].float())
    with pytest.raises(RuntimeError, match="no gradient"):
        quantize(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError):
        linear_fp8(q, qs[:, :1], w, ws)


def test_distillation_on_the_cpu():
    from addernetcuda_amd.distill import distillation_loss
    g = torch.Generator().manual_seed(2)
    l = torch.randn(9, 40, generator=g, dtype=torch.float64).requires_grad_(True)
    t, i = torch.randn(9, 40, generator=g, dtype=torch.float64).topk(6, 1)
    y = torch.randint(0, 40, (9,), generator=g)
    t[0] = -float("inf")
    t[1, 2:] = -float("inf")
    y[3] = -100
    for labels in (y, None):
        for alpha in (0.0, 0.3, 1.0):
            loss = distillation_loss(l, t, i, labels, 3.0, alpha)
            want = B.distillation(l, t, i, labels, 3.0, alpha, -100)
            assert abs(float(loss.detach() - want["loss"][0])) < 1e-12
            assert torch.allclose(torch.autograd.grad(loss, l)[0], want["grad"][0], atol=1e-12)
    assert float(distillation_loss(l, t, i, torch.full_like(y, -100)).detach()) == 0
    i[0], i[1, 3] = -1, 99   # (beside -infinity: any number)
    i[5, 2] = 40
    y[6] = -3
    loss = distillation_loss(l, t, i, y, 2.0, 0.5)
    assert torch.isnan(loss.detach())
    bad = torch.isnan(torch.autograd.grad(loss, l)[0]).all(1)
    assert bad.nonzero().flatten().tolist() == [5, 6]


def test_8_bit_layers_keep_their_types():
    from addernetcuda_amd.fp8 import CODES, LinearFp8
    from addernetcuda_amd.linear import LinearAct
    made = LinearFp8.of(LinearAct(130, 20, act="relu"))
    x = torch.randn(3, 130)
    with torch.no_grad():
        want = made(x)
    for change in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu"), lambda m: m.float()):
        change(made)
        assert made.weight.dtype == CODES and made.weight_scale.dtype == made.bias.dtype == torch.float32
        with torch.no_grad():
            assert torch.equal(made(x), want)
    assert not list(made.parameters()) and set(made.state_dict()) == {"weight", "weight_scale", "bias"}
    assert LinearFp8(8, 8).to("meta").weight.device.type == "meta"


def test_gated_sizes_take_their_kernels_and_no_size_another():
    import random
    from tests.test_gpu_gated import BF16, F32, KERNELS, gated_kernel
    for (dtype, *kernel), (rows, k, h) in KERNELS.items():
        assert gated_kernel(rows, k, h, dtype, kernel[0] == 2) == tuple(kernel), (dtype, kernel)
    r = random.Random(7)
    for _ in range(10000):
        rows, k, h = (int(2 ** r.uniform(0, 15)) for _ in range(3))
        for dtype in (F32, BF16):
            for aligned in (False, True):
                for outputs in (1, 2):
                    got = gated_kernel(rows, k, h, dtype, aligned, outputs)
                    assert any(key[:3] == (dtype, *got[:2]) for key in KERNELS), (rows, k, h, got)
