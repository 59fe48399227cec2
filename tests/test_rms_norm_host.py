"""``rms_norm`` and ``rms_norm_fp8`` with ``eps=None``: as ``F.rms_norm``'s, the machine epsilon of the type that the norm is computed in."""
import pytest
import torch
import torch.nn.functional as F


def values(dtype):
    return (torch.randn(7, 200, generator=torch.Generator().manual_seed(2)) * 2.0 ** -11).to(dtype)   # (mean squares of some two such epsilons)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_no_eps(dtype):
    from addernetcuda_amd.fp8 import rms_norm_fp8
    from addernetcuda_amd.rms_norm import rms_norm
    x = values(dtype)
    eps = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps
    assert torch.equal(rms_norm(x, None, None), F.rms_norm(x, (200,), None, None))
    y, s = rms_norm(x, None, None, residual=x)
    assert torch.equal(s, x + x) and torch.equal(y, rms_norm(x, None, eps, residual=x)[0])
    for got, want in zip(rms_norm_fp8(x, None, None), rms_norm_fp8(x, None, eps)):
        assert torch.equal(got.float(), want.float())
    with pytest.raises(RuntimeError, match="must not be negative"):
        rms_norm(x, None, -1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_eps_in_the_kernels(dtype, gpu):
    from addernetcuda_amd.fp8 import rms_norm_fp8
    from addernetcuda_amd.rms_norm import rms_norm
    x, eps = values(dtype).cuda(), torch.finfo(torch.float32).eps
    assert torch.equal(rms_norm(x, None, None), rms_norm(x, None, eps))
    assert all(torch.equal(p, q) for p, q in zip(rms_norm(x, None, None, residual=x), rms_norm(x, None, eps, residual=x)))
    for got, want in zip(rms_norm_fp8(x, None, None), rms_norm_fp8(x, None, eps)):
        assert torch.equal(got.float(), want.float())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y, s = rms_norm(x.bfloat16(), None, None, residual=x.float())
        assert torch.equal(y, rms_norm(s, None, eps))
