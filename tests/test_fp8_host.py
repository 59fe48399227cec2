"""8-bit codes and layers where torch's operators compute them: CPU tensors, and types that the kernels do not take."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_what_is_no_number_stays_alone_in_its_block(dtype):
    """As in the kernels: the other values of the block keep their codes and their scale; one that is infinite makes the block none."""
    from addernetcuda_amd.fp8 import quantize, quantize_weight, values
    g = torch.Generator().manual_seed(1)
    clean = torch.randn(150, 300, generator=g).to(dtype)
    x = clean.clone()
    clean[0, 5] = 0
    x[0, 5], x[1, 130] = float("nan"), float("inf")
    for make, rows in ((quantize, slice(1, 2)), (quantize_weight, slice(0, 128))):
        (q, s), (want, want_s) = make(x), make(clean)
        v, w = values(q, s), values(want, want_s)
        bad = torch.isnan(v)
        assert bad[0, 5] and bad[rows, 128:256].all()
        bad[0, 5] = bad[rows, 128:256] = False
        assert not bad.any()
        here = torch.ones_like(bad)
        here[0, 5] = here[rows, 128:256] = False
        assert torch.equal(v[here], w[here])
    assert torch.equal(quantize(torch.full((2, 128), float("nan"), dtype=dtype))[1], torch.full((2, 1), 2.0 ** -100) / 448)
    z = torch.cat([x, torch.ones_like(x)], 1)
    assert torch.equal(torch.isnan(values(*quantize(z, gate="none"))), torch.isnan(values(*quantize(x))))
