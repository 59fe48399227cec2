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


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_layers_answer_in_the_type_of_their_input(dtype, device):
    """Types that the products do not have: the float32 result, rounded once (float64: as it is)."""
    from addernetcuda_amd.fp8 import LinearFp8, quantize
    g = torch.Generator().manual_seed(4)
    layer = torch.nn.Linear(130, 20)
    x, r = torch.randn(3, 130, generator=g).to(dtype).to(device), torch.randn(3, 20, generator=g).to(dtype).to(device)
    made = LinearFp8.of(layer).to(device)
    gated = LinearFp8.of(torch.nn.Linear(65, 20), gate="silu").to(device)
    with torch.no_grad():
        assert torch.equal(made(x), made(x.float()).to(dtype)) and made(x).dtype == dtype
        for y in (made(x, residual=r), made(quantize(x), residual=r)):
            assert y.dtype == dtype and torch.equal(y, made(x.float(), residual=r.float()).to(dtype))
        assert gated(x).dtype == dtype


def test_a_gated_layer_by_itself_is_refused():
    """Its halves meet in the layer behind it: ``of`` would give both, activated, side by side."""
    from addernetcuda_amd.fp8 import LinearFp8, RMSNormFp8, serve_fp8
    from addernetcuda_amd.gated import GatedLinear
    from addernetcuda_amd.models import GatedMLP
    with pytest.raises(ValueError, match="gated"):
        LinearFp8.of(GatedLinear(256, 128))
    block = torch.nn.Sequential(GatedMLP(64, 40, act="gelu"))
    weight = block[0].gated.weight.detach().clone()
    serve_fp8(block)
    assert isinstance(block[0].norm, RMSNormFp8) and block[0].gated.act == "none" and block[0].down.gate == "gelu"
    assert block[0].gated.weight.shape == weight.shape == (80, 64)
    with torch.no_grad():
        assert block(torch.randn(5, 64)).shape == (5, 64)
    with pytest.raises(ValueError):
        serve_fp8(block)


@pytest.mark.gpu
def test_torchs_operators_give_the_kernels_codes_and_scales(gpu):
    """float64 values that are float32 numbers, which torch's operators take: bit for bit what the kernels make of those."""
    from addernetcuda_amd.fp8 import quantize, quantize_weight
    x = (torch.randn(300, 400, generator=torch.Generator().manual_seed(6)) * torch.exp(torch.randn(300, 1, generator=torch.Generator().manual_seed(7)))).cuda()
    for make in (quantize, quantize_weight):
        for got, want in zip(make(x.double()), make(x)):
            assert torch.equal(got.float(), want.float())
