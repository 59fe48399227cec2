"""What a bfloat16 gated layer keeps of its two sums for the backward, element by element: the input is the identity, so that the sums are the weights, and
without an activation the gradient of one half of the weight is what was kept of the other."""
import pytest
import torch

pytestmark = pytest.mark.gpu
V = 2.0 ** -8
# few rows, tiles through registers (a width of 8 k + 4) and streamed ones, with shares of k or without
SIZES = [(16, 24), (36, 30), (68, 100), (132, 70), (264, 136), (520, 1030)]


def gradients(wg, wu, act, dy=None):
    """The gradients of both halves of the weight for an input that is the identity."""
    from addernetcuda_amd.gated import gated_linear
    h, k = wg.shape
    x = torch.eye(k, device="cuda", dtype=torch.bfloat16)
    w = torch.cat([wg, wu]).requires_grad_(True)
    y = gated_linear(x, w, None, act)
    return torch.autograd.grad(y, w, torch.ones_like(y) if dy is None else dy)[0].split(h)


def spread(k, h, lo, hi, seed):
    """Values of all magnitudes from 2^lo to 2^hi, neighbours of any; some are zero."""
    g = torch.Generator().manual_seed(seed + k)
    v = torch.randn(h, k, generator=g).sign() * torch.exp2(torch.rand(h, k, generator=g) * (hi - lo) + lo)
    v[torch.rand(h, k, generator=g) < 0.02] = 0
    return v.bfloat16().cuda()


@pytest.mark.parametrize("lo,hi", [(-30.0, 0.0), (-16.0, 1.0), (-13.0, 15.0), (0.0, 20.0), (-100.0, -60.0)])
@pytest.mark.parametrize("k,h", SIZES)
def test_small_values_beside_large_ones(k, h, lo, hi, gpu):
    """Off by half a step of bfloat16 (the first of four by a whole one) at most, whatever stands beside it, and half a step for dz."""
    wg, wu = spread(k, h, lo, hi, 1), spread(k, h, lo, hi, 2)
    first = torch.arange(h, device="cuda")[:, None] % 4 == 0
    far = torch.where(first, 2 * V, V).double()
    for got, want in zip(gradients(wg, wu, "none"), (wu.double(), wg.double())):
        assert not got[want == 0].any()
        assert ((got.double() - want).abs() <= ((1 + far) * (1 + V) - 1) * want.abs()).all()


@pytest.mark.parametrize("k,h", SIZES)
def test_a_relus_gate_is_kept_as_it_is(k, h, gpu):
    """bfloat16 weights are sums that bfloat16 holds: the up half's gradient is the gate's positive part itself."""
    wg, wu = spread(k, h, -20.0, 4.0, 3), spread(k, h, -3.0, 3.0, 4)
    gate, up = gradients(wg, wu, "relu")
    assert torch.equal(up, wg.clamp(min=0))
    assert torch.equal(gate != 0, (wg > 0) & (wu != 0))


def test_first_columns_are_not_all_off_the_same_way(gpu):
    """The last bit of the first of four says how they are kept: over many values that makes them neither smaller nor larger.  A value's error is at
    most a step, 2^-7 of it, evenly on both sides: the mean of n is within 5 of its deviations, 2^-7 / sqrt(n), of zero; one side would be 2^-8."""
    k, h = 512, 1024
    for lo, hi in ((-4.0, 4.0), (17.0, 20.0)):
        wg, wu = spread(k, h, lo, hi, 5), spread(k, h, lo, hi, 6)
        for got, want in zip(gradients(wg, wu, "none"), (wu.double(), wg.double())):
            some = want[::4] != 0
            off = (got[::4].double() / want[::4])[some] - 1
            assert abs(float(off.mean())) < 5 * 2 * V / off.numel() ** 0.5 + 2.0 ** -13
