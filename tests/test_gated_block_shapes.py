"""What is added to a gated block's input may be of any shape that meets it, as between torch's modules."""
import copy

import pytest
import torch

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("x,added", [((4, 5, 48), (48,)), ((4, 5, 48), (4, 1, 48)), ((5, 48), (4, 5, 48)), ((4, 1, 48), (1, 5, 48)), ((4, 5, 48), (4, 5, 48))])
def test_what_is_added_is_broadcast(x, added, device):
    """float32: three products of 48 or 64 terms between the two, each off by 1e-6 of its size."""
    from addernetcuda_amd.fp8 import serve_fp8
    from addernetcuda_amd.models import GatedMLP
    torch.manual_seed(2)
    block, plain = GatedMLP(48, 64).to(device), GatedMLP(48, 64, fused=False).to(device)
    plain.load_state_dict(block.state_dict())
    x, added = torch.randn(x, device=device), torch.randn(added, device=device)
    got, want = block(x, added=added), plain(x, added=added)
    assert got.shape == want.shape == torch.broadcast_shapes(x.shape, added.shape)
    assert torch.allclose(got, want, rtol=1e-4, atol=1e-4)
    served = serve_fp8(torch.nn.Sequential(copy.deepcopy(block)))[0]
    with torch.no_grad():
        assert float((served(x, added=added) - want).norm()) < 0.1 * float(want.norm())
