"""8-bit products of rows far from each other: the last token of long sequences, a weight's rows out of a wide matrix."""
import pytest
import torch

from tests import block_bounds as B
from tests.layer_bounds import within
from tests.test_gpu_fp8 import codes, weight

pytestmark = pytest.mark.gpu


def far(t, stride):
    """The same rows, `stride` codes apart."""
    big = torch.zeros(t.shape[0] * stride, dtype=torch.uint8, device="cuda").view(t.shape[0], stride)
    big[:, -t.shape[1]:] = t.view(torch.uint8)
    return big.view(torch.float8_e4m3fn)[:, -t.shape[1]:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("stride", [(1 << 23) - 16, 1 << 23, (1 << 23) + 4096, (1 << 23) + 7])
@pytest.mark.parametrize("rows,k,n", [(3, 512, 40), (70, 200, 40)])
def test_rows_far_apart(rows, k, n, stride, dtype, gpu):
    from addernetcuda_amd.fp8 import linear_fp8
    (x, xs), (w, ws) = codes(rows, k), weight(n, k)
    want = B.linear_codes(x, xs, w, ws, None, None, "none", dtype)
    assert far(x, stride).stride(0) == stride
    within(linear_fp8(far(x, stride), xs, w, ws, dtype=dtype), want, "x")
    within(linear_fp8(x, xs, far(w, stride), ws, dtype=dtype), want, "weight")


def test_the_last_token_of_long_sequences(gpu):
    from addernetcuda_amd.fp8 import linear_fp8, quantize
    x = torch.randn(4, 2100, 4096, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    (q, s), (w, ws) = quantize(x), weight(300, 4096)
    last = q[:, -1], s[:, -1]
    assert last[0].stride(0) > 1 << 23
    within(linear_fp8(*last, w, ws), B.linear_codes(*last, w, ws, None, None, "none", torch.bfloat16), "last token")
