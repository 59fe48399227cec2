"""Each kernel that an 8-bit product can take -- few rows (1) by 16 or 32 of them, streamed (2) by its shape -- with shares of k and without, at a size that takes it: widths
that are a multiple of neither 16 nor 128, so that both operands are copied and the last block is masked beside the shares, and widths of whole blocks."""
import ctypes
import random

import pytest
import torch

F32, BF16 = torch.float32, torch.bfloat16
# (type, family and shape, shares of k): sizes (rows, k, n)
KERNELS = {(F32, 101, False): [(5, 1003, 70)], (F32, 102, False): [(17, 515, 40)], (F32, 200, False): [(1531, 203, 1900), (2048, 256, 2048)],
           (F32, 200, True): [(1263, 3373, 802), (70, 5120, 6925)], (F32, 201, False): [(27, 1, 1), (300, 300, 200)], (F32, 201, True): [(2, 7220, 1), (40, 7168, 60)],
           (BF16, 101, False): [(5, 1003, 70)], (BF16, 102, False): [(17, 515, 40)], (BF16, 200, False): [(1531, 203, 1900), (2048, 256, 2048)],
           (BF16, 200, True): [(1373, 3213, 755), (70, 5760, 2862)], (BF16, 201, False): [(40, 141, 30), (300, 300, 200)], (BF16, 201, True): [(1, 6156, 1), (40, 7168, 60)],
           (BF16, 202, False): [(1300, 201, 5906), (4096, 1024, 4096)], (BF16, 202, True): [(1504, 5674, 2900), (1504, 5760, 2900)]}


def kernel(rows, k, n, dtype):
    from addernetcuda_amd._lib import lib
    v = ctypes.c_int()
    assert lib.adder_linear_codes_kernel(rows, k, n, int(dtype == BF16), ctypes.byref(v)) == 0
    return v.value // 100, v.value % 100 > 1


def test_sizes_take_their_kernels_and_no_size_another():
    for (dtype, *want), sizes in KERNELS.items():
        for size in sizes:
            assert kernel(*size, dtype) == tuple(want), (dtype, want, size)
    r = random.Random(3)
    for _ in range(20000):
        size = [int(2 ** r.uniform(0, 14)) for _ in range(3)]
        for dtype in (F32, BF16):
            assert (dtype, *kernel(*size, dtype)) in KERNELS, size


@pytest.mark.gpu
@pytest.mark.parametrize("key", KERNELS, ids=str)
def test_kernels(key, gpu):
    from addernetcuda_amd.fp8 import linear_fp8
    from tests import block_bounds as B
    from tests.layer_bounds import within
    from tests.test_gpu_fp8 import codes, normal, weight
    dtype = key[0]
    for rows, k, n in KERNELS[key]:
        (x, xs), (w, ws) = codes(rows, k), weight(n, k)
        b, r = normal(n, seed=2).to(dtype).cuda(), normal(rows, n, seed=3).to(dtype).cuda()
        plain, full = linear_fp8(x, xs, w, ws, dtype=dtype), linear_fp8(x, xs, w, ws, b, r, "gelu", dtype)
        for at in [slice(0, 300), slice(rows - 300, rows)] if rows > 300 else [slice(0, rows)]:
            within(plain[at], B.linear_codes(x[at], xs[at], w, ws, None, None, "none", dtype), f"{(rows, k, n)}, rows {at}")
            within(full[at], B.linear_codes(x[at], xs[at], w, ws, b, r[at], "gelu", dtype), f"{(rows, k, n)} with everything, rows {at}")
        assert torch.equal(plain, linear_fp8(x, xs, w, ws, dtype=dtype))
