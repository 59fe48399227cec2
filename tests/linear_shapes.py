"""A size for every compiled shape of the linear layers' product kernels (csrc/linear*.hip) in every layout that they are compiled for -- the forward
has k along the rows of both operands, the input gradient across those of the second, the weight gradient across those of both --, with the
sums in one launch and as shares of k where there are both.  No side is a whole tile where that can be had.
test_linear_shapes holds the list against the library's own answers, test_gpu_linear_shapes runs it."""
import ctypes

F32, BF16 = 0, 1        # adder_type
FWD, GX, GW = 0, 1, 2   # the product of adder_linear_kernel
ROWS, STREAM, STAGED = 1, 2, 3


def linear_kernel(rows, k, n, product, dtype, aligned, outputs=1):
    """(family, shape, shares of k) of the kernel that the library takes for a layer k -> n."""
    from addernetcuda_amd._lib import lib, check
    kernel = ctypes.c_int(-1)
    check(lib.adder_linear_kernel(rows, k, n, product, dtype, int(aligned), outputs, ctypes.byref(kernel)), "adder_linear_kernel")
    return kernel.value // 10000, kernel.value // 100 % 100, kernel.value % 100


# (type, product, family, shape, whether k is shared): (rows, in_features, out_features).  Streamed: 256 x 256, 128 x 256, 128 x 128 and 64 x 64 results a workgroup
# (the second is taken for shares of long sums alone); staged: 128 x 128, 64 x 64 and (float32) both with twice the waves.
SHAPES = {
    (F32, FWD, ROWS, 1, False): (1, 162, 72),
    (F32, FWD, ROWS, 2, False): (23, 167, 65),
    (F32, FWD, ROWS, 4, False): (37, 170, 73),
    (F32, FWD, STAGED, 0, False): (2893, 97, 1733),
    (F32, FWD, STAGED, 0, True): (1214, 1240, 1815),
    (F32, FWD, STAGED, 1, False): (1034, 186, 79),
    (F32, FWD, STAGED, 1, True): (68, 381, 73),
    (F32, FWD, STAGED, 2, False): (2040, 163, 2033),
    (F32, FWD, STAGED, 2, True): (867, 808, 1209),
    (F32, FWD, STAGED, 3, False): (1026, 276, 173),
    (F32, FWD, STAGED, 3, True): (1, 4152, 1),
    (F32, GX, STAGED, 0, False): (2893, 1733, 97),
    (F32, GX, STAGED, 0, True): (1182, 1708, 1146),
    (F32, GX, STAGED, 1, False): (76, 88, 157),
    (F32, GX, STAGED, 1, True): (69, 66, 167),
    (F32, GX, STAGED, 2, False): (2040, 2033, 163),
    (F32, GX, STAGED, 2, True): (770, 1263, 758),
    (F32, GX, STAGED, 3, False): (520, 333, 265),
    (F32, GX, STAGED, 3, True): (1, 1, 4135),
    (F32, GW, STAGED, 0, False): (95, 1481, 3402),
    (F32, GW, STAGED, 0, True): (1229, 1802, 1170),
    (F32, GW, STAGED, 1, False): (158, 91, 85),
    (F32, GW, STAGED, 1, True): (161, 65, 82),
    (F32, GW, STAGED, 2, False): (163, 2033, 2040),
    (F32, GW, STAGED, 2, True): (750, 1240, 804),
    (F32, GW, STAGED, 3, False): (271, 430, 409),
    (F32, GW, STAGED, 3, True): (4103, 1, 1),
    (BF16, FWD, ROWS, 1, False): (1, 322, 65),
    (BF16, FWD, ROWS, 2, False): (25, 515, 67),
    (BF16, FWD, ROWS, 4, False): (37, 459, 75),
    (BF16, FWD, STREAM, 0, False): (3308, 1096, 3915),
    (BF16, FWD, STREAM, 0, True): (2406, 14488, 1851),
    (BF16, FWD, STREAM, 1, True): (927, 18936, 6099),
    (BF16, FWD, STREAM, 2, False): (386, 328, 7083),
    (BF16, FWD, STREAM, 2, True): (1099, 4520, 1003),
    (BF16, FWD, STREAM, 3, False): (83, 328, 65),
    (BF16, FWD, STREAM, 3, True): (84, 1096, 67),
    (BF16, FWD, STAGED, 0, False): (1540, 735, 1960),
    (BF16, FWD, STAGED, 0, True): (920, 3950, 1203),
    (BF16, FWD, STAGED, 1, False): (65, 323, 77),
    (BF16, FWD, STAGED, 1, True): (66, 1085, 71),
    (BF16, GX, STREAM, 0, False): (4329, 2904, 984),
    (BF16, GX, STREAM, 0, True): (844, 5352, 7912),
    (BF16, GX, STREAM, 1, True): (3669, 1432, 17312),
    (BF16, GX, STREAM, 2, False): (385, 7088, 336),
    (BF16, GX, STREAM, 2, True): (422, 2328, 3784),
    (BF16, GX, STREAM, 3, False): (67, 72, 392),
    (BF16, GX, STREAM, 3, True): (83, 72, 1176),
    (BF16, GX, STAGED, 0, False): (2440, 2074, 157),
    (BF16, GX, STAGED, 0, True): (1294, 810, 3417),
    (BF16, GX, STAGED, 1, False): (71, 71, 345),
    (BF16, GX, STAGED, 1, True): (65, 78, 1042),
    (BF16, GW, STREAM, 0, False): (974, 4575, 2776),
    (BF16, GW, STREAM, 0, True): (6195, 2620, 1576),
    (BF16, GW, STREAM, 1, True): (20712, 924, 5992),
    (BF16, GW, STREAM, 2, False): (331, 8376, 336),
    (BF16, GW, STREAM, 2, True): (4142, 1093, 952),
    (BF16, GW, STREAM, 3, False): (379, 75, 72),
    (BF16, GW, STREAM, 3, True): (1094, 66, 72),
    (BF16, GW, STAGED, 0, False): (137, 1752, 2947),
    (BF16, GW, STAGED, 0, True): (3803, 923, 1109),
    (BF16, GW, STAGED, 1, False): (374, 68, 68),
    (BF16, GW, STAGED, 1, True): (947, 72, 85),
}
