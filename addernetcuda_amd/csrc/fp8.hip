// e4m3 codes with a scale for each block: of 128 neighbouring values of a row (activations), or of 128 x 128 values (weights).
//     top = max(largest magnitude of the block, 2^-100),   scale = top / 448,   code = e4m3(v 448 / top), to nearest even
// A value that is no number keeps a code that is none; a block with an infinite one has an infinite scale and is no number as a whole.
// Memory decides: every value is read once, a byte written.  8192 x 8192 in bfloat16 36 us (5.6 TB/s), with a SiLU's gate 27 us (6.2 TB/s); a weight of
// 4096 x 4096 12 us.
#include "blocks.hpp"

namespace adder {

static constexpr int kQuantThreads = 256;

// 128 / V neighbouring lanes have a block; the blocks lie one after the other.  GATED: rows of 2 D values, v = act(first half) * second half.
template <class T, bool GATED>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(const T *__restrict__ x, long x_stride, Act act, uint8_t *__restrict__ q,
                                                                 float *__restrict__ scale, long blocks, int per_row, int D) {
    constexpr int V = Chunk<T>::n, L = kCodeBlock / V;
    const int lane = threadIdx.x % L;
    for (long i = ((long)blockIdx.x * kQuantThreads + threadIdx.x) / L; i < blocks; i += (long)gridDim.x * kQuantThreads / L) {
        const long row = blocks <= 0x7fffffffL ? (long)((unsigned)i / (unsigned)per_row) : i / per_row;
        const int at = (int)(i - row * per_row) * kCodeBlock + lane * V;
        float v[V], top = kCodeLeast;
        load_part(x + row * x_stride + at, D - at, v);
        if constexpr (GATED) {
            float u[V];
            load_part(x + row * x_stride + D + at, D - at, u);
            switch (act) {   // (outside the loop: one branch for all values)
                case Act::relu:
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = activate<kExactAct<T>>(v[e], Act::relu) * u[e];
                    break;
                case Act::gelu:
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = activate<kExactAct<T>>(v[e], Act::gelu) * u[e];
                    break;
                case Act::silu:
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = activate<kExactAct<T>>(v[e], Act::silu) * u[e];
                    break;
                default:
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] *= u[e];
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, at + e < D ? fabsf(v[e]) : 0.f);
        top = lanes_max<L>(top);
        const float by = kCodeTop / top;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= by;
        store_codes(q + row * D + at, D - at, v);
        if (lane == 0) scale[i] = top / kCodeTop;
    }
}

// A workgroup a block of 128 x 128: 128 / V lanes have a row of it.  Run once for a weight.
template <class T>
__global__ __launch_bounds__(kQuantThreads) void quantize_weight_kernel(const T *__restrict__ w, long w_stride, uint8_t *__restrict__ q,
                                                                        float *__restrict__ scale, long rows, int D) {
    constexpr int V = Chunk<T>::n, L = kCodeBlock / V, PER = kQuantThreads / L, STEPS = kCodeBlock / PER;
    __shared__ float lds[kQuantThreads / 64];
    const int at = (int)blockIdx.x * kCodeBlock + (int)(threadIdx.x % L) * V;
    const long row0 = (long)blockIdx.y * kCodeBlock + threadIdx.x / L;
    float v[STEPS][V], top = kCodeLeast;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const long row = row0 + s * PER;
        load_part(w + row * w_stride + at, row < rows ? D - at : 0, v[s]);
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(v[s][e]));
    }
    top = lanes_max<64>(top);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQuantThreads / 64; ++i) top = fmaxf(top, lds[i]);
    const float by = kCodeTop / top;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const long row = row0 + s * PER;
#pragma unroll
        for (int e = 0; e < V; ++e) v[s][e] *= by;
        store_codes(q + row * D + at, row < rows ? D - at : 0, v[s]);
    }
    if (threadIdx.x == 0) scale[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = top / kCodeTop;
}

template <class T>
int launch_quantize(const T *x, long x_stride, bool gated, Act act, uint8_t *q, float *scale, long rows, int D, hipStream_t s) {
    const int per_row = (D + kCodeBlock - 1) / kCodeBlock;
    const long blocks = rows * per_row, groups = ceil_div_l(blocks, kQuantThreads / (kCodeBlock / Chunk<T>::n));
    const dim3 grid((unsigned)(groups < 16384 ? groups : 16384)), threads(kQuantThreads);
    if (gated) hipLaunchKernelGGL((quantize_kernel<T, true>), grid, threads, 0, s, x, x_stride, act, q, scale, blocks, per_row, D);
    else hipLaunchKernelGGL((quantize_kernel<T, false>), grid, threads, 0, s, x, x_stride, act, q, scale, blocks, per_row, D);
    return check_launch();
}
template <class T>
int launch_quantize_weight(const T *w, long w_stride, uint8_t *q, float *scale, long rows, int D, hipStream_t s) {
    hipLaunchKernelGGL(quantize_weight_kernel<T>, dim3((unsigned)ceil_div(D, kCodeBlock), (unsigned)ceil_div_l(rows, kCodeBlock)), dim3(kQuantThreads), 0, s,
                       w, w_stride, q, scale, rows, D);
    return check_launch();
}

#define ADDER_CODES_INSTANCE(T)                                                                                          \
    template int launch_quantize<T>(const T *, long, bool, Act, uint8_t *, float *, long, int, hipStream_t);              \
    template int launch_quantize_weight<T>(const T *, long, uint8_t *, float *, long, int, hipStream_t);
ADDER_CODES_INSTANCE(float)
ADDER_CODES_INSTANCE(bf16_t)

}  // namespace adder
