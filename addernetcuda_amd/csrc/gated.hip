// Gated linear layer: g = x wg' + bg, u = x wu' + bu, y = act(g) u (linear*.hip); here what its backward takes from g and u,
//     dg = dy u act'(g),   du = dy act(g),
// as one matrix of rows [dg du], for the two products gx = [dg du] w and gw = [dg du]' x, and the bias's gradient, its column sums.
// Memory decides: dy, g and u are read and dg and du written, 8192 x 4096 in bfloat16 with a SiLU 55 us (6.1 TB/s).  bfloat16: g and u are what the forward kept of them (keep_gate, keep_group), dz is
// rounded to the type of the products' operands, and the bias's sums are not.
#include "blocks.hpp"

namespace adder {

static constexpr int kGatedThreads = 256;

template <class T, Act ACT>
__global__ __launch_bounds__(kGatedThreads) void gated_bwd_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ z, T *__restrict__ dz,
                                                                  float *__restrict__ part, long rows, long N) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = ((long)blockIdx.x * 64 + lane) * V;
    const int left = N - n < V ? (int)(N - n < 0 ? 0 : N - n) : V;
    float sum[2][V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[0][e] = sum[1][e] = 0.f;
    for (long m = (long)blockIdx.y * 4 + wave; m < rows; m += (long)gridDim.y * 4) {
        float d[V], g[V], u[V];
        load_part(dy + m * dy_stride + n, left, d);
        const uint4 gate = load_raw_part(z + m * 2 * N + n, left);
        if constexpr (ACT == Act::relu) unpack(gate, g);
        else unpack_kept(gate, g);
        unpack_kept(load_raw_part(z + m * 2 * N + N + n, left), u);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float a, s;
            both<kExactAct<T>>(g[e], ACT, a, s);
            // (a ReLU selects: where it is off, an infinite dy or one that is no number goes no further)
            g[e] = ACT == Act::relu && s == 0.f ? 0.f : d[e] * u[e] * s;
            u[e] = ACT == Act::relu && s == 0.f ? 0.f : d[e] * a;
            sum[0][e] += g[e];
            sum[1][e] += u[e];
        }
        if (dz) {
            store_part(dz + m * 2 * N + n, left, g);
            store_part(dz + m * 2 * N + N + n, left, u);
        }
    }
    if (!part) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (h) __syncthreads();
#pragma unroll
        for (int e = 0; e < V; ++e) lds[wave][e * 64 + lane] = sum[h][e];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int i = 1; i < 4; ++i) sum[h][e] += lds[i][e * 64 + lane];
                if (e < left) part[(long)blockIdx.y * 2 * N + h * N + n + e] = sum[h][e];
            }
        }
    }
}

// Shares of the rows: a row a wave, as long as there are no more workgroups than four a compute unit
int gated_bwd_parts(long rows, long N) {
    const long columns = ceil_div_l(N, 512), need = ceil_div_l(rows, 4), most = ceil_div_l(1024, columns);
    return (int)(need < most ? need : most);
}

template <class T>
int launch_gated_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div_l(N, 64 * Chunk<T>::n), gated_bwd_parts(rows, N)), threads(kGatedThreads);
    switch (act) {
        case Act::relu: hipLaunchKernelGGL((gated_bwd_kernel<T, Act::relu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        case Act::gelu: hipLaunchKernelGGL((gated_bwd_kernel<T, Act::gelu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        case Act::silu: hipLaunchKernelGGL((gated_bwd_kernel<T, Act::silu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        default: hipLaunchKernelGGL((gated_bwd_kernel<T, Act::none>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N);
    }
    return check_launch();
}
template int launch_gated_bwd<float>(const float *, long, const float *, float *, float *, Act, long, long, hipStream_t);
template int launch_gated_bwd<bf16_t>(const bf16_t *, long, const bf16_t *, bf16_t *, float *, Act, long, long, hipStream_t);

}  // namespace adder
