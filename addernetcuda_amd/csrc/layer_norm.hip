// Layer normalisation over the last dimension of a tensor, forward and backward:
//     mean, var = of a row's D values (biased),  rstd = 1 / sqrt(var + eps),  h = (x - mean) * rstd,  y = h * w + b
//     g = dy * w,  gx = rstd * (g - mean(g) - h * mean(g * h)),  gw = sum over rows of dy * h,  gb = sum over rows of dy
// Memory decides: the forward has to read x and write y, the backward to read x and dy and write gx.  A row stays in registers
// from its one load on (G lanes with at most 16 values each), so the variance is that of the differences from the mean, with
// no second read and none of the cancellation of E[x^2] - mean^2.  All sums are 32 bits.
// 16384 x 1024 in bfloat16: forward 14.9 us (4.5 TB/s; a copy of as much takes 10), backward 19.2 us (5.2 TB/s) and 3.8 us for the
// fold of the columns; 3001 x 777 in float32 8.1, 9 and 3 us; 8 x 512 3.2 us, a launch.
#include "layers.hpp"

namespace adder {

static constexpr int kNormValues = 16;    // per lane
template <class T>
static constexpr int kNormChunks = kNormValues / Chunk<T>::n;
static constexpr int kNormFwdThreads = 256, kNormBwdThreads = 512;

// Sum over the G lanes that share a row, in every one of them.  G > 64: through LDS, and every wave of the workgroup has to come.
template <int G>
__device__ __forceinline__ float row_sum(float v, float *lds) {
    v = lanes_sum<(G < 64 ? G : 64)>(v);
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6, first = wave / (G / 64) * (G / 64);
        __syncthreads();   // (the last sum has been read)
        if ((threadIdx.x & 63) == 0) lds[wave] = v;
        __syncthreads();
        v = lds[first];
#pragma unroll
        for (int i = 1; i < G / 64; ++i) v += lds[first + i];
    }
    return v;
}

// 1 / sqrt(var + eps) of a row from the sum of the squares of its values' differences from the (rounded) mean and the mean of those differences: `rest`
// is the mean's rounding, without which a row whose values are large beside their spread loses its digits.  Where the squares leave the range of a
// float the variance is infinite and the row becomes its bias, as the formula in float32 has it; where they are not numbers, nor is the row.
__device__ __forceinline__ float norm_rstd(float squares, float inv, float &rest, float eps) {
    const float mean = squares * inv, off = rest * rest;
    const bool holds = mean < __builtin_inff() && off < __builtin_inff();
    rest = holds ? rest : 0.f;
    return 1.f / sqrtf((holds ? fmaxf(fmaf(squares, inv, -off), 0.f) : mean < __builtin_inff() ? off : mean) + eps);
}

template <class T, class W, int G>
__global__ __launch_bounds__(G > kNormFwdThreads ? G : kNormFwdThreads) void layer_norm_fwd_kernel(
    const T *__restrict__ x, long x_stride, const W *__restrict__ w, const W *__restrict__ b, T *__restrict__ y,
    float *__restrict__ mean, float *__restrict__ rstd, float eps, long rows, int D) {
    constexpr int V = Chunk<T>::n, C = kNormChunks<T>, THREADS = G > kNormFwdThreads ? G : kNormFwdThreads, PER = THREADS / G;
    __shared__ float lds[16];
    const int lane = threadIdx.x % G;
    const float inv = 1.f / (float)D;
    float wv[C][V], bv[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (lane + c * G) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) { wv[c][e] = 1.f; bv[c][e] = 0.f; }
        if (w) load_values<V>(w + at, D - at, wv[c]);
        if (b) load_values<V>(b + at, D - at, bv[c]);
    }
    for (long base = (long)blockIdx.x * PER; base < rows; base += (long)gridDim.x * PER) {   // (all waves together)
        const long row = base + threadIdx.x / G;
        const int width = row < rows ? D : 0;
        const T *px = x + row * x_stride;
        float v[C][V], s = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) load_part(px + (lane + c * G) * V, width - (lane + c * G) * V, v[c]);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[c][e];
        const float mu = row_sum<G>(s, lds) * inv;
        float q = 0.f, r = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[c][e] -= mu;
                const float d = (lane + c * G) * V + e < D ? v[c][e] : 0.f;
                r += d;
                q = fmaf(d, d, q);
            }
        r = row_sum<G>(r, lds) * inv;
        const float rs = norm_rstd(row_sum<G>(q, lds), inv, r, eps);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf((v[c][e] - r) * rs, wv[c][e], bv[c][e]);
            store_part(y + row * D + (lane + c * G) * V, width - (lane + c * G) * V, o);
        }
        if (mean && lane == 0 && width) {
            mean[row] = mu + r;
            rstd[row] = rs;
        }
    }
}

// The workgroups walk over the rows and keep the columns' sums of dy * h and dy of their rows in registers; at the end the
// lanes of a wave that hold the same columns add theirs, then the waves through LDS, and the workgroup writes one slab of 2 D
// floats, which launch_fold_columns adds up: no atomics, the same bits every run.
template <class T, class W, int G>
__global__ __launch_bounds__(G > kNormBwdThreads ? G : kNormBwdThreads) void layer_norm_bwd_kernel(
    const T *__restrict__ dy, long dy_stride, const T *__restrict__ x, long x_stride, const W *__restrict__ w,
    const float *__restrict__ mean, const float *__restrict__ rstd, T *__restrict__ gx, float *__restrict__ part, long rows, int D) {
    constexpr int V = Chunk<T>::n, C = kNormChunks<T>, THREADS = G > kNormBwdThreads ? G : kNormBwdThreads, PER = THREADS / G;
    __shared__ float lds[16];
    constexpr int LANES = G < 64 ? G : 64, SHARE = G < 64 ? THREADS / 64 : PER;   // lanes of a wave with columns of their own; LDS copies of the columns
    __shared__ __align__(16) float fold[SHARE > 1 ? SHARE * G * kNormValues : 4];
    const int lane = threadIdx.x % G;
    const float inv = 1.f / (float)D;
    float wv[C][V], sw[C][V], sb[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (lane + c * G) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) { wv[c][e] = 1.f; sw[c][e] = sb[c][e] = 0.f; }
        if (w) load_values<V>(w + at, D - at, wv[c]);
    }
    for (long base = (long)blockIdx.x * PER; base < rows; base += (long)gridDim.x * PER) {   // (all waves together)
        const long row = base + threadIdx.x / G;
        const int width = row < rows ? D : 0;
        const T *px = x + row * x_stride, *pg = dy + row * dy_stride;
        const float mu = width ? mean[row] : 0.f, rs = width ? rstd[row] : 0.f;
        float h[C][V], g[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            load_part(px + (lane + c * G) * V, width - (lane + c * G) * V, h[c]);
            load_part(pg + (lane + c * G) * V, width - (lane + c * G) * V, g[c]);
        }
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[c][e] = (h[c][e] - mu) * rs;   // (beside the row: not zero, but its g is)
                sw[c][e] = fmaf(g[c][e], h[c][e], sw[c][e]);
                sb[c][e] += g[c][e];
                g[c][e] *= wv[c][e];
                s1 += g[c][e];
                s2 = fmaf(g[c][e], h[c][e], s2);
            }
        s1 = row_sum<G>(s1, lds) * inv;
        s2 = row_sum<G>(s2, lds) * inv;
        if (gx) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = rs * (g[c][e] - s1 - h[c][e] * s2);
                store_part(gx + row * D + (lane + c * G) * V, width - (lane + c * G) * V, o);
            }
        }
    }
    if (!part) return;
    float *slab = part + (size_t)blockIdx.x * 2 * D;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float (&t)[C][V] = k ? sb : sw;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e)
#pragma unroll
                for (int off = LANES; off < 64; off *= 2) t[c][e] += __shfl_xor(t[c][e], off, 64);
        if constexpr (SHARE == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int q = 0; q < V; q += 4) {
                    const float u[4] = {t[c][q], t[c][q + 1], t[c][q + 2], t[c][q + 3]};
                    const int at = (lane + c * G) * V + q;
                    store_part(slab + (size_t)k * D + at, D - at, u);
                }
        } else {
            const int copy = threadIdx.x / (G < 64 ? 64 : G);
            if (k) __syncthreads();
            if ((threadIdx.x & 63) < LANES)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int q = 0; q < V; q += 4)
                        *reinterpret_cast<float4 *>(fold + copy * (G * kNormValues) + (lane + c * G) * V + q) =
                            make_float4(t[c][q], t[c][q + 1], t[c][q + 2], t[c][q + 3]);
            __syncthreads();
            for (int i = threadIdx.x; i < D; i += THREADS) {
                float u = fold[i];
#pragma unroll
                for (int r = 1; r < SHARE; ++r) u += fold[r * (G * kNormValues) + i];
                slab[(size_t)k * D + i] = u;
            }
        }
    }
}

// Rows longer than kNormRegisterWidth: one workgroup a row, which reads it again (from its L2, as long as that holds it) for each of the sums.
static constexpr int kNormWide = 1024;
template <class T, class W>
__global__ __launch_bounds__(kNormWide) void layer_norm_wide_fwd_kernel(const T *__restrict__ x, long x_stride,
                                                                        const W *__restrict__ w, const W *__restrict__ b,
                                                                        T *__restrict__ y, float *__restrict__ mean,
                                                                        float *__restrict__ rstd, float eps, long rows, int D) {
    __shared__ float lds[16];
    const float inv = 1.f / (float)D;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *px = x + row * x_stride;
        float s = 0.f, q = 0.f, r = 0.f;
        for (int i = threadIdx.x; i < D; i += kNormWide) s += ldf(px + i);
        const float mu = row_sum<kNormWide>(s, lds) * inv;
        for (int i = threadIdx.x; i < D; i += kNormWide) {
            const float d = ldf(px + i) - mu;
            r += d;
            q = fmaf(d, d, q);
        }
        r = row_sum<kNormWide>(r, lds) * inv;
        const float rs = norm_rstd(row_sum<kNormWide>(q, lds), inv, r, eps);
        for (int i = threadIdx.x; i < D; i += kNormWide)
            put(y + row * D + i, fmaf((ldf(px + i) - mu - r) * rs, w ? ldf(w + i) : 1.f, b ? ldf(b + i) : 0.f));
        if (mean && threadIdx.x == 0) {
            mean[row] = mu + r;
            rstd[row] = rs;
        }
    }
}

template <class T, class W>
__global__ __launch_bounds__(kNormWide) void layer_norm_wide_gx_kernel(const T *__restrict__ dy, long dy_stride,
                                                                       const T *__restrict__ x, long x_stride,
                                                                       const W *__restrict__ w, const float *__restrict__ mean,
                                                                       const float *__restrict__ rstd, T *__restrict__ gx,
                                                                       long rows, int D) {
    __shared__ float lds[16];
    const float inv = 1.f / (float)D;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *px = x + row * x_stride, *pg = dy + row * dy_stride;
        const float mu = mean[row], rs = rstd[row];
        float s1 = 0.f, s2 = 0.f;
        for (int i = threadIdx.x; i < D; i += kNormWide) {
            const float g = ldf(pg + i) * (w ? ldf(w + i) : 1.f);
            s1 += g;
            s2 = fmaf(g, (ldf(px + i) - mu) * rs, s2);
        }
        s1 = row_sum<kNormWide>(s1, lds) * inv;
        s2 = row_sum<kNormWide>(s2, lds) * inv;
        for (int i = threadIdx.x; i < D; i += kNormWide)
            put(gx + row * D + i, rs * (ldf(pg + i) * (w ? ldf(w + i) : 1.f) - s1 - (ldf(px + i) - mu) * rs * s2));
    }
}

// ... and their columns' sums: a thread a column, gridDim.y shares of the rows, a slab each
template <class T>
__global__ __launch_bounds__(256) void layer_norm_wide_columns_kernel(const T *__restrict__ dy, long dy_stride,
                                                                      const T *__restrict__ x, long x_stride,
                                                                      const float *__restrict__ mean,
                                                                      const float *__restrict__ rstd, float *__restrict__ part,
                                                                      long rows, int D) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= D) return;
    float sw = 0.f, sb = 0.f;
    for (long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float g = ldf(dy + row * dy_stride + i);
        sw = fmaf(g, (ldf(x + row * x_stride + i) - mean[row]) * rstd[row], sw);
        sb += g;
    }
    float *slab = part + (size_t)blockIdx.y * 2 * D;
    slab[i] = sw;
    slab[(size_t)D + i] = sb;
}

// 32 columns and 32 shares of the slabs a workgroup: 2.5 to 5 us, half of it the launch
static constexpr int kFoldColumns = 32, kFoldShares = 32;
template <class T>
__global__ __launch_bounds__(kFoldColumns *kFoldShares) void fold_columns_kernel(const float *__restrict__ part, int parts, int K,
                                                                                 long cols, const FoldOut out) {
    __shared__ float lds[kFoldShares][kFoldColumns];
    const int k = blockIdx.y, cx = threadIdx.x % kFoldColumns, share = threadIdx.x / kFoldColumns;
    const long c = (long)blockIdx.x * kFoldColumns + cx;
    T *o = static_cast<T *>(out.p[k]);
    if (!o) return;
    float t = 0.f;
    if (c < cols)
#pragma unroll 8
        for (int i = share; i < parts; i += kFoldShares) t += part[((size_t)i * K + k) * cols + c];
    lds[share][cx] = t;
    __syncthreads();
    if (share == 0 && c < cols) {
#pragma unroll
        for (int i = 1; i < kFoldShares; ++i) t += lds[i][cx];
        put(o + c, t);
    }
}

template <class T>
int launch_fold_columns(const float *part, int parts, int K, long cols, const FoldOut &out, hipStream_t s) {
    hipLaunchKernelGGL(fold_columns_kernel<T>, dim3((unsigned)ceil_div_l(cols, kFoldColumns), K), dim3(kFoldColumns * kFoldShares), 0,
                       s, part, parts, K, cols, out);
    return check_launch();
}
template int launch_fold_columns<float>(const float *, int, int, long, const FoldOut &, hipStream_t);
template int launch_fold_columns<bf16_t>(const float *, int, int, long, const FoldOut &, hipStream_t);

// Lanes per row: as few as hold it with 16 values each, so that the lanes are full and few steps join them
static int norm_lanes(int D) {
    int g = 8;
    while (g * kNormValues < D) g *= 2;
    return g;
}

// At most three workgroups a compute unit, which walk over the rows with the weight in registers: 512 workgroups take 15.5 us for 16384 x 1024 in
// bfloat16 instead of 13.6, 2048 take 17.9 us for 2048 x 8192 instead of 15.6 and 8.0 for 32768 x 256 instead of 6.9
static int norm_fwd_blocks(long rows, int G) {
    const long per = G > kNormFwdThreads ? 1 : kNormFwdThreads / G, need = ceil_div_l(rows, per), most = 768;
    return (int)(need < most ? need : most);
}

// One workgroup of eight waves a compute unit, each with a slab: 128 take 25.8 us with the fold for 16384 x 1024 in bfloat16 instead of
// 19.2 and 512 take 17.6, but 30.5 for 2048 x 8192 instead of 25.1, whose slabs are as large as its tensors
int layer_norm_bwd_parts(long rows, int D) {
    if (D > kNormRegisterWidth) return (int)(rows < 64 ? rows : 64);
    const int G = norm_lanes(D);
    const long per = G > kNormBwdThreads ? 1 : kNormBwdThreads / G, need = ceil_div_l(rows, per), most = 256;
    return (int)(need < most ? need : most);
}

#define ADDER_NORM_LANES(G, CALL)            \
    switch (G) {                             \
        case 8: CALL(8); break;              \
        case 16: CALL(16); break;            \
        case 32: CALL(32); break;            \
        case 64: CALL(64); break;            \
        case 128: CALL(128); break;          \
        case 256: CALL(256); break;          \
        case 512: CALL(512); break;          \
        default: CALL(1024); break;          \
    }

template <class T, class W>
int launch_layer_norm_fwd(const T *x, long x_stride, const W *w, const W *b, T *y, float *mean, float *rstd, float eps, long rows,
                          int D, hipStream_t s) {
    if (D > kNormRegisterWidth) {
        hipLaunchKernelGGL((layer_norm_wide_fwd_kernel<T, W>), dim3((unsigned)(rows < 4096 ? rows : 4096)), dim3(kNormWide), 0, s, x,
                           x_stride, w, b, y, mean, rstd, eps, rows, D);
        return check_launch();
    }
    const int G = norm_lanes(D);
#define ADDER_CALL(g)                                                                                                          \
    hipLaunchKernelGGL((layer_norm_fwd_kernel<T, W, g>), dim3(norm_fwd_blocks(rows, g)),                                       \
                       dim3(g > kNormFwdThreads ? g : kNormFwdThreads), 0, s, x, x_stride, w, b, y, mean, rstd, eps, rows, D)
    ADDER_NORM_LANES(G, ADDER_CALL)
#undef ADDER_CALL
    return check_launch();
}

template <class T, class W>
int launch_layer_norm_bwd(const T *dy, long dy_stride, const T *x, long x_stride, const W *w, const float *mean, const float *rstd,
                          T *gx, W *gw, W *gb, long rows, int D, float *part, hipStream_t s) {
    const int parts = layer_norm_bwd_parts(rows, D);
    float *sums = gw || gb ? part : nullptr;
    if (D > kNormRegisterWidth) {
        if (gx) {
            hipLaunchKernelGGL((layer_norm_wide_gx_kernel<T, W>), dim3((unsigned)(rows < 4096 ? rows : 4096)), dim3(kNormWide), 0, s,
                               dy, dy_stride, x, x_stride, w, mean, rstd, gx, rows, D);
            if (int rc = check_launch()) return rc;
        }
        if (sums) {
            hipLaunchKernelGGL((layer_norm_wide_columns_kernel<T>), dim3((unsigned)ceil_div(D, 256), parts), dim3(256), 0, s, dy,
                               dy_stride, x, x_stride, mean, rstd, sums, rows, D);
            if (int rc = check_launch()) return rc;
        }
    } else {
        const int G = norm_lanes(D);
#define ADDER_CALL(g)                                                                                                     \
    hipLaunchKernelGGL((layer_norm_bwd_kernel<T, W, g>), dim3(parts), dim3(g > kNormBwdThreads ? g : kNormBwdThreads), 0, \
                       s, dy, dy_stride, x, x_stride, w, mean, rstd, gx, sums, rows, D)
        ADDER_NORM_LANES(G, ADDER_CALL)
#undef ADDER_CALL
        if (int rc = check_launch()) return rc;
    }
    if (!sums) return ADDER_OK;
    return launch_fold_columns<W>(sums, parts, 2, D, FoldOut{{gw, gb}}, s);
}

#define ADDER_NORM_INSTANCE(T, W)                                                                                                 \
    template int launch_layer_norm_fwd<T, W>(const T *, long, const W *, const W *, T *, float *, float *, float, long, int,       \
                                             hipStream_t);                                                                        \
    template int launch_layer_norm_bwd<T, W>(const T *, long, const T *, long, const W *, const float *, const float *, T *, W *, \
                                             W *, long, int, float *, hipStream_t);
ADDER_NORM_INSTANCE(float, float)
ADDER_NORM_INSTANCE(bf16_t, bf16_t)
ADDER_NORM_INSTANCE(bf16_t, float)

}  // namespace adder
