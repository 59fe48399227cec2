// Root-mean-square normalisation over the last dimension, with the addition in front of it:
//     s = x + r,   rstd = 1 / sqrt(mean(s^2) + eps),   h = s rstd,   y = h w
//     gs = ds + rstd (g - h mean(g h)) with g = dy w,   gx = gr = gs,   gw = sum over rows of dy h
// ds is the gradient of s where that goes on as the shortcut.  y comes as values, or as e4m3 codes with a scale for each 128 of them.
// Memory decides: the forward reads x and r and writes s and y, the backward reads dy, ds and s and writes gs.  A row stays in
// registers from its one load on (G lanes with 16 values each); sums are 32 bits, and y is taken from s before that is rounded.  The backward reads s
// as it was rounded, as a norm behind an addition of its own would: with bfloat16 rows the weight's gradient is 0.0024 from float64 then, 0.0016 from
// x and r, which would be a fifth row to read beside dy, ds, s and gs, a quarter more time.
// 16384 x 2048 in bfloat16 with a shortcut: forward 42 us (6.4 TB/s), backward 48 (5.6 TB/s) and 4 for the fold of the columns; 8192 x 4096 to codes 38 us
// (6.2 TB/s); 3001 x 777 in float32 7, 9 and 3 us; one row of 4096 2.6 us, a launch.
#include "blocks.hpp"

namespace adder {

template <class T>
static constexpr int kRmsChunks = kNormValues / Chunk<T>::n;
static constexpr int kRmsFwdThreads = 256, kRmsBwdThreads = 512, kRmsWide = 1024;

// Codes and scales of a row whose lane holds v[c] at (lane + c G) V: 128 / V neighbouring lanes have a block.
template <int V, int C, int G>
__device__ __forceinline__ void put_codes(const float (&v)[C][V], uint8_t *q, float *scale, int lane, int width) {
    constexpr int L = kCodeBlock / V;
    static_assert(G >= L, "a block lies in one step's lanes");
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (lane + c * G) * V;
        float top = kCodeLeast;
#pragma unroll
        for (int e = 0; e < V; ++e) top = fmaxf(top, at + e < width ? fabsf(v[c][e]) : 0.f);
        top = lanes_max<L>(top);
        const float by = kCodeTop / top;
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = v[c][e] * by;
        store_codes(q + at, width - at, o);
        if (lane % L == 0 && at < width) scale[at / kCodeBlock] = top / kCodeTop;
    }
}

template <class T, class W, int G, bool CODES>
__global__ __launch_bounds__(G > kRmsFwdThreads ? G : kRmsFwdThreads) void rms_norm_fwd_kernel(const RmsRows p) {
    constexpr int V = Chunk<T>::n, C = kRmsChunks<T>, THREADS = G > kRmsFwdThreads ? G : kRmsFwdThreads, PER = THREADS / G;
    __shared__ float lds[16];
    const int lane = threadIdx.x % G, D = p.D;
    const T *x = static_cast<const T *>(p.x), *r = static_cast<const T *>(p.r);
    const W *w = static_cast<const W *>(p.w);
    T *sum = static_cast<T *>(p.sum);
    const float inv = 1.f / (float)D;
    float wv[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (lane + c * G) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) wv[c][e] = 1.f;
        if (w) load_values<V>(w + at, D - at, wv[c]);
    }
    for (long base = (long)blockIdx.x * PER; base < p.rows; base += (long)gridDim.x * PER) {   // (all waves together)
        const long row = base + threadIdx.x / G;
        const int width = row < p.rows ? D : 0;
        float v[C][V], q = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) load_part(x + row * p.x_stride + (lane + c * G) * V, width - (lane + c * G) * V, v[c]);
        if (r) {
            float u[C][V];
#pragma unroll
            for (int c = 0; c < C; ++c) load_part(r + row * p.r_stride + (lane + c * G) * V, width - (lane + c * G) * V, u[c]);
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) v[c][e] += u[c][e];
        }
        if (sum) {
#pragma unroll
            for (int c = 0; c < C; ++c) store_part(sum + row * D + (lane + c * G) * V, width - (lane + c * G) * V, v[c]);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) q = fmaf(v[c][e], v[c][e], q);
        const float rs = 1.f / sqrtf(fmaf(row_sum<G>(q, lds), inv, p.eps));
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) v[c][e] = v[c][e] * rs * wv[c][e];
        if constexpr (CODES) {
            put_codes<V, C, G>(v, static_cast<uint8_t *>(p.y) + row * D, p.scale + row * ((D + kCodeBlock - 1) / kCodeBlock), lane, width);
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c)
                store_part(static_cast<T *>(p.y) + row * D + (lane + c * G) * V, width - (lane + c * G) * V, v[c]);
        }
        if (p.rstd && lane == 0 && width) p.rstd[row] = rs;
    }
}

// The workgroups walk over the rows and keep the columns' sums of dy h of their rows in registers; at the end the lanes of a wave that
// hold the same columns add theirs, then the waves through LDS, and the workgroup writes one slab of D floats, which
// launch_fold_columns adds up: no atomics, the same bits every run.
template <class T, class W, int G>
__global__ __launch_bounds__(G > kRmsBwdThreads ? G : kRmsBwdThreads) void rms_norm_bwd_kernel(
    const T *__restrict__ dy, long dy_stride, const T *__restrict__ ds, long ds_stride, const T *__restrict__ x, long x_stride,
    const W *__restrict__ w, const float *__restrict__ rstd, T *__restrict__ gx, float *__restrict__ part, long rows, int D) {
    constexpr int V = Chunk<T>::n, C = kRmsChunks<T>, THREADS = G > kRmsBwdThreads ? G : kRmsBwdThreads, PER = THREADS / G;
    constexpr int LANES = G < 64 ? G : 64, SHARE = G < 64 ? THREADS / 64 : PER;   // lanes of a wave with columns of their own; LDS copies of the columns
    __shared__ float lds[16];
    __shared__ __align__(16) float fold[SHARE > 1 ? SHARE * G * kNormValues : 4];
    const int lane = threadIdx.x % G;
    const float inv = 1.f / (float)D;
    float wv[C][V], sw[C][V];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = (lane + c * G) * V;
#pragma unroll
        for (int e = 0; e < V; ++e) { wv[c][e] = 1.f; sw[c][e] = 0.f; }
        if (w) load_values<V>(w + at, D - at, wv[c]);
    }
    for (long base = (long)blockIdx.x * PER; base < rows; base += (long)gridDim.x * PER) {   // (all waves together)
        const long row = base + threadIdx.x / G;
        const int width = row < rows ? D : 0;
        const float rs = width ? rstd[row] : 0.f;
        float h[C][V], g[C][V], s = 0.f;
        uint4 d[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = (lane + c * G) * V;
            load_part(x + row * x_stride + at, width - at, h[c]);
            load_part(dy + row * dy_stride + at, width - at, g[c]);
            d[c] = ds ? load_raw_part(ds + row * ds_stride + at, width - at) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[c][e] *= rs;
                sw[c][e] = fmaf(g[c][e], h[c][e], sw[c][e]);
                g[c][e] *= wv[c][e];
                s = fmaf(g[c][e], h[c][e], s);
            }
        s = row_sum<G>(s, lds) * inv;
        if (gx) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float o[V];
                unpack(d[c], o);
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = fmaf(rs, g[c][e] - h[c][e] * s, o[e]);
                store_part(gx + row * D + (lane + c * G) * V, width - (lane + c * G) * V, o);
            }
        }
    }
    if (!part) return;
    float *slab = part + (size_t)blockIdx.x * D;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
            for (int off = LANES; off < 64; off *= 2) sw[c][e] += __shfl_xor(sw[c][e], off, 64);
    if constexpr (SHARE == 1) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int q = 0; q < V; q += 4) {
                const float u[4] = {sw[c][q], sw[c][q + 1], sw[c][q + 2], sw[c][q + 3]};
                const int at = (lane + c * G) * V + q;
                store_part(slab + at, D - at, u);
            }
    } else {
        const int copy = threadIdx.x / (G < 64 ? 64 : G);
        if ((threadIdx.x & 63) < LANES)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int q = 0; q < V; q += 4)
                    *reinterpret_cast<float4 *>(fold + copy * (G * kNormValues) + (lane + c * G) * V + q) =
                        make_float4(sw[c][q], sw[c][q + 1], sw[c][q + 2], sw[c][q + 3]);
        __syncthreads();
        for (int i = threadIdx.x; i < D; i += THREADS) {
            float u = fold[i];
#pragma unroll
            for (int r = 1; r < SHARE; ++r) u += fold[r * (G * kNormValues) + i];
            slab[i] = u;
        }
    }
}

// Rows longer than kNormRegisterWidth: one workgroup a row, which reads it again (from its L2, as long as that holds it).
template <class T, class W>
__global__ __launch_bounds__(kRmsWide) void rms_norm_wide_fwd_kernel(const RmsRows p) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[16];
    const int D = p.D;
    const T *x = static_cast<const T *>(p.x), *r = static_cast<const T *>(p.r);
    const W *w = static_cast<const W *>(p.w);
    T *sum = static_cast<T *>(p.sum);
    const float inv = 1.f / (float)D;
    for (long row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T *px = x + row * p.x_stride, *pr = r ? r + row * p.r_stride : nullptr;
        auto at = [&](int i) { return ldf(px + i) + (pr ? ldf(pr + i) : 0.f); };
        auto chunk = [&](int i, float (&v)[V]) {
            load_part(px + i, D - i, v);
            if (pr) {
                float u[V];
                load_part(pr + i, D - i, u);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] += u[e];
            }
        };
        float q = 0.f;
#pragma unroll 2
        for (int i = threadIdx.x * V; i < D; i += kRmsWide * V) {
            float v[V];
            chunk(i, v);
            if (sum) store_part(sum + row * D + i, D - i, v);
#pragma unroll
            for (int e = 0; e < V; ++e) q = fmaf(v[e], v[e], q);
        }
        const float rs = 1.f / sqrtf(fmaf(row_sum<kRmsWide>(q, lds), inv, p.eps));
        if (p.scale) {   // a wave a block of codes, two values a lane
            const int blocks = (D + kCodeBlock - 1) / kCodeBlock;
            for (int b = threadIdx.x >> 6; b < blocks; b += kRmsWide / 64) {
                const int i = b * kCodeBlock + (threadIdx.x & 63) * 2;
                float v[2], top = kCodeLeast;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    v[e] = i + e < D ? at(i + e) * rs * (w ? ldf(w + i + e) : 1.f) : 0.f;
                    top = fmaxf(top, fabsf(v[e]));
                }
                top = lanes_max<64>(top);
                const float by = kCodeTop / top;
                const uint32_t u = pack_codes(v[0] * by, v[1] * by, 0.f, 0.f);
                uint8_t *o = static_cast<uint8_t *>(p.y) + row * D + i;
                if (i < D) o[0] = (uint8_t)u;
                if (i + 1 < D) o[1] = (uint8_t)(u >> 8);
                if ((threadIdx.x & 63) == 0) p.scale[row * blocks + b] = top / kCodeTop;
            }
        } else {
#pragma unroll 2
            for (int i = threadIdx.x * V; i < D; i += kRmsWide * V) {
                float v[V], wv[V];
                chunk(i, v);
                if (w) load_values<V>(w + i, D - i, wv);
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = w ? v[e] * rs * wv[e] : v[e] * rs;
                store_part(static_cast<T *>(p.y) + row * D + i, D - i, v);
            }
        }
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rs;
    }
}

template <class T, class W>
__global__ __launch_bounds__(kRmsWide) void rms_norm_wide_gx_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ ds,
                                                                    long ds_stride, const T *__restrict__ x, long x_stride,
                                                                    const W *__restrict__ w, const float *__restrict__ rstd,
                                                                    T *__restrict__ gx, long rows, int D) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[16];
    const float inv = 1.f / (float)D;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *px = x + row * x_stride, *pg = dy + row * dy_stride, *pd = ds ? ds + row * ds_stride : nullptr;
        const float rs = rstd[row];
        auto chunk = [&](int i, float (&g)[V], float (&h)[V]) {   // dy w and s rstd
            load_part(pg + i, D - i, g);
            load_part(px + i, D - i, h);
            float wv[V];
            if (w) load_values<V>(w + i, D - i, wv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                g[e] = w ? g[e] * wv[e] : g[e];
                h[e] *= rs;
            }
        };
        float s = 0.f;
#pragma unroll 2
        for (int i = threadIdx.x * V; i < D; i += kRmsWide * V) {
            float g[V], h[V];
            chunk(i, g, h);
#pragma unroll
            for (int e = 0; e < V; ++e) s = fmaf(g[e], h[e], s);
        }
        s = row_sum<kRmsWide>(s, lds) * inv;
        for (int i = threadIdx.x * V; i < D; i += kRmsWide * V) {
            float g[V], h[V], o[V];
            chunk(i, g, h);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = 0.f;
            if (pd) load_part(pd + i, D - i, o);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(rs, g[e] - h[e] * s, o[e]);
            store_part(gx + row * D + i, D - i, o);
        }
    }
}

// ... and their columns' sums: a thread a column, gridDim.y shares of the rows, a slab each
template <class T>
__global__ __launch_bounds__(256) void rms_norm_wide_columns_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ x,
                                                                    long x_stride, const float *__restrict__ rstd,
                                                                    float *__restrict__ part, long rows, int D) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= D) return;
    float s = 0.f;
    for (long row = blockIdx.y; row < rows; row += gridDim.y) s = fmaf(ldf(dy + row * dy_stride + i), ldf(x + row * x_stride + i) * rstd[row], s);
    part[(size_t)blockIdx.y * D + i] = s;
}

// At most three workgroups a compute unit, which walk over the rows with the weight in registers
static int rms_fwd_blocks(long rows, int G) {
    const long per = G > kRmsFwdThreads ? 1 : kRmsFwdThreads / G, need = ceil_div_l(rows, per), most = 768;
    return (int)(need < most ? need : most);
}

// One workgroup a compute unit, each with a slab
int rms_norm_bwd_parts(long rows, int D) {
    if (D > kNormRegisterWidth) return (int)(rows < 64 ? rows : 64);
    const int G = norm_lanes(D);
    const long per = G > kRmsBwdThreads ? 1 : kRmsBwdThreads / G, need = ceil_div_l(rows, per), most = 256;
    return (int)(need < most ? need : most);
}

template <class T, class W>
int launch_rms_norm_fwd(const RmsRows &p, hipStream_t s) {
    if (p.D > kNormRegisterWidth) {
        hipLaunchKernelGGL((rms_norm_wide_fwd_kernel<T, W>), dim3((unsigned)(p.rows < 4096 ? p.rows : 4096)), dim3(kRmsWide), 0, s, p);
        return check_launch();
    }
    constexpr int L = kCodeBlock / Chunk<T>::n;   // lanes that a block of codes needs
    int G = norm_lanes(p.D);
    if (p.scale && G < L) G = L;
#define ADDER_RMS_FWD(g, codes) \
    hipLaunchKernelGGL((rms_norm_fwd_kernel<T, W, g, codes>), dim3(rms_fwd_blocks(p.rows, g)), dim3(g > kRmsFwdThreads ? g : kRmsFwdThreads), 0, s, p)
#define ADDER_CALL(g)                                                                              \
    if (!p.scale) ADDER_RMS_FWD(g, false);                                                         \
    else if constexpr (g >= L) ADDER_RMS_FWD(g, true)
    ADDER_NORM_LANES(G, ADDER_CALL)
#undef ADDER_CALL
#undef ADDER_RMS_FWD
    return check_launch();
}

template <class T, class W>
int launch_rms_norm_bwd(const T *dy, long dy_stride, const T *ds, long ds_stride, const T *x, long x_stride, const W *w, const float *rstd, T *gx,
                        W *gw, long rows, int D, float *part, hipStream_t s) {
    const int parts = rms_norm_bwd_parts(rows, D);
    float *sums = gw ? part : nullptr;
    if (D > kNormRegisterWidth) {
        if (gx) {
            hipLaunchKernelGGL((rms_norm_wide_gx_kernel<T, W>), dim3((unsigned)(rows < 4096 ? rows : 4096)), dim3(kRmsWide), 0, s, dy, dy_stride, ds,
                               ds_stride, x, x_stride, w, rstd, gx, rows, D);
            if (int rc = check_launch()) return rc;
        }
        if (sums) {
            hipLaunchKernelGGL((rms_norm_wide_columns_kernel<T>), dim3((unsigned)ceil_div(D, 256), parts), dim3(256), 0, s, dy, dy_stride, x, x_stride,
                               rstd, sums, rows, D);
            if (int rc = check_launch()) return rc;
        }
    } else {
        const int G = norm_lanes(D);
#define ADDER_CALL(g)                                                                                                                    \
    hipLaunchKernelGGL((rms_norm_bwd_kernel<T, W, g>), dim3(parts), dim3(g > kRmsBwdThreads ? g : kRmsBwdThreads), 0, s, dy, dy_stride, \
                       ds, ds_stride, x, x_stride, w, rstd, gx, sums, rows, D)
        ADDER_NORM_LANES(G, ADDER_CALL)
#undef ADDER_CALL
        if (int rc = check_launch()) return rc;
    }
    if (!sums) return ADDER_OK;
    return launch_fold_columns<W>(sums, parts, 1, D, FoldOut{{gw, nullptr}}, s);
}

#define ADDER_RMS_INSTANCE(T, W)                                                                                                          \
    template int launch_rms_norm_fwd<T, W>(const RmsRows &, hipStream_t);                                                                 \
    template int launch_rms_norm_bwd<T, W>(const T *, long, const T *, long, const T *, long, const W *, const float *, T *, W *, long,   \
                                           int, float *, hipStream_t);
ADDER_RMS_INSTANCE(float, float)
ADDER_RMS_INSTANCE(bf16_t, bf16_t)
ADDER_RMS_INSTANCE(bf16_t, float)

}  // namespace adder
