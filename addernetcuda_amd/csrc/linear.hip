// Linear layers: y = act(x w' + b) + r and its gradients,
//     z = x w' + b,   dz = dy * act'(z),   gx = dz w,   gw = dz' x,   gb = sum over rows of dz.
// All three products are out[m, n] = sum_k A(m, k) B(n, k) with k along or across the rows of either operand.  Here: which kernel a
// product takes, the join of sums that were split over k, and the pass over dy.
#include "product.hpp"

namespace adder {

// The shares of the sums added up in their order, and the epilogue: four results a thread
template <class T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs p) {
    const long groups = (p.N + 3) / 4, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.M * groups) return;
    const long m = i / groups, n = i % groups * 4;
    const int cnt = p.N - n < 4 ? (int)(p.N - n) : 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const float *q = p.part + ((long)s * p.M + m) * p.N + n;
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        if (cnt == 4) {
            ld_strip<4>(q, t);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < cnt) t[e] = q[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
    }
    finish<T>(p, m, n, cnt, v);
}

// ---- which kernel ---------------------------------------------------------------------------------------------------
// A launch's time is estimated as rounds * (steps * step + tile) us for every shape and number of shares of k, and the least is
// taken: rounds of as many workgroups as the card holds, steps of 64 (float32: 32) values of k a workgroup, `step` measured on a full
// card (8192^3), `alone` where a compute unit has one workgroup only, `tile` the epilogue, the first loads and the start.  Shares of k
// pay for their sums' way through memory (5 TB/s both ways) and the join's launch.
struct Shape { int bm, bn, per_cu; float step, alone, tile; };
//                                     8192^3 in bfloat16 (float32), TFLOP/s
static constexpr Shape kStreamShapes[] = {
    {256, 256, 1, 1.6f, 1.6f, 8.f},    // 1320
    {128, 256, 1, 0.93f, 0.93f, 4.5f}, // 1155
    {128, 128, 2, 0.92f, 0.65f, 4.5f}, // 1155
};
template <class T>
static constexpr Shape kStagedShapes[] = {
    {128, 128, 2, 1.1f, 0.9f, 5.f},    // 960
    {64, 64, 4, 0.84f, 0.5f, 4.f},     // 636
};
template <>
constexpr Shape kStagedShapes<float>[] = {
    {128, 128, 2, 2.8f, 2.0f, 6.f},    // (190)
    {64, 64, 4, 1.75f, 0.8f, 5.f},     // (153)
};
static constexpr int kCUs = 256, kSplitMax = 16;

struct ProductPlan { int shape, splits; long k_share; };

template <int N>
static ProductPlan plan_product(const Shape (&shapes)[N], int bk, long M, long N_, long K) {
    static constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, kSplitMax};
    ProductPlan best{0, 1, K};
    float least = 0.f;
    const long steps = ceil_div_l(K, bk);
    for (int i = 0; i < N; ++i) {
        const Shape &h = shapes[i];
        const float tiles = (float)ceil_div_l(M, h.bm) * (float)ceil_div_l(N_, h.bn);
        for (int splits : kSplits) {
            if (splits > steps || (splits > 1 && tiles * splits > 4.f * kCUs)) break;
            const long share = ceil_div_l(steps, splits);
            const float groups = tiles * splits;
            const float rounds = ceilf(groups / (kCUs * h.per_cu));
            float us = rounds * (share * (groups <= kCUs ? h.alone : h.step) + h.tile);
            if (splits > 1) us += 4.f + (float)M * (float)N_ * splits * 8.f / 5e6f;
            if (least == 0.f || us < least) {
                least = us;
                const int used = (int)ceil_div_l(steps, share);
                best = ProductPlan{i, used, used > 1 ? share * bk : K};
            }
        }
    }
    return best;
}
template <class T>
static ProductPlan plan_staged(long M, long N, long K) { return plan_product(kStagedShapes<T>, sizeof(T) == 4 ? 32 : 64, M, N, K); }
static ProductPlan plan_stream(long M, long N, long K) { return plan_product(kStreamShapes, 64, M, N, K); }

// Loads of 16 aligned bytes fit a bfloat16 operand: base and rows begin at multiples of them, and what a tile's last load brings
// beside the operand it can be told from by k alone (k along: rows of whole loads) or is never stored (k across).  A tile's rows
// lie within 2^32 bytes of each other.
static bool fits_stream(const void *p, long ld, bool across, long K) {
    return !(reinterpret_cast<uintptr_t>(p) & 15) && !(ld & 7) && (across || !(K & 7)) && ld < (1L << 22);
}

static size_t split_bytes(const ProductPlan &p, long M, long N) { return p.splits > 1 ? sizeof(float) * (size_t)p.splits * M * N : 0; }

template <class T>
size_t product_workspace_bytes(long M, long N, long K) {
    const size_t staged = split_bytes(plan_staged<T>(M, N, K), M, N);
    if (sizeof(T) == 4) return staged;
    const size_t stream = split_bytes(plan_stream(M, N, K), M, N);
    return stream > staged ? stream : staged;
}

template <class T>
int launch_product(const Product &q, void *ws, hipStream_t s) {
    const bool stream = sizeof(T) == 2 && fits_stream(q.a, q.lda, q.a_across, q.K) && fits_stream(q.b, q.ldb, q.b_across, q.K);
    const ProductPlan plan = stream ? plan_stream(q.M, q.N, q.K) : plan_staged<T>(q.M, q.N, q.K);
    const ProductArgs p{q.a, q.b, q.bias, q.res, q.out, q.pre, static_cast<float *>(ws), q.lda, q.ldb, q.ldr, q.M, q.N, q.K, plan.k_share, 0, 0,
                        plan.splits, q.act};
    const int rc = stream ? launch_product_stream(p, q.a_across, q.b_across, static_cast<StreamShape>(plan.shape), s)
                          : launch_product_staged<T>(p, q.a_across, q.b_across, plan.shape == 1, s);
    if (rc || plan.splits == 1) return rc;
    hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)ceil_div_l(q.M * ((q.N + 3) / 4), 256)), dim3(256), 0, s, p);
    return check_launch();
}

// ---- the activation's derivative and the bias's gradient ---------------------------------------------------------------
// A workgroup takes 64 lanes' chunks of columns and a share of the rows: its four waves walk over the rows, and their column
// sums are added through LDS into one slab per share.
template <class T>
__global__ __launch_bounds__(256) void act_bwd_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ z,
                                                      T *__restrict__ dz, float *__restrict__ part, Act act, long rows, long N) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = ((long)blockIdx.x * 64 + lane) * V;
    const int left = N - n < V ? (int)(N - n < 0 ? 0 : N - n) : V;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    for (long m = (long)blockIdx.y * 4 + wave; m < rows; m += (long)gridDim.y * 4) {
        float g[V], v[V];
        load_part(dy + m * dy_stride + n, left, g);
        if (act != Act::none) {
            load_part(z + m * N + n, left, v);
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] *= slope<kExactAct<T>>(v[e], act);
            if (dz) store_part(dz + m * N + n, left, g);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += g[e];
    }
    if (!part) return;
#pragma unroll
    for (int e = 0; e < V; ++e) lds[wave][e * 64 + lane] = sum[e];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
#pragma unroll
            for (int i = 1; i < 4; ++i) sum[e] += lds[i][e * 64 + lane];
            if (e < left) part[(long)blockIdx.y * N + n + e] = sum[e];
        }
    }
}

int act_bwd_parts(long rows, long N) {
    const long columns = ceil_div_l(N, 256), need = ceil_div_l(rows, 16), most = ceil_div_l(1024, columns);
    return (int)(need < most ? need : most);
}

template <class T>
int launch_act_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s) {
    hipLaunchKernelGGL(act_bwd_kernel<T>, dim3((unsigned)ceil_div_l(N, 64 * Chunk<T>::n), act_bwd_parts(rows, N)), dim3(256), 0, s, dy,
                       dy_stride, z, dz, part, act, rows, N);
    return check_launch();
}

#define ADDER_LINEAR_INSTANCE(T)                                                                                      \
    template size_t product_workspace_bytes<T>(long, long, long);                                                     \
    template int launch_product<T>(const Product &, void *, hipStream_t);                                            \
    template int launch_act_bwd<T>(const T *, long, const T *, T *, float *, Act, long, long, hipStream_t);
ADDER_LINEAR_INSTANCE(float)
ADDER_LINEAR_INSTANCE(bf16_t)

}  // namespace adder
