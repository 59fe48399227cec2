// Linear layers: y = act(x w' + b) + r and its gradients,
//     z = x w' + b,   dz = dy * act'(z),   gx = dz w,   gw = dz' x,   gb = sum over rows of dz.
// All three products are out[m, n] = sum_k A(m, k) B(n, k) with k along or across the rows of either operand.  Here: which kernel a
// product takes, the join of sums that were split over k, and the pass over dy.
#include "product.hpp"

namespace adder {

// The shares of the sums added up in their order, and the epilogue: four results a thread.  Memory decides, or the launch: two shares of
// 4096 x 1024 12 us (42 MB), four of 128 x 512 3 us.
template <class T, bool GATED>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs p) {
    const long columns = GATED ? p.half : p.N, groups = (columns + 3) / 4, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.M * groups) return;
    const long m = i / groups, n = i % groups * 4;
    const int cnt = columns - n < 4 ? (int)(columns - n) : 4;
    const long share = p.M * p.N;
    const auto sum = [&](long column, float (&v)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = 0.f;
        const float *q = p.part + m * p.N + column;
        int s = 0;
        if (GATED || cnt == 4) {   // (gated: whole groups of sixteen)
            for (; s + 4 <= p.splits; s += 4) {   // (four loads under way)
                float t[4][4];
#pragma unroll
                for (int u = 0; u < 4; ++u) ld_strip<4>(q + (s + u) * share, t[u]);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += t[u][e];
            }
        }
        for (; s < p.splits; ++s) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += e < cnt ? q[s * share + e] : 0.f;
        }
    };
    float v[4];
    if constexpr (GATED) {
        float u[4];
        const long column = (n >> 4) * 32 + (n & 15);
        sum(column, v);
        sum(column + 16, u);
        finish_gated<T>(p, m, n, cnt, v, u);
    } else {
        sum(n, v);
        finish<T>(p, m, n, cnt, v);
    }
}

template <class T>
int launch_product_join(const ProductArgs &p, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div_l(p.M * (((p.half ? p.half : p.N) + 3) / 4), 256));
    if (p.half) hipLaunchKernelGGL((product_join_kernel<T, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((product_join_kernel<T, false>), grid, dim3(256), 0, s, p);
    return check_launch();
}

// ---- which kernel ---------------------------------------------------------------------------------------------------
// (the estimate: product.hpp)
//                                       8192^3, TFLOP/s
static constexpr Shape kStreamShapes[] = {
    {256, 256, 1, 1.55f, 1.55f, 10.f},   // 1305
    {128, 256, 1, 0.9f, 0.9f, 4.f},      // 1146 (taken for shares of long sums: 616 x 28360 -> 16568 in 821 us, 1028 without it)
    {128, 128, 2, 0.87f, 0.65f, 3.5f},   // 1177
    {64, 64, 2, 0.38f, 0.2f, 1.5f},      //  719
};
// Gated layers, whose results are half as many columns (8192 x 1024 -> 4096 with what the backward needs: 151, 182, 174, 287 us)
static constexpr Shape kGatedShapes[] = {
    {256, 256, 1, 1.55f, 1.55f, 6.1f},
    {128, 256, 1, 0.9f, 0.9f, 3.f},
    {128, 128, 2, 0.87f, 0.65f, 3.75f},
    {64, 64, 2, 0.38f, 0.2f, 1.5f},
};
template <class T>
static constexpr Shape kStagedShapes[] = {
    {128, 128, 2, 1.f, 0.6f, 3.5f},      // 1033
    {64, 64, 4, 0.78f, 0.25f, 1.5f},     //  701
};
template <>
constexpr Shape kStagedShapes<float>[] = {
    {128, 128, 2, 2.3f, 1.9f, 3.5f},     //  220
    {64, 64, 3, 1.25f, 0.65f, 1.5f},     //  161
    {128, 128, 1, 1.15f, 1.15f, 3.5f},   //  204 (step: that of one or two rounds, 2048^3)
    {64, 64, 1, 0.53f, 0.53f, 2.5f},     //  147
};
// The kernel for few rows likewise: workgroups of 16 columns and 16, 32 or 64 rows, whose waves take turns along k, 128 bytes of every
// row at a time (us each, with the rows' share of the second-level caches: 4096 x 4096, full workgroups)
static constexpr long kRowsMost = 1024, kRowsColumns = 1L << 25;   // within which the estimate finds it the fastest, and its launch has few enough threads
template <class T>
static float rows_us(long M, long N, long K) {
    static constexpr float kTurn[2][3] = {{1.2f, 2.1f, 1.95f}, {1.75f, 2.5f, 2.2f}};
    const int mt = M <= 16 ? 0 : M <= 32 ? 1 : 2;
    const float groups = (float)ceil_div_l(N, 16) * (float)ceil_div_l(M, 16 << mt);
    const long turns = ceil_div_l(ceil_div_l(K, 8 * Chunk<T>::n), mt == 2 ? 8 : 16);
    return 3.f + ceilf(groups / kCUs) * (1.3f + turns * kTurn[sizeof(T) == 4][mt]);
}

template <class T>
static ProductPlan plan_staged(long M, long N, long K, int outputs) { return plan_product(kStagedShapes<T>, sizeof(T) == 4 ? 32 : 64, M, N, K, outputs); }
static ProductPlan plan_stream(long M, long N, long K, int outputs, bool gated) { return plan_product(gated ? kGatedShapes : kStreamShapes, 64, M, N, K, outputs); }

// Loads of 16 aligned bytes fit a bfloat16 operand: base and rows begin at multiples of them, and what a tile's last load brings
// beside the operand it can be told from by k alone (k along: rows of whole loads) or is never stored (k across).  A tile's rows
// lie within 2^32 bytes of each other.
static bool aligned16(const void *p, long ld) { return !(reinterpret_cast<uintptr_t>(p) & 15) && !(ld & 7) && ld < (1L << 22); }
static bool fits_stream(bool across, long K) { return across || !(K & 7); }

static size_t split_bytes(const ProductPlan &p, long M, long N) { return p.splits > 1 ? sizeof(float) * (size_t)p.splits * M * N : 0; }

template <class T>
size_t product_workspace_bytes(long M, long N, long K, bool gated) {
    size_t most = 0;   // whichever kernel strides and alignments leave, with and without a second output
    for (int outputs = 1; outputs <= 2; ++outputs) {
        const size_t staged = split_bytes(plan_staged<T>(M, N, K, outputs), M, N), stream = sizeof(T) == 2 ? split_bytes(plan_stream(M, N, K, outputs, gated), M, N) : 0;
        if (staged > most) most = staged;
        if (stream > most) most = stream;
    }
    return most;
}

// The one choice that a launch and adder_linear_kernel make
enum class Family { rows = 1, stream, staged };
struct Choice { Family family; ProductPlan plan; };
template <class T>
static Choice choose_product(long M, long N, long K, bool a_across, bool b_across, bool aligned, int outputs, bool gated) {
    const bool stream = sizeof(T) == 2 && aligned && fits_stream(a_across, K) && fits_stream(b_across, K);
    const ProductPlan plan = stream ? plan_stream(M, N, K, outputs, gated) : plan_staged<T>(M, N, K, outputs);
    if (!a_across && !b_across && M <= kRowsMost && N <= kRowsColumns && rows_us<T>(M, N, K) < plan.us) return {Family::rows, ProductPlan{0, 1, K, 0.f}};
    return {stream ? Family::stream : Family::staged, plan};
}
template <class T>
int product_kernel(long M, long N, long K, bool a_across, bool b_across, bool aligned, int outputs, bool gated) {
    const Choice c = choose_product<T>(M, N, K, a_across, b_across, aligned, outputs, gated);
    return static_cast<int>(c.family) * 10000 + (c.family == Family::rows ? product_rows_tiles(M) : c.plan.shape) * 100 + c.plan.splits;
}

template <class T>
int launch_product(const Product &q, void *ws, hipStream_t s) {
    const bool aligned = aligned16(q.a, q.lda) && aligned16(q.b, q.ldb) && (!q.half || (q.half + 256) * q.ldb < (1L << 31));   // (gated: a tile's rows are half the weight apart)
    const Choice c = choose_product<T>(q.M, q.N, q.K, q.a_across, q.b_across, aligned, q.pre ? 2 : 1, q.half != 0);
    const ProductPlan &plan = c.plan;
    const ProductArgs p{q.a, q.b, q.bias, q.res, q.out, q.pre, static_cast<float *>(ws), q.lda, q.ldb, q.ldr, q.M, q.N, q.K, plan.k_share, 0, 0,
                        plan.splits, q.act, q.half};
    const int rc = c.family == Family::rows ? launch_product_rows<T>(p, s)
                 : c.family == Family::stream ? launch_product_stream(p, q.a_across, q.b_across, static_cast<StreamShape>(plan.shape), s)
                 : launch_product_staged<T>(p, q.a_across, q.b_across, static_cast<StagedShape>(plan.shape), s);
    if (rc || plan.splits == 1) return rc;
    return launch_product_join<T>(p, s);
}

// ---- the activation's derivative and the bias's gradient ---------------------------------------------------------------
// Memory decides: dy and z are read and dz is written, 41 us for 8192 x 4096 in bfloat16 with a GELU (4.9 TB/s).  A workgroup takes 64 lanes'
// chunks of columns and a share of the rows; its four waves walk over the rows, and their column sums are added through LDS into
// one slab a share.  bfloat16: dz is rounded to the type of the products' operands, and the bias's sums are not; gradients are then 0.0023 from float64
// where a float32 dz, as two bfloat16 parts, would give 0.0017 for twice the products' work.  A row at a time and up to four workgroups a compute unit: two or four rows under way in a wave are no faster where there
// are many (53 us with what follows, all three) and leave waves out where there are few (128 x 512: 9.9 and 10.8 us instead of 9.5);
// 2048 workgroups leave more slabs to fold (16384 x 512: 23.4 us instead of 21.1).
template <class T, Act ACT>
__global__ __launch_bounds__(256) void act_bwd_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ z,
                                                      T *__restrict__ dz, float *__restrict__ part, long rows, long N) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = ((long)blockIdx.x * 64 + lane) * V;
    const int left = N - n < V ? (int)(N - n < 0 ? 0 : N - n) : V;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    for (long m = (long)blockIdx.y * 4 + wave; m < rows; m += (long)gridDim.y * 4) {
        float d[V];
        load_part(dy + m * dy_stride + n, left, d);
        if constexpr (ACT != Act::none) {
            float w[V];
            const uint4 u = load_raw_part(z + m * N + n, left);
            if constexpr (keeps_half(sizeof(T), ACT)) unpack_half(u, w);
            else unpack(u, w);
#pragma unroll
            for (int e = 0; e < V; ++e)   // (a ReLU selects: where it is off, an infinite dy or one that is no number goes no further)
                d[e] = ACT != Act::relu ? d[e] * slope<kExactAct<T>>(w[e], ACT) : w[e] <= 0.f ? 0.f : d[e];
            if (dz) store_part(dz + m * N + n, left, d);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += d[e];   // (columns that do not exist: dy of zero times the slope at zero)
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

// Shares of the rows: a row a wave, as long as there are no more workgroups than four a compute unit
int act_bwd_parts(long rows, long N) {
    const long columns = ceil_div_l(N, 512), need = ceil_div_l(rows, 4), most = ceil_div_l(4 * kCUs, columns);
    return (int)(need < most ? need : most);
}

template <class T>
int launch_act_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div_l(N, 64 * Chunk<T>::n), act_bwd_parts(rows, N)), threads(256);
    switch (act) {
        case Act::relu: hipLaunchKernelGGL((act_bwd_kernel<T, Act::relu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        case Act::gelu: hipLaunchKernelGGL((act_bwd_kernel<T, Act::gelu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        case Act::silu: hipLaunchKernelGGL((act_bwd_kernel<T, Act::silu>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N); break;
        default: hipLaunchKernelGGL((act_bwd_kernel<T, Act::none>), grid, threads, 0, s, dy, dy_stride, z, dz, part, rows, N);
    }
    return check_launch();
}

#define ADDER_LINEAR_INSTANCE(T)                                                                                      \
    template size_t product_workspace_bytes<T>(long, long, long, bool);                                                \
    template int launch_product<T>(const Product &, void *, hipStream_t);                                            \
    template int launch_product_join<T>(const ProductArgs &, hipStream_t);                                            \
    template int product_kernel<T>(long, long, long, bool, bool, bool, int, bool);                                   \
    template int launch_act_bwd<T>(const T *, long, const T *, T *, float *, Act, long, long, hipStream_t);
ADDER_LINEAR_INSTANCE(float)
ADDER_LINEAR_INSTANCE(bf16_t)

}  // namespace adder
