// The loss against a teacher's K largest logits t at the classes i, and the labels y, over all C classes of the logits l, and its gradient:
//     q = softmax(l / T),  o = softmax(l),  p = softmax(t / T) over the K
//     row = a T^2 sum_k p_k (log p_k - log q[i_k]) - (1 - a) log o[y],     loss = sum of the rows that count / their number
//     dl = 1 / number (a T (q - p at the classes i) + (1 - a) (o - 1 at y))
// Memory decides: l is read and dl written.  Where there are rows enough a workgroup keeps a row in registers: it reads it once, and
// writes the gradient for a loss whose own gradient is one on the way; the backward of any other computes it again.  Where rows are few
// and long several workgroups share one, and the gradient is the backward's.  All sums in a fixed order.
#include "blocks.hpp"

namespace adder {

static constexpr int kTeacherMost = ADDER_DISTILL_TOP_MAX;
static constexpr float kLog2e = 1.44269504f;
// What a row's loss and gradient are made of.  m, top: the largest logit, the teacher's; log_*: logarithms of the sums of exponentials
// behind them; by_*: factors of q and o in the gradient, zero where that part is not there (no teacher's logit above -infinity, a row that
// does not count), not a number where a class does not exist.  Behind the last row's: the rows that count, in m.
struct RowStats { float m, log_o, log_q, top, log_p, by_q, by_o, spare; };
static_assert(sizeof(RowStats) == kDistillStats * sizeof(float), "a row's statistics");

__device__ __forceinline__ float teacher_logit(const DistillArgs &a, long at) {
    return a.top_bf16 ? ldf(static_cast<const bf16_t *>(a.top) + at) : static_cast<const float *>(a.top)[at];
}
__device__ __forceinline__ bool exists(const DistillArgs &a, long long c) { return c >= 0 && c < a.classes; }
__device__ __forceinline__ bool counts(const DistillArgs &a, long row) { return !a.target || a.target[row] != a.ignore; }
__device__ __forceinline__ bool wants_q(const DistillArgs &a) { return !a.target || a.alpha != 0.f; }
__device__ __forceinline__ bool wants_o(const DistillArgs &a) { return a.target && a.alpha != 1.f; }

// chunk of a row of which `valid` values exist; -infinity in place of the others
template <class T>
__device__ __forceinline__ uint4 load_logits(const T *p, int valid) {
    constexpr int n = Chunk<T>::n;
    if (valid >= n) return load_raw(p);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = n == 4 ? 0xff800000u : 0xff80ff80u;
#pragma unroll
    for (int e = 0; e < n - 1; ++e)
        if (e < valid) {
            if constexpr (n == 4) w[e] = __float_as_uint(p[e]);
            else w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | (uint32_t)p[e] << 16 : (w[e / 2] & 0xffff0000u) | p[e];
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int WAVES>
__device__ __forceinline__ float group_max(float v, float *lds) {   // (beside a number, one that is none is left out: the sums find it)
    v = lanes_max<64>(v);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v = fmaxf(v, lds[i]);
    }
    return v;
}
template <int WAVES>
__device__ __forceinline__ float group_sum(float v, float *lds) {
    v = lanes_sum<64>(v);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int i = 1; i < WAVES; ++i) v += lds[i];
    }
    return v;
}

// A thread's logits in registers: their largest, and the sums of exponentials behind the row's (or the piece's) largest
template <class T, int C>
__device__ __forceinline__ float chunks_max(const uint4 (&u)[C]) {
    float m = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float v[Chunk<T>::n];
        unpack(u[c], v);
#pragma unroll
        for (int e = 0; e < Chunk<T>::n; ++e) m = fmaxf(m, v[e]);
    }
    return m;
}
template <class T, int C>
__device__ __forceinline__ void chunks_sums(const DistillArgs &a, const uint4 (&u)[C], float m, float &s_o, float &s_q) {
    const float k = kLog2e / a.temperature;
    const bool q = wants_q(a), o = wants_o(a), same = a.temperature == 1.f;
    const float one = q ? k : kLog2e;
    s_o = s_q = 0.f;
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float v[Chunk<T>::n];
        unpack(u[c], v);
        if (q && o && !same) {
#pragma unroll
            for (int e = 0; e < Chunk<T>::n; ++e) {
                s_q += __builtin_amdgcn_exp2f((v[e] - m) * k);
                s_o += __builtin_amdgcn_exp2f((v[e] - m) * kLog2e);
            }
        } else {
#pragma unroll
            for (int e = 0; e < Chunk<T>::n; ++e) s += __builtin_amdgcn_exp2f((v[e] - m) * one);
        }
    }
    if (!(q && o && !same)) s_o = s_q = s;
}

// One wave: the teacher's softmax and the factors of the gradient
__device__ __forceinline__ void teacher(const DistillArgs &a, long row, int lane, RowStats &r) {
    const float k = kLog2e / a.temperature, nan = __builtin_nanf("");
    const bool on = counts(a, row);
    r.top = r.log_p = r.by_q = 0.f;
    if (on && wants_q(a)) {
        float m = -__builtin_inff(), s = 0.f;
        bool bad = false;
        for (int j = lane; j < a.K; j += 64) {
            const float t = teacher_logit(a, row * a.K + j);
            m = fmaxf(m, t);
            bad = bad || !exists(a, a.idx[row * a.K + j]) || t != t;
        }
        m = lanes_max<64>(m);
        const bool taught = m > -__builtin_inff();
        for (int j = lane; j < a.K; j += 64) s += taught ? __builtin_amdgcn_exp2f((teacher_logit(a, row * a.K + j) - m) * k) : 0.f;
        s = lanes_sum<64>(s);
        r.top = taught ? m : 0.f;
        r.log_p = taught ? logf(s) : 0.f;
        r.by_q = __any(bad) ? nan : taught ? (a.target ? a.alpha : 1.f) * a.temperature : 0.f;
    }
    r.by_o = on && wants_o(a) ? exists(a, a.target[row]) ? 1.f - a.alpha : nan : 0.f;
}
// ... and the row's loss, once its own statistics are there
template <class T>
__device__ __forceinline__ float row_loss(const DistillArgs &a, long row, int lane, const RowStats &r) {
    const T *l = static_cast<const T *>(a.logits) + row * a.stride;
    const float inv = 1.f / a.temperature;
    float loss = 0.f;
    if (r.by_q != 0.f) {   // (also where it is no number)
        float kd = 0.f;
        for (int j = lane; j < a.K; j += 64) {
            const long long i = a.idx[row * a.K + j];
            const float log_p = (teacher_logit(a, row * a.K + j) - r.top) * inv - r.log_p, p = expf(log_p);
            const float log_q = exists(a, i) ? (ldf(l + i) - r.m) * inv - r.log_q : 0.f;
            kd += p == 0.f ? 0.f : p * (log_p - log_q);
        }
        loss = r.by_q * a.temperature * lanes_sum<64>(kd);
    }
    if (r.by_o != 0.f) {
        const long long y = a.target[row];
        loss -= r.by_o * (exists(a, y) ? ldf(l + y) - r.m - r.log_o : 0.f);
    }
    return loss;
}

// The classes at which something is taken off the gradient, in LDS: the teacher's, and the label behind them
struct Sparse { int idx[kTeacherMost + 1]; float off[kTeacherMost + 1]; };
__device__ __forceinline__ void fill_sparse(const DistillArgs &a, long row, const RowStats &r, float by_q, float by_o, Sparse &sp, int threads) {
    const float inv = 1.f / a.temperature;
    for (int j = threadIdx.x; j <= a.K; j += threads) {
        const bool label = j == a.K, there = label ? by_o != 0.f : by_q != 0.f;
        const long long i = !there ? -1 : label ? a.target[row] : a.idx[row * a.K + j];
        sp.idx[j] = exists(a, i) ? (int)i : -1;
        sp.off[j] = !there ? 0.f : label ? by_o : by_q * expf((teacher_logit(a, row * a.K + j) - r.top) * inv - r.log_p);
    }
}
// What the dense part of a row's gradient needs, for a loss whose gradient is `up`
struct Dense { float m, k, by_q, by_o, log_q, log_o; };
__device__ __forceinline__ Dense dense_of(const DistillArgs &a, const RowStats &r, float up) {
    return {r.m, kLog2e / a.temperature, r.by_q != 0.f ? r.by_q * up : 0.f, r.by_o != 0.f ? r.by_o * up : 0.f, r.log_q * kLog2e, r.log_o * kLog2e};
}
__device__ __forceinline__ float gradient(float l, const Dense &d) {
    const float x = l - d.m;
    float g = 0.f;
    if (d.by_q != 0.f) g = d.by_q * __builtin_amdgcn_exp2f(fmaf(x, d.k, -d.log_q));
    if (d.by_o != 0.f) g = fmaf(d.by_o, __builtin_amdgcn_exp2f(fmaf(x, kLog2e, -d.log_o)), g);
    return g;
}
// The gradient of `n` classes from `first` on, a thread's chunks at (thread + c THREADS): everywhere first, then again where something is taken
// off -- once a class, by the first of its entries.  (All threads together; behind it `sp` may be filled anew after a barrier.)
template <class T, int THREADS, int C>
__device__ __forceinline__ void put_gradient(const DistillArgs &a, long row, const Dense &d, const uint4 (&u)[C], int first, int end, Sparse &sp) {
    constexpr int V = Chunk<T>::n;
    T *out = static_cast<T *>(a.grad) + row * a.classes;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = first + ((int)threadIdx.x + c * THREADS) * V;
        float v[V];
        unpack(u[c], v);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = gradient(v[e], d);
        store_part(out + at, end - at, v);
    }
    __syncthreads();
    const T *l = static_cast<const T *>(a.logits) + row * a.stride;
    for (int j = threadIdx.x; j <= a.K; j += THREADS) {
        const int i = sp.idx[j];
        if (i < first || i >= end) continue;
        bool again = false;
        for (int h = 0; h < j; ++h) again = again || sp.idx[h] == i;
        if (again) continue;
        float off = 0.f;
        for (int h = j; h <= a.K; ++h) off += sp.idx[h] == i ? sp.off[h] : 0.f;
        put(out + i, gradient(ldf(l + i), d) - off);
    }
}

// The rows that count, at least one: by one workgroup
__global__ __launch_bounds__(1024) void distill_count_kernel(const DistillArgs a) {
    __shared__ float lds[16];
    int n = 0;
    for (long i = threadIdx.x; i < a.rows; i += 1024) n += counts(a, i);
    const float v = group_sum<16>((float)n, lds);   // (a thread's share is below 2^24)
    if (threadIdx.x == 0) a.stats[a.rows * kDistillStats] = fmaxf(v, 1.f);
}
// ... and with the rows' losses their mean
__global__ __launch_bounds__(1024) void distill_mean_kernel(const DistillArgs a, const float *__restrict__ losses) {
    __shared__ float lds[16];
    int n = 0;
    float s = 0.f;
    for (long i = threadIdx.x; i < a.rows; i += 1024) {
        n += counts(a, i);
        s += losses[i];
    }
    const float v = fmaxf(group_sum<16>((float)n, lds), 1.f);
    s = group_sum<16>(s, lds);
    if (threadIdx.x == 0) {
        a.stats[a.rows * kDistillStats] = v;
        a.loss[0] = s / v;
    }
}

// ---- a row in a workgroup's registers --------------------------------------------------------------------------------------
template <class T, int THREADS, int C, bool GRAD>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(const DistillArgs a, float *__restrict__ losses) {
    constexpr int V = Chunk<T>::n, WAVES = THREADS / 64;
    __shared__ float lds[16];
    __shared__ RowStats shared;
    __shared__ Sparse sp;
    const int lane = threadIdx.x & 63;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *l = static_cast<const T *>(a.logits) + row * a.stride;
        uint4 u[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = ((int)threadIdx.x + c * THREADS) * V;
            u[c] = load_logits(l + at, a.classes - at);
        }
        RowStats r;
        if (threadIdx.x < 64) teacher(a, row, lane, r);
        r.m = group_max<WAVES>(chunks_max<T, C>(u), lds);
        float s_o, s_q;
        chunks_sums<T, C>(a, u, r.m, s_o, s_q);
        r.log_o = logf(group_sum<WAVES>(s_o, lds));
        r.log_q = logf(group_sum<WAVES>(s_q, lds));
        r.spare = 0.f;
        if (threadIdx.x < 64) {
            const float loss = row_loss<T>(a, row, lane, r);
            if (lane == 0) {
                losses[row] = loss;
                reinterpret_cast<RowStats *>(a.stats)[row] = shared = r;
            }
        }
        if constexpr (GRAD) {
            __syncthreads();
            r = shared;
            const Dense d = dense_of(a, r, 1.f / (a.target ? a.stats[a.rows * kDistillStats] : (float)a.rows));
            fill_sparse(a, row, r, d.by_q, d.by_o, sp, THREADS);
            put_gradient<T, THREADS, C>(a, row, d, u, 0, a.classes, sp);
        }
        __syncthreads();   // (what is shared may be written again)
    }
}

// ---- a row shared by workgroups ----------------------------------------------------------------------------------------------
static constexpr int kPieceThreads = 256, kPieceChunks = 4;
template <class T>
static constexpr int kPiece = kPieceThreads * kPieceChunks * Chunk<T>::n;
struct PieceSums { float m, s_o, s_q; };

template <class T>
__global__ __launch_bounds__(kPieceThreads) void distill_piece_kernel(const DistillArgs a, PieceSums *__restrict__ parts, int pieces) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[16];
    const long items = a.rows * pieces;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long row = i / pieces;
        const int first = (int)(i - row * pieces) * kPiece<T>;
        const T *l = static_cast<const T *>(a.logits) + row * a.stride;
        uint4 u[kPieceChunks];
#pragma unroll
        for (int c = 0; c < kPieceChunks; ++c) {
            const int at = first + ((int)threadIdx.x + c * kPieceThreads) * V;
            u[c] = load_logits(l + at, a.classes - at);
        }
        const float m = group_max<kPieceThreads / 64>(chunks_max<T, kPieceChunks>(u), lds);
        float s_o, s_q;
        // (a piece whose logits are all -infinity adds nothing; one with a value that is no number, or +infinity, is no number)
        chunks_sums<T, kPieceChunks>(a, u, m > -__builtin_inff() ? m : 0.f, s_o, s_q);
        s_o = group_sum<kPieceThreads / 64>(s_o, lds);
        s_q = group_sum<kPieceThreads / 64>(s_q, lds);
        if (threadIdx.x == 0) parts[i] = PieceSums{m, s_o, s_q};
    }
}
// a wave a row
template <class T>
__global__ __launch_bounds__(64) void distill_join_kernel(const DistillArgs a, const PieceSums *__restrict__ parts, int pieces, float *__restrict__ losses) {
    const int lane = threadIdx.x;
    const float k = kLog2e / a.temperature;
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        RowStats r;
        teacher(a, row, lane, r);
        const PieceSums *q = parts + row * pieces;
        float m = -__builtin_inff(), s_o = 0.f, s_q = 0.f;
        for (int i = lane; i < pieces; i += 64) m = fmaxf(m, q[i].m);
        r.m = lanes_max<64>(m);
        for (int i = lane; i < pieces; i += 64) {
            const PieceSums t = q[i];
            // (a piece of -infinity: no sums, or none that is a number)
            s_o += t.m > -__builtin_inff() ? t.s_o * __builtin_amdgcn_exp2f((t.m - r.m) * kLog2e) : t.s_o;
            s_q += t.m > -__builtin_inff() ? t.s_q * __builtin_amdgcn_exp2f((t.m - r.m) * (wants_q(a) ? k : kLog2e)) : t.s_q;
        }
        r.log_o = logf(lanes_sum<64>(s_o));
        r.log_q = logf(lanes_sum<64>(s_q));
        if (!(r.m > -__builtin_inff())) r.log_o = r.log_q = __builtin_nanf("");
        r.spare = 0.f;
        const float loss = row_loss<T>(a, row, lane, r);
        if (lane == 0) {
            losses[row] = loss;
            reinterpret_cast<RowStats *>(a.stats)[row] = r;
        }
    }
}

// The backward, a piece at a time.  Nothing to do where the forward's gradient was for this loss's own.
template <class T>
__global__ __launch_bounds__(kPieceThreads) void distill_grad_kernel(const DistillArgs a, int pieces) {
    constexpr int V = Chunk<T>::n;
    __shared__ Sparse sp;
    const float up = a.grad_loss[0];
    if (a.unit && up == 1.f) return;
    const long items = a.rows * pieces;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long row = i / pieces;
        const int first = (int)(i - row * pieces) * kPiece<T>, end = first + kPiece<T> < a.classes ? first + kPiece<T> : a.classes;
        const T *l = static_cast<const T *>(a.logits) + row * a.stride;
        uint4 u[kPieceChunks];
#pragma unroll
        for (int c = 0; c < kPieceChunks; ++c) {
            const int at = first + ((int)threadIdx.x + c * kPieceThreads) * V;
            u[c] = load_logits(l + at, a.classes - at);
        }
        const RowStats r = reinterpret_cast<const RowStats *>(a.stats)[row];
        const Dense d = dense_of(a, r, up / a.stats[a.rows * kDistillStats]);
        fill_sparse(a, row, r, d.by_q, d.by_o, sp, kPieceThreads);
        put_gradient<T, kPieceThreads, kPieceChunks>(a, row, d, u, first, end, sp);
        __syncthreads();
    }
}

template <class T>
static long pieces_of(int classes) { return ceil_div_l(classes, kPiece<T>); }

// Rows that fit a workgroup's registers stay there where they are one piece, or where there is one for every compute unit
static constexpr int kRowChunks = 8192;
bool distill_in_rows(long rows, int classes, int type) {
    const long chunks = ceil_div_l(classes, type == ADDER_TYPE_BF16 ? 8 : 4);
    return chunks <= kPieceThreads * kPieceChunks || (chunks <= kRowChunks && rows >= 256);
}
size_t distill_workspace_bytes(long rows, int classes, int type) {
    const long pieces = type == ADDER_TYPE_BF16 ? pieces_of<bf16_t>(classes) : pieces_of<float>(classes);
    return sizeof(float) * (size_t)rows + (distill_in_rows(rows, classes, type) ? 0 : sizeof(PieceSums) * (size_t)rows * pieces);
}

static int most(long n, long groups) { return (int)(n < groups ? n : groups); }

template <class T, int THREADS, int C>
static void launch_row(const DistillArgs &a, float *losses, hipStream_t s) {
    const dim3 grid(most(a.rows, 1L << 20)), threads(THREADS);
    if (a.grad) hipLaunchKernelGGL((distill_row_kernel<T, THREADS, C, true>), grid, threads, 0, s, a, losses);
    else hipLaunchKernelGGL((distill_row_kernel<T, THREADS, C, false>), grid, threads, 0, s, a, losses);
}

template <class T>
int launch_distill_fwd(const DistillArgs &a, void *ws, hipStream_t s) {
    float *losses = static_cast<float *>(ws);
    if (distill_in_rows(a.rows, a.classes, sizeof(T) == 2 ? ADDER_TYPE_BF16 : ADDER_TYPE_F32)) {
        if (a.grad && a.target) {
            hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(1024), 0, s, a);
            if (int rc = check_launch()) return rc;
        }
        const long chunks = ceil_div_l(a.classes, Chunk<T>::n);
        if (chunks <= 64) launch_row<T, 64, 1>(a, losses, s);
        else if (chunks <= 256) launch_row<T, 256, 1>(a, losses, s);
        else if (chunks <= 512) launch_row<T, 256, 2>(a, losses, s);
        else if (chunks <= 1024) launch_row<T, 256, 4>(a, losses, s);
        else if (chunks <= 2048) launch_row<T, 512, 4>(a, losses, s);
        else if (chunks <= 4096) launch_row<T, 512, 8>(a, losses, s);
        else launch_row<T, 1024, 8>(a, losses, s);
    } else {
        const int pieces = (int)pieces_of<T>(a.classes);
        PieceSums *parts = reinterpret_cast<PieceSums *>(losses + a.rows);
        hipLaunchKernelGGL(distill_piece_kernel<T>, dim3(most(a.rows * pieces, 1L << 20)), dim3(kPieceThreads), 0, s, a, parts, pieces);
        if (int rc = check_launch()) return rc;
        hipLaunchKernelGGL(distill_join_kernel<T>, dim3(most(a.rows, 1L << 20)), dim3(64), 0, s, a, parts, pieces, losses);
    }
    if (int rc = check_launch()) return rc;
    hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, s, a, losses);
    return check_launch();
}

template <class T>
int launch_distill_bwd(const DistillArgs &a, hipStream_t s) {
    const int pieces = (int)pieces_of<T>(a.classes);
    hipLaunchKernelGGL(distill_grad_kernel<T>, dim3(most(a.rows * pieces, 4096)), dim3(kPieceThreads), 0, s, a, pieces);
    return check_launch();
}

#define ADDER_DISTILL_INSTANCE(T)                                              \
    template int launch_distill_fwd<T>(const DistillArgs &, void *, hipStream_t); \
    template int launch_distill_bwd<T>(const DistillArgs &, hipStream_t);
ADDER_DISTILL_INSTANCE(float)
ADDER_DISTILL_INSTANCE(bf16_t)

}  // namespace adder
