// The loss against a teacher's K largest logits t at the classes i, and the labels y, over all C classes of the logits l, and its gradient:
//     q = softmax(l / T),  o = softmax(l),  p = softmax(t / T) over the K
//     row = a T^2 sum_k p_k (log p_k - log q[i_k]) - (1 - a) log o[y],     loss = sum of the rows that count / their number
//     dl = 1 / number (a T (q - p at the classes i) + (1 - a) (o - 1 at y))
// Memory decides: l is read and dl written.  Where there are rows enough a workgroup keeps a row in registers: it reads it once, and
// writes the gradient for a loss whose own gradient is one on the way; the backward of any other computes it again.  Where rows are few
// and long several workgroups share one, and the gradient is the backward's.  All sums in a fixed order.
// 4096 x 32000 in bfloat16, 64 of the teacher's, T = 2: 108 to 116 us (4.5 to 4.9 TB/s), and 4 each for the rows that count, the mean and the backward that
// finds nothing to do; 256 x 1000 in float32 6.2 us.
#include "blocks.hpp"

#include <type_traits>

namespace adder {

static constexpr int kTeacherMost = ADDER_DISTILL_TOP_MAX;
static constexpr float kLog2e = 1.44269504f;
// What a row's loss and gradient are made of.  m, top: the largest logit, the teacher's; log_*: logarithms of the sums of exponentials
// behind them; by_*: factors of q and o in the gradient, zero where that part is not there (no teacher's logit above -infinity, a row that
// does not count), not a number where a class does not exist or a teacher's logit is +infinity or none.  Behind the last row's: the rows that count, in m.
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
// (a row's offsets are 32 bits: its base is one for the workgroup)
template <class T>
__device__ __forceinline__ T *from(T *row, int at) {
    return reinterpret_cast<T *>(reinterpret_cast<char *>(const_cast<std::remove_const_t<T> *>(row)) + (unsigned)at * (unsigned)sizeof(T));
}
// A thread's chunks, (thread + c THREADS) from `first` on, of `classes` logits; the one chunk that ends beyond them is put together once.
template <class T, int THREADS, int C>
__device__ __forceinline__ void load_chunks(const T *l, int first, int classes, uint4 (&u)[C]) {
    constexpr int V = Chunk<T>::n;
    const int whole = classes & ~(V - 1);
    const uint32_t none = V == 4 ? 0xff800000u : 0xff80ff80u;
    uint4 tail = make_uint4(none, none, none, none);
    if (whole < classes && whole >= first && whole < first + THREADS * C * V) tail = load_logits(l + whole, classes - whole);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int at = first + ((int)threadIdx.x + c * THREADS) * V;
        u[c] = make_uint4(none, none, none, none);
        if (at < whole) u[c] = load_raw(from(l, at));
        else if (at == whole) u[c] = tail;
    }
}

// Largest, and sums, over a workgroup: every wave leaves its own in a place of its own, and reads all behind a barrier that the caller has
__device__ __forceinline__ void leave(float *lds, float v) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
}
template <int WAVES>
__device__ __forceinline__ float all_max(const float *lds) {   // (beside a number, one that is none is left out: the sums find it)
    float v = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = fmaxf(v, lds[i]);
    return v;
}
template <int WAVES>
__device__ __forceinline__ float all_sum(const float *lds) {
    float v = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v += lds[i];
    return v;
}
template <int WAVES>
__device__ __forceinline__ float group_sum(float v, float *lds) {
    leave(lds, lanes_sum<64>(v));
    __syncthreads();
    v = all_sum<WAVES>(lds);
    __syncthreads();
    return v;
}

// How the exponentials of l / T and of l come: one of them (the other is not wanted, or T is one), the second as a power of the first (T two or
// four: a multiplication where an instruction for an exponential takes the time of four), or each by itself.
// The exponents are of differences from the row's largest, (l - m) / T: l / T - m / T would save an instruction (104 us for 108 at 4096 x 32000)
// and lose digits, and all of them where a row lies far from zero or is masked by the type's lowest value.
enum class Both { one, square, fourth, apart };
__device__ __forceinline__ Both both_of(const DistillArgs &a) {
    if (!wants_q(a) || !wants_o(a) || a.temperature == 1.f) return Both::one;
    return a.temperature == 2.f ? Both::square : a.temperature == 4.f ? Both::fourth : Both::apart;
}
__device__ __forceinline__ float scale_q(const DistillArgs &a) { return wants_q(a) ? kLog2e / a.temperature : kLog2e; }
template <Both B>
__device__ __forceinline__ void add_exponentials(float v, float k, float m, float &s_q, float &s_o) {   // of (v - m) k ln 2 and v - m
    const float q = __builtin_amdgcn_exp2f((v - m) * k), p = q * q;
    s_q += q;
    if constexpr (B == Both::square) s_o = fmaf(q, q, s_o);
    if constexpr (B == Both::fourth) s_o = fmaf(p, p, s_o);
    if constexpr (B == Both::apart) s_o += __builtin_amdgcn_exp2f((v - m) * kLog2e);
}
template <class F>
__device__ __forceinline__ void by_mode(Both b, const F &f) {
    switch (b) {
        case Both::one: f(std::integral_constant<Both, Both::one>{}); break;
        case Both::square: f(std::integral_constant<Both, Both::square>{}); break;
        case Both::fourth: f(std::integral_constant<Both, Both::fourth>{}); break;
        default: f(std::integral_constant<Both, Both::apart>{});
    }
}

// The chunks stay as they are from one walk over them to the next (else the compiler keeps their values as floats, twice the registers)
template <int C>
__device__ __forceinline__ void pack_again(uint4 (&u)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) asm volatile("" : "+v"(u[c].x), "+v"(u[c].y), "+v"(u[c].z), "+v"(u[c].w));
}
template <class T, int C>
__device__ __forceinline__ float chunks_max(const uint4 (&u)[C]) {
    float m = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float v[Chunk<T>::n];
        unpack(u[c], v);
#pragma unroll
        for (int e = 0; e < Chunk<T>::n; e += 2) m = fmaxf(fmaxf(m, v[e]), v[e + 1]);
    }
    return m;
}
// A thread's sums of the exponentials behind m
template <class T, int C>
__device__ __forceinline__ void chunks_sums(const DistillArgs &a, const uint4 (&u)[C], float m, float &s_o, float &s_q) {
    const float k = scale_q(a);
    float o = 0.f, q = 0.f;
    by_mode(both_of(a), [&](auto mode) {
        constexpr Both B = decltype(mode)::value;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float v[Chunk<T>::n];
            unpack(u[c], v);
#pragma unroll
            for (int e = 0; e < Chunk<T>::n; ++e) add_exponentials<B>(v[e], k, m, q, o);
            __builtin_amdgcn_sched_barrier(0);   // (one chunk's values at a time)
        }
        if constexpr (B == Both::one) o = q;
    });
    s_o = o;
    s_q = q;
}

// The classes that the teacher and, behind them, the label name, in LDS: the class (-1: none, or none that exists), the teacher's logit and later
// what is taken off the gradient there, the student's logit
struct Sparse {
    int idx[kTeacherMost + 1];
    float off[kTeacherMost + 1], logit[kTeacherMost + 1];
};
// One entry on its way: first its class and the teacher's logit, then the student's there
struct Entry { long long i; float t; };
__device__ __forceinline__ Entry load_entry(const DistillArgs &a, long row, int j) {
    const bool label = j == a.K, none = j > a.K || !counts(a, row) || !(label ? wants_o(a) : wants_q(a));
    return {none ? -1 : label ? a.target[row] : a.idx[row * a.K + j], j < a.K ? teacher_logit(a, row * a.K + j) : 0.f};
}
template <class T>
__device__ __forceinline__ void put_entry(const DistillArgs &a, const T *l, int j, const Entry &e, Sparse &sp) {
    const bool there = exists(a, e.i);
    const float v = there ? ldf(l + e.i) : 0.f;
    sp.idx[j] = there ? (int)e.i : -1;
    sp.off[j] = e.t;
    sp.logit[j] = v;
}
// All entries, and what `between` loads; a thread's first entry is on its way before that, so that nothing waits twice
template <class T, class F>
__device__ __forceinline__ void fill_sparse(const DistillArgs &a, long row, Sparse &sp, int threads, const F &between) {
    const T *l = static_cast<const T *>(a.logits) + row * a.stride;
    int j = threadIdx.x;
    const Entry e = load_entry(a, row, j);
    between(l);
    if (j <= a.K) put_entry(a, l, j, e, sp);
    for (j += threads; j <= a.K; j += threads) put_entry(a, l, j, load_entry(a, row, j), sp);
}
// A row with a logit of +infinity, or one that is no number, or nothing but -infinity, is no number as a whole
__device__ __forceinline__ float log_sum(float s) { return s > 0.f && s < __builtin_inff() ? logf(s) : __builtin_nanf(""); }
// One wave: the teacher's softmax and the factors of the gradient
__device__ __forceinline__ void teacher(const DistillArgs &a, long row, const Sparse &sp, RowStats &r) {
    const int lane = threadIdx.x & 63;
    const float k = kLog2e / a.temperature, nan = __builtin_nanf("");
    const bool on = counts(a, row);
    r.top = r.log_p = r.by_q = 0.f;
    if (on && wants_q(a)) {
        float m = -__builtin_inff(), s = 0.f;
        bool bad = false;
        for (int j = lane; j < a.K; j += 64) {
            const float t = sp.off[j];
            m = fmaxf(m, t);
            bad = bad || (sp.idx[j] < 0 && t > -__builtin_inff()) || !(t < __builtin_inff());   // (one of -infinity may name any class)
        }
        m = lanes_max<64>(m);
        const bool taught = m > -__builtin_inff();
        for (int j = lane; j < a.K; j += 64) s += taught ? __builtin_amdgcn_exp2f((sp.off[j] - m) * k) : 0.f;
        s = lanes_sum<64>(s);
        r.top = taught ? m : 0.f;
        r.log_p = taught ? logf(s) : 0.f;
        r.by_q = __any(bad) ? nan : taught ? (a.target ? a.alpha : 1.f) * a.temperature : 0.f;
    }
    r.by_o = on && wants_o(a) ? sp.idx[a.K] >= 0 ? 1.f - a.alpha : nan : 0.f;
}
// ... and the row's loss, once its own statistics are there
__device__ __forceinline__ float row_loss(const DistillArgs &a, const Sparse &sp, const RowStats &r) {
    const float inv = 1.f / a.temperature;
    float loss = 0.f;
    if (r.by_q != 0.f) {   // (also where it is no number)
        float kd = 0.f;
        for (int j = threadIdx.x & 63; j < a.K; j += 64) {
            const float log_p = (sp.off[j] - r.top) * inv - r.log_p, p = expf(log_p), log_q = (sp.logit[j] - r.m) * inv - r.log_q;
            kd += p == 0.f ? 0.f : p * (log_p - log_q);
        }
        loss = r.by_q * a.temperature * lanes_sum<64>(kd);
    }
    if (r.by_o != 0.f) loss -= r.by_o * (sp.logit[a.K] - r.m - r.log_o);
    return loss;
}

// The dense part of a row's gradient: q and o are the exponentials behind m, times these
struct Dense { float m, k, by_q, by_o; };
__device__ __forceinline__ Dense dense_of(const DistillArgs &a, const RowStats &r, float up) {
    const float k = scale_q(a);
    Dense d{r.m, k, r.by_q != 0.f ? r.by_q * up * expf(-r.log_q) : 0.f, r.by_o != 0.f ? r.by_o * up * expf(-r.log_o) : 0.f};
    if (both_of(a) == Both::one) d.by_q += d.by_o;
    return d;
}
template <Both B>
__device__ __forceinline__ float gradient(float l, const Dense &d) {
    const float q = __builtin_amdgcn_exp2f((l - d.m) * d.k);
    if constexpr (B == Both::one) return d.by_q * q;
    else if constexpr (B == Both::square) return q * fmaf(d.by_o, q, d.by_q);
    else if constexpr (B == Both::fourth) return q * fmaf(d.by_o, q * q * q, d.by_q);
    else return fmaf(d.by_q, q, d.by_o * __builtin_amdgcn_exp2f((l - d.m) * kLog2e));
}
// The teacher's logits in `sp` become what is taken off the gradient
__device__ __forceinline__ void fill_off(const DistillArgs &a, const RowStats &r, float up, Sparse &sp, int threads) {
    const float inv = 1.f / a.temperature;
    for (int j = threadIdx.x; j <= a.K; j += threads) {
        const float by = j == a.K ? r.by_o : r.by_q;
        sp.off[j] = by == 0.f ? 0.f : j == a.K ? by * up : by * up * expf((sp.off[j] - r.top) * inv - r.log_p);
    }
}
// The gradient of the classes from `first` to `end`: everywhere first, then again where something is taken off -- once a class, by the first of
// its entries.  (All threads together.  `sp` was filled by these threads; behind it, it may be filled anew after a barrier.)
template <class T, int THREADS, int C>
__device__ __forceinline__ void put_gradient(const DistillArgs &a, long row, const Dense &d, const uint4 (&u)[C], int first, int end, const Sparse &sp) {
    constexpr int V = Chunk<T>::n;
    T *out = static_cast<T *>(a.grad) + row * a.classes;
    const int whole = end & ~(V - 1);   // (pieces begin at multiples of V)
    const bool none = d.by_q == 0.f && d.by_o == 0.f;   // (a row that does not count, whatever its logits are)
    by_mode(both_of(a), [&](auto mode) {
        uint4 tail = make_uint4(0, 0, 0, 0);
        bool mine = false;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int at = first + ((int)threadIdx.x + c * THREADS) * V;
            float v[V];
            unpack(u[c], v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = gradient<decltype(mode)::value>(v[e], d);
            uint4 o = pack(v);
            if (none) o = make_uint4(0, 0, 0, 0);
            if (at < whole) store_raw(from(out, at), o);
            if (at == whole) {
                tail = o;
                mine = true;
            }
            __builtin_amdgcn_sched_barrier(0);   // (one chunk's values at a time)
        }
        if (mine && whole < end) {
            float v[V];
            unpack(tail, v);
            store_part(out + whole, end - whole, v);
        }
        __syncthreads();
        if (none) return;
        // eight entries a wave, eight lanes each, which share the entries that may name the same class
        const int lane = threadIdx.x & 63, part = lane & 7;
        for (int j0 = (int)(threadIdx.x >> 6) * 8; j0 <= a.K; j0 += THREADS / 8) {
            const int j = j0 + (lane >> 3), i = j <= a.K ? sp.idx[j] : -1;
            const bool in = i >= first && i < end;
            float off = 0.f, before = 0.f;
#pragma unroll 4
            for (int h = part; h <= a.K; h += 8) {
                const bool same = in && sp.idx[h] == i;
                before += same && h < j ? 1.f : 0.f;
                off += same ? sp.off[h] : 0.f;
            }
            off = lanes_sum<8>(off);
            before = lanes_sum<8>(before);
            if (in && part == 0 && before == 0.f) put(out + i, gradient<decltype(mode)::value>(sp.logit[j], d) - off);
        }
    });
}

// The rows that count, at least one: by one workgroup
__global__ __launch_bounds__(1024) void distill_count_kernel(const DistillArgs a) {
    __shared__ float lds[16];
    int n = 0;
#pragma unroll 4
    for (long i = threadIdx.x; i < a.rows; i += 1024) n += counts(a, i);
    const float v = group_sum<16>((float)n, lds);   // (a thread's share is below 2^24)
    if (threadIdx.x == 0) a.stats[a.rows * kDistillStats] = fmaxf(v, 1.f);
}
// ... and with the rows' losses their mean
__global__ __launch_bounds__(1024) void distill_mean_kernel(const DistillArgs a, const float *__restrict__ losses) {
    __shared__ float lds[16];
    int n = 0;
    float s = 0.f;
#pragma unroll 4
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

// Up to so many rows every workgroup of up to so many threads counts those that count itself (a launch of 2 us less; the larger ones have no
// registers left for it: 4096 x 32000 took 155 us instead of 120)
static constexpr long kCountRows = 2048;
static constexpr int kCountThreads = 256;

// ---- a row in a workgroup's registers --------------------------------------------------------------------------------------
template <class T, int THREADS, int C>
__global__ __launch_bounds__(THREADS) void distill_row_kernel(const DistillArgs a, float *__restrict__ losses, long row0) {
    constexpr int WAVES = THREADS / 64;
    __shared__ float lds[4][WAVES];
    __shared__ RowStats shared;
    __shared__ Sparse sp;
    const long row = row0 + blockIdx.x;
    // the rows that count: few are counted here, beside the loads
    const bool count_here = THREADS <= kCountThreads && a.grad && a.target && a.rows <= kCountRows;
    float n = a.grad && a.target && !count_here ? a.stats[a.rows * kDistillStats] : (float)a.rows;
    uint4 u[C];
    fill_sparse<T>(a, row, sp, THREADS, [&](const T *l) { load_chunks<T, THREADS, C>(l, 0, a.classes, u); });
    if (count_here) {
        n = 0.f;
        for (int i = threadIdx.x; i < a.rows; i += THREADS) n += counts(a, i) ? 1.f : 0.f;
        leave(lds[3], lanes_sum<64>(n));
    }
    leave(lds[0], lanes_max<64>(chunks_max<T, C>(u)));
    __syncthreads();
    if (count_here) n = fmaxf(all_sum<WAVES>(lds[3]), 1.f);
    const float m = all_max<WAVES>(lds[0]);
    RowStats r;
    if (threadIdx.x < 64) {
        teacher(a, row, sp, r);
        if (threadIdx.x == 0) shared = r;
    }
    float s_o, s_q;
    pack_again(u);
    chunks_sums<T, C>(a, u, m, s_o, s_q);
    pack_again(u);
    leave(lds[1], lanes_sum<64>(s_o));
    leave(lds[2], lanes_sum<64>(s_q));
    __syncthreads();
    r = shared;
    r.m = m;
    r.log_o = log_sum(all_sum<WAVES>(lds[1]));
    r.log_q = log_sum(all_sum<WAVES>(lds[2]));
    r.spare = 0.f;
    if (threadIdx.x < 64) {
        const float loss = row_loss(a, sp, r);
        if (threadIdx.x == 0) {
            losses[row] = loss;
            reinterpret_cast<RowStats *>(a.stats)[row] = r;
        }
    }
    if (!a.grad) return;
    const float up = 1.f / n;
    if constexpr (WAVES > 1) __syncthreads();   // (the loss has been taken from the teacher's logits)
    fill_off(a, r, up, sp, THREADS);
    put_gradient<T, THREADS, C>(a, row, dense_of(a, r, up), u, 0, a.classes, sp);
}

// ---- a row shared by workgroups ----------------------------------------------------------------------------------------------
static constexpr int kPieceThreads = 256, kPieceChunks = 4;
template <class T>
static constexpr int kPiece = kPieceThreads * kPieceChunks * Chunk<T>::n;
struct PieceSums { float m, s_o, s_q; };

template <class T>
__global__ __launch_bounds__(kPieceThreads) void distill_piece_kernel(const DistillArgs a, PieceSums *__restrict__ parts, int pieces) {
    constexpr int WAVES = kPieceThreads / 64;
    __shared__ float lds[3][WAVES];
    const long items = a.rows * pieces;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long row = i / pieces;
        uint4 u[kPieceChunks];
        load_chunks<T, kPieceThreads, kPieceChunks>(static_cast<const T *>(a.logits) + row * a.stride, (int)(i - row * pieces) * kPiece<T>, a.classes, u);
        leave(lds[0], lanes_max<64>(chunks_max<T, kPieceChunks>(u)));
        __syncthreads();
        const float m = all_max<WAVES>(lds[0]);
        float s_o, s_q;
        pack_again(u);
        // (a piece whose logits are all -infinity adds nothing; one with a value that is no number, or +infinity, is no number)
        chunks_sums<T, kPieceChunks>(a, u, m > -__builtin_inff() ? m : 0.f, s_o, s_q);
        leave(lds[1], lanes_sum<64>(s_o));
        leave(lds[2], lanes_sum<64>(s_q));
        __syncthreads();
        if (threadIdx.x == 0) parts[i] = PieceSums{m, all_sum<WAVES>(lds[1]), all_sum<WAVES>(lds[2])};
    }
}
// a wave a row
template <class T>
__global__ __launch_bounds__(64) void distill_join_kernel(const DistillArgs a, const PieceSums *__restrict__ parts, int pieces, float *__restrict__ losses) {
    __shared__ Sparse sp;
    const int lane = threadIdx.x;
    const float k = scale_q(a);
    for (long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        fill_sparse<T>(a, row, sp, 64, [](const T *) {});
        const PieceSums *q = parts + row * pieces;
        float m = -__builtin_inff(), s_o = 0.f, s_q = 0.f;
        for (int i = lane; i < pieces; i += 64) m = fmaxf(m, q[i].m);
        m = lanes_max<64>(m);
        for (int i = lane; i < pieces; i += 64) {
            const PieceSums t = q[i];
            // (a piece of -infinity: no sums, or none that is a number)
            const bool some = t.m > -__builtin_inff();
            s_o += some ? t.s_o * __builtin_amdgcn_exp2f((t.m - m) * (both_of(a) == Both::one ? k : kLog2e)) : t.s_o;
            s_q += some ? t.s_q * __builtin_amdgcn_exp2f((t.m - m) * k) : t.s_q;
        }
        __syncthreads();
        RowStats r;
        teacher(a, row, sp, r);
        r.m = m;
        r.log_o = log_sum(lanes_sum<64>(s_o));
        r.log_q = log_sum(lanes_sum<64>(s_q));
        r.spare = 0.f;
        const float loss = row_loss(a, sp, r);
        if (lane == 0) {
            losses[row] = loss;
            reinterpret_cast<RowStats *>(a.stats)[row] = r;
        }
        __syncthreads();
    }
}

// The backward, a piece at a time.  Nothing to do where the forward's gradient was for this loss's own.
template <class T>
__global__ __launch_bounds__(kPieceThreads) void distill_grad_kernel(const DistillArgs a, int pieces) {
    __shared__ Sparse sp;
    const float loss_grad = a.grad_loss[0];
    if (a.unit && loss_grad == 1.f) return;
    const float up = loss_grad / a.stats[a.rows * kDistillStats];
    const long items = a.rows * pieces;
    for (long i = blockIdx.x; i < items; i += gridDim.x) {
        const long row = i / pieces;
        const int first = (int)(i - row * pieces) * kPiece<T>, end = a.classes - first < kPiece<T> ? a.classes : first + kPiece<T>;
        uint4 u[kPieceChunks];
        fill_sparse<T>(a, row, sp, kPieceThreads, [&](const T *l) { load_chunks<T, kPieceThreads, kPieceChunks>(l, first, a.classes, u); });
        const RowStats r = reinterpret_cast<const RowStats *>(a.stats)[row];
        fill_off(a, r, up, sp, kPieceThreads);   // (a thread's own entries)
        put_gradient<T, kPieceThreads, kPieceChunks>(a, row, dense_of(a, r, up), u, first, end, sp);
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
    for (long row = 0; row < a.rows; row += 1L << 20)   // (a launch has at most 2^32 threads)
        hipLaunchKernelGGL((distill_row_kernel<T, THREADS, C>), dim3(most(a.rows - row, 1L << 20)), dim3(THREADS), 0, s, a, losses, row);
}

template <class T>
int launch_distill_fwd(const DistillArgs &a, void *ws, hipStream_t s) {
    float *losses = static_cast<float *>(ws);
    if (distill_in_rows(a.rows, a.classes, sizeof(T) == 2 ? ADDER_TYPE_BF16 : ADDER_TYPE_F32)) {
        const long chunks = ceil_div_l(a.classes, Chunk<T>::n);
        if (a.grad && a.target && (a.rows > kCountRows || chunks > kCountThreads * 4)) {   // (as the shapes below)
            hipLaunchKernelGGL(distill_count_kernel, dim3(1), dim3(1024), 0, s, a);
            if (int rc = check_launch()) return rc;
        }
        if (chunks <= 64) launch_row<T, 64, 1>(a, losses, s);
        else if (chunks <= 256) launch_row<T, 256, 1>(a, losses, s);
        else if (chunks <= 512) launch_row<T, 256, 2>(a, losses, s);
        else if (chunks <= 1024) launch_row<T, 256, 4>(a, losses, s);
        else if (chunks <= 2048) launch_row<T, 512, 4>(a, losses, s);
        else if (chunks <= 4096) launch_row<T, 1024, 4>(a, losses, s);
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
    hipLaunchKernelGGL(distill_grad_kernel<T>, dim3(most(a.rows * pieces, 1024)), dim3(kPieceThreads), 0, s, a, pieces);
    return check_launch();
}

#define ADDER_DISTILL_INSTANCE(T)                                              \
    template int launch_distill_fwd<T>(const DistillArgs &, void *, hipStream_t); \
    template int launch_distill_bwd<T>(const DistillArgs &, hipStream_t);
ADDER_DISTILL_INSTANCE(float)
ADDER_DISTILL_INSTANCE(bf16_t)

}  // namespace adder
