// The AdamW step for many tensors in one launch:
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//     p = p (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// with the moments held as floats, or as 8-bit codes of blocks of kStateBlock values that share the largest magnitude among
// them as their scale s:
//     m = sign(q) s (q / 127)^2, q in -127 .. 127,      v = s (q / 255)^4, q in 0 .. 255.
// The roots give small values more codes than a straight scale would (the second moment reaches down to 2e-10 of the block's
// largest), and they need no table.  Codes go to the nearest; a second moment that is not zero keeps a code that is not zero,
// since its root divides.  The parameter is updated with the moments before they are rounded.
// Memory decides: 28 bytes a float parameter with moments of 32 bits, 16 with moments of 8.  67 million float values: 340 us (5.5 TB/s)
// and 205 us (5.2 TB/s); in bfloat16 264 us (22 bytes, 5.6 TB/s) and 147 us (10 bytes, 4.6 TB/s: the roots and roundings of the codes
// begin to count).  65 small tensors, 272 000 values: 4.9 us.  The table of tensors travels by value in the kernel arguments, as
// that of the SGD step does.
#include "layers.hpp"

namespace adder {

// 1 / (1 - b1^t), 1 / sqrt(1 - b2^t): from the host, or from the device where the step count lives there
struct Corrections { float c1, c2; };
__device__ __forceinline__ Corrections corrections(const AdamWArgs &a) {
    return a.corr ? Corrections{a.corr[0], a.corr[1]} : Corrections{a.c1, a.c2};
}

struct AdamWBatch {
    void *p[kAdamWBatchMax];
    const void *g[kAdamWBatchMax];
    float *m[kAdamWBatchMax], *v[kAdamWBatchMax];
    int n[kAdamWBatchMax];
    int first_block[kAdamWBatchMax + 1];   // workgroups [first_block[t], first_block[t + 1]) belong to tensor t
};
struct AdamW8Batch {
    void *p[kAdamW8BatchMax];
    const void *g[kAdamW8BatchMax];
    int8_t *m[kAdamW8BatchMax];
    uint8_t *v[kAdamW8BatchMax];
    float *ms[kAdamW8BatchMax], *vs[kAdamW8BatchMax];
    int n[kAdamW8BatchMax];
    int first_block[kAdamW8BatchMax + 1];
};

// the last tensor whose first workgroup is not behind this one
template <class B>
__device__ __forceinline__ int tensor_of(const B &b, int count) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.first_block[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// The moments are rounded product by product, as the formulas are in float32.  The update's root and reciprocal are the plain instructions
// (one unit in its last place each).  The root's takes moments below the smallest normal float for zero; beside an eps of less than a
// root of those it is the exact one.
__device__ __forceinline__ float adamw_value(float p, float g, float &m, float &v, const AdamWArgs &a, const Corrections &c,
                                             float rate, float decay) {
    {
#pragma clang fp contract(off)
        m = a.b1 * m + a.one_b1 * g;
        v = a.b2 * v + a.one_b2 * g * g;
    }
    const float root = a.eps < 1e-12f ? sqrtf(v) : __builtin_amdgcn_sqrtf(v);
    return fmaf(-rate * c.c1, m * __builtin_amdgcn_rcpf(fmaf(root, c.c2, a.eps)), p * decay);
}

static constexpr int kAdamWThreads = 256, kAdamWChunk = 4 * kAdamWThreads;

// Up to four values at p, of which `left` exist
template <class T>
__device__ __forceinline__ void ld4(const T *p, int left, float (&v)[4]) {
    if (left >= 4) {
        ld_strip<4>(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = e < left ? ldf(p + e) : 0.f;
    }
}
template <class T>
__device__ __forceinline__ void st4(T *p, int left, const float (&v)[4]) {
    if (left >= 4) {
        put4(p, v);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < left) put(p + e, v[e]);
    }
}
typedef uint8_t u8x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ uint32_t ld_codes(const void *p, int left) {
    const uint8_t *q = static_cast<const uint8_t *>(p);
    if (left >= 4) return __builtin_bit_cast(uint32_t, *reinterpret_cast<const u8x4_any *>(q));
    uint32_t u = 0;
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (e < left) u |= (uint32_t)q[e] << (8 * e);
    return u;
}
__device__ __forceinline__ void st_codes(void *p, int left, uint32_t u) {
    uint8_t *q = static_cast<uint8_t *>(p);
    if (left >= 4) {
        *reinterpret_cast<u8x4_any *>(q) = __builtin_bit_cast(u8x4_any, u);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < left) q[e] = (uint8_t)(u >> (8 * e));
    }
}

template <class T>
__global__ __launch_bounds__(kAdamWThreads) void adamw_kernel(const AdamWBatch b, int count, const AdamWArgs a) {
    const int t = tensor_of(b, count);
    const int i = ((int)blockIdx.x - b.first_block[t]) * kAdamWChunk + (int)threadIdx.x * 4, left = b.n[t] - i;
    if (left <= 0) return;
    T *p = static_cast<T *>(b.p[t]) + i;
    const T *g = static_cast<const T *>(b.g[t]) + i;
    float *m = b.m[t] + i, *v = b.v[t] + i;
    const Corrections c = corrections(a);
    const float rate = a.lr_ptr ? *a.lr_ptr : a.lr, decay = a.lr_ptr ? 1.f - rate * a.weight_decay : a.decay;
    float pv[4], gv[4], mv[4], vv[4];
    ld4(p, left, pv);
    ld4(g, left, gv);
    ld4(m, left, mv);
    ld4(v, left, vv);
#pragma unroll
    for (int e = 0; e < 4; ++e) pv[e] = adamw_value(pv[e], gv[e], mv[e], vv[e], a, c, rate, decay);
    st4(p, left, pv);
    st4(m, left, mv);
    st4(v, left, vv);
}

// The larger of two values, not a number where one of them is none (fmaxf passes over it)
__device__ __forceinline__ float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Largest of G neighbouring lanes' values (32 or 64); not a number where one of them is none or infinite.
template <int G>
__device__ __forceinline__ float lanes_scale(float t) {
    t = maximum(t, dpp_row_move<0xB1>(t));
    t = maximum(t, dpp_row_move<0x4E>(t));
    t = maximum(t, dpp_row_move<0x141>(t));
    t = maximum(t, dpp_row_move<0x140>(t));
    t = maximum(t, __shfl_xor(t, 16, 64));
    if constexpr (G == 64) t = maximum(t, __shfl_xor(t, 32, 64));
    return t < __builtin_inff() ? t : __builtin_nanf("");
}

// What a value is multiplied with towards its code.  Scales of zero, below the smallest normal float, or not a number: codes of zero.
__device__ __forceinline__ float inverse(float scale) { return scale >= 0x1p-126f ? 1.f / scale : 0.f; }

__device__ __forceinline__ float first_moment(int q, float s) {
    const float d = (float)q * (1.f / 127.f);
    return s * (d * fabsf(d));
}
__device__ __forceinline__ float second_moment(unsigned q, float s) {
    const float r = (float)q, r2 = r * r;   // (exact)
    return r2 * r2 * (1.f / (255.f * 255.f * 255.f * 255.f)) * s;
}
// On the way to a code: a / s for a <= s and y = 1 / s, and a root; correctly rounded where EXACT, else to a unit in the last place.  Exact in
// float32, so that codes are those of the formulas in float32 arithmetic: else two in a million, next to a tie, go the other way, which the
// parameters of a step later show (67 million values: 205 us instead of 192).  A bfloat16 parameter does not (147 us).
template <bool EXACT>
__device__ __forceinline__ float share(float a, float s, float y) {
    const float d = a * y;
    return EXACT ? fmaf(fmaf(-s, d, a), y, d) : d;
}
template <bool EXACT>
__device__ __forceinline__ float root(float x) {
    if constexpr (!EXACT) return __builtin_amdgcn_sqrtf(x);
    const float y = __builtin_amdgcn_rsqf(fmaxf(x, 0x1p-120f)), g = x * y;
    return fmaf(fmaf(-g, g, x), 0.5f * y, g);
}

// A lane takes a chunk of 16 bytes of the parameter: a wave one block of the state in float32, two in bfloat16 (one: 165 us instead of 147
// for 64M values).  The block's largest moments are known only behind the update of all its values, so both stay in registers.
template <class T>
static constexpr int kAdamW8Chunk = Chunk<T>::n * kAdamWThreads;
template <class T>
__global__ __launch_bounds__(kAdamWThreads) void adamw_8bit_kernel(const AdamW8Batch b, int count, const AdamWArgs a) {
    constexpr int V = Chunk<T>::n, LANES = kStateBlock / V;
    constexpr bool EXACT = sizeof(T) == 4;
    static_assert(LANES == 64 || LANES == 32, "whole waves or halves");
    const int t = tensor_of(b, count);
    const int i = ((int)blockIdx.x - b.first_block[t]) * kAdamW8Chunk<T> + (int)threadIdx.x * V, left = b.n[t] - i;
    if (__all(left <= 0)) return;
    T *p = static_cast<T *>(b.p[t]) + i;
    const T *g = static_cast<const T *>(b.g[t]) + i;
    const int block = (left > 0 ? i : b.n[t] - 1) / kStateBlock;   // (lanes beside the tensor: the last one, of which they read and write no value)
    const Corrections c = corrections(a);
    const float rate = a.lr_ptr ? *a.lr_ptr : a.lr, decay = a.lr_ptr ? 1.f - rate * a.weight_decay : a.decay;
    const float ms = b.ms[t][block], vs = b.vs[t][block];
    float pv[V], gv[V], mv[V], vv[V];
    load_part(p, left, pv);
    load_part(g, left, gv);
    uint32_t mq[V / 4], vq[V / 4];
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
        mq[h] = ld_codes(b.m[t] + i + 4 * h, left - 4 * h);
        vq[h] = ld_codes(b.v[t] + i + 4 * h, left - 4 * h);
    }
    float mtop = 0.f, vtop = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {   // (beside the tensor: zeros)
        mv[e] = first_moment((int8_t)(mq[e / 4] >> (8 * (e & 3))), ms);
        vv[e] = second_moment((vq[e / 4] >> (8 * (e & 3))) & 255u, vs);
        pv[e] = adamw_value(pv[e], gv[e], mv[e], vv[e], a, c, rate, decay);
        mtop = maximum(mtop, fabsf(mv[e]));
        vtop = maximum(vtop, vv[e]);
    }
    store_part(p, left, pv);
    const float ns = lanes_scale<LANES>(mtop), ws = lanes_scale<LANES>(vtop);
    const float im = inverse(ns), iv = inverse(ws);
#pragma unroll
    for (int h = 0; h < V / 4; ++h) {
        mq[h] = vq[h] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float m = mv[4 * h + e], v = vv[4 * h + e];
            const float rm = copysignf(rintf(127.f * root<EXACT>(share<EXACT>(fabsf(m), ns, im))), m);
            const float rv = rintf(255.f * root<EXACT>(root<EXACT>(share<EXACT>(v, ws, iv))));
            mq[h] = __builtin_amdgcn_cvt_pk_u8_f32(rm < 0.f ? rm + 256.f : rm, e, mq[h]);   // (two's complement)
            vq[h] = __builtin_amdgcn_cvt_pk_u8_f32(fmaxf(rv, v > 0.f ? 1.f : 0.f), e, vq[h]);
        }
        st_codes(b.m[t] + i + 4 * h, left - 4 * h, mq[h]);
        st_codes(b.v[t] + i + 4 * h, left - 4 * h, vq[h]);
    }
    if ((threadIdx.x & (LANES - 1)) == 0 && left > 0) {
        b.ms[t][block] = ns;
        b.vs[t][block] = ws;
    }
}

// step[0] += 1, and the corrections of the new count: for steps whose count lives on the device, so that a captured graph counts
// on.  In 64 bits: 1 - b2^t is a difference of nearly equal numbers for the first steps.
__global__ void adamw_advance_kernel(float *step, double ln_b1, double ln_b2, float *corr) {
    const double t = (double)*step + 1.0;
    *step = (float)t;
    corr[0] = (float)(-1.0 / expm1(t * ln_b1));
    corr[1] = (float)(1.0 / sqrt(-expm1(t * ln_b2)));
}

// Eight codes a thread, a bfloat16 store of 16 bytes: 38 us for 64M values (5.2 TB/s; four a thread: 58 us)
static constexpr int kValuesPer = 8;
template <class T>
__global__ __launch_bounds__(256) void state_values_kernel(const void *codes, int is_signed, const float *__restrict__ scales,
                                                           T *__restrict__ out, long n) {
    const long i = ((long)blockIdx.x * 256 + threadIdx.x) * kValuesPer;
    if (i >= n) return;
    const int left = (int)(n - i < kValuesPer ? n - i : kValuesPer);
    const float s = scales[i / kStateBlock];
    const uint8_t *from = static_cast<const uint8_t *>(codes) + i;
    uint32_t q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) q[h] = ld_codes(from + 4 * h, left - 4 * h);
    float v[kValuesPer];
#pragma unroll
    for (int e = 0; e < kValuesPer; ++e) {
        const unsigned u = (q[e / 4] >> (8 * (e & 3))) & 255u;
        v[e] = is_signed ? first_moment((int8_t)u, s) : second_moment(u, s);
    }
    if constexpr (sizeof(T) == 2) {
        store_part(out + i, left, v);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float w[4] = {v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]};
            store_part(out + i + 4 * h, left - 4 * h, w);
        }
    }
}

template <class B, class F>
static int fill_blocks(B &b, int count, const long *n, int chunk, F more) {
    int blocks = 0;
    for (int t = 0; t < count; ++t) {
        b.n[t] = (int)n[t];
        b.first_block[t] = blocks;
        blocks += (int)ceil_div_l(n[t], chunk);
        more(t);
    }
    b.first_block[count] = blocks;
    return blocks;
}

template <class T>
int launch_adamw(int count, void *const *p, const void *const *g, float *const *m, float *const *v, const long *n, const AdamWArgs &a,
                 hipStream_t s) {
    AdamWBatch b;
    const int blocks = fill_blocks(b, count, n, kAdamWChunk, [&](int t) {
        b.p[t] = p[t]; b.g[t] = g[t]; b.m[t] = m[t]; b.v[t] = v[t];
    });
    hipLaunchKernelGGL(adamw_kernel<T>, dim3(blocks), dim3(kAdamWThreads), 0, s, b, count, a);
    return check_launch();
}

template <class T>
int launch_adamw_8bit(int count, void *const *p, const void *const *g, int8_t *const *m, uint8_t *const *v, float *const *ms,
                      float *const *vs, const long *n, const AdamWArgs &a, hipStream_t s) {
    AdamW8Batch b;
    const int blocks = fill_blocks(b, count, n, kAdamW8Chunk<T>, [&](int t) {
        b.p[t] = p[t]; b.g[t] = g[t]; b.m[t] = m[t]; b.v[t] = v[t]; b.ms[t] = ms[t]; b.vs[t] = vs[t];
    });
    hipLaunchKernelGGL(adamw_8bit_kernel<T>, dim3(blocks), dim3(kAdamWThreads), 0, s, b, count, a);
    return check_launch();
}

int launch_adamw_advance(float *step, double ln_b1, double ln_b2, float *corr, hipStream_t s) {
    hipLaunchKernelGGL(adamw_advance_kernel, dim3(1), dim3(1), 0, s, step, ln_b1, ln_b2, corr);
    return check_launch();
}

template <class T>
int launch_state_values(const void *codes, int is_signed, const float *scales, T *out, long n, hipStream_t s) {
    hipLaunchKernelGGL(state_values_kernel<T>, dim3((unsigned)ceil_div_l(n, 256 * kValuesPer)), dim3(256), 0, s, codes, is_signed, scales, out, n);
    return check_launch();
}

#define ADDER_ADAMW_INSTANCE(T)                                                                                                      \
    template int launch_adamw<T>(int, void *const *, const void *const *, float *const *, float *const *, const long *,             \
                                 const AdamWArgs &, hipStream_t);                                                                   \
    template int launch_adamw_8bit<T>(int, void *const *, const void *const *, int8_t *const *, uint8_t *const *, float *const *,   \
                                      float *const *, const long *, const AdamWArgs &, hipStream_t);                                \
    template int launch_state_values<T>(const void *, int, const float *, T *, long, hipStream_t);
ADDER_ADAMW_INSTANCE(float)
ADDER_ADAMW_INSTANCE(bf16_t)

}  // namespace adder
