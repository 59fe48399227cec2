// Device and host helpers of the layers that are not adder layers: layer normalisation (layer_norm.hip), linear layers
// (linear*.hip) and the AdamW step (adamw.hip).
#pragma once
#include "common.hpp"

namespace adder {

// Values of 16 bytes that lie side by side in memory, at an address aligned to one value only (global memory takes loads and
// stores of any alignment), as floats.
typedef uint16_t u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t u32x4_any4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_any2 __attribute__((ext_vector_type(4), aligned(2)));
template <class T>
struct Chunk;
template <>
struct Chunk<float> {
    static constexpr int n = 4;
    typedef u32x4_any4 raw;
};
template <>
struct Chunk<bf16_t> {
    static constexpr int n = 8;
    typedef u32x4_any2 raw;
};
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ void unpack(const uint4 &u, float (&v)[8]) {
    v[0] = __uint_as_float(u.x << 16); v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16); v[3] = __uint_as_float(u.y & 0xffff0000u);
    v[4] = __uint_as_float(u.z << 16); v[5] = __uint_as_float(u.z & 0xffff0000u);
    v[6] = __uint_as_float(u.w << 16); v[7] = __uint_as_float(u.w & 0xffff0000u);
}
// Two floats rounded to bfloat16, to nearest even, not-a-number kept (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    const pair p = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ bf16_t round_bf16(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
__device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
__device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
}
__device__ __forceinline__ void put(float *p, float v) { *p = v; }
__device__ __forceinline__ void put(bf16_t *p, float v) { *p = round_bf16(v); }
// four values at an address aligned to one
__device__ __forceinline__ void put4(float *p, const float (&v)[4]) { st_strip<4>(p, v); }
__device__ __forceinline__ void put4(bf16_t *p, const float (&v)[4]) {
    const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
    *reinterpret_cast<u16x4_any *>(p) = u16x4_any{(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
}

template <class T>
__device__ __forceinline__ uint4 load_raw(const T *p) {
    const typename Chunk<T>::raw u = *reinterpret_cast<const typename Chunk<T>::raw *>(p);
    return make_uint4(u.x, u.y, u.z, u.w);
}
template <class T>
__device__ __forceinline__ void store_raw(T *p, const uint4 &v) {
    *reinterpret_cast<typename Chunk<T>::raw *>(p) = typename Chunk<T>::raw{v.x, v.y, v.z, v.w};
}
// The chunk at p of which the first `valid` values exist (any number, below one: none); zeros in place of the others.
template <class T>
__device__ __forceinline__ uint4 load_raw_part(const T *p, int valid) {
    constexpr int n = Chunk<T>::n;
    if (valid >= n) return load_raw(p);
    uint4 u = make_uint4(0, 0, 0, 0);
    if (valid > 0) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < n - 1; ++e)
            if (e < valid) {
                if constexpr (n == 4) w[e] = __float_as_uint(p[e]);
                else w[e / 2] |= (uint32_t)p[e] << (16 * (e & 1));
            }
        u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return u;
}
template <class T, int N>
__device__ __forceinline__ void load_part(const T *p, int valid, float (&v)[N]) {
    static_assert(N == Chunk<T>::n, "one chunk");
    const uint4 u = load_raw_part(p, valid);
    unpack(u, v);
}
template <class T, int N>
__device__ __forceinline__ void store_part(T *p, int valid, const float (&v)[N]) {
    static_assert(N == Chunk<T>::n, "one chunk");
    if (valid >= N) {
        store_raw(p, pack(v));
    } else {
#pragma unroll
        for (int e = 0; e < N - 1; ++e)
            if (e < valid) put(p + e, v[e]);
    }
}
// N values (a chunk's worth of another type) at p, of which `valid` exist
template <int N>
__device__ __forceinline__ void load_values(const float *p, int valid, float (&v)[N]) {
#pragma unroll
    for (int h = 0; h < N; h += 4) {
        float q[4];
        load_part(p + h, valid - h, q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[h + e] = q[e];
    }
}
template <int N>
__device__ __forceinline__ void load_values(const bf16_t *p, int valid, float (&v)[N]) {
    static_assert(N == 8, "a chunk of bfloat16");
    load_part(p, valid, v);
}

// Sum over G neighbouring lanes (a power of two up to 64), in every one of them.
template <int G>
__device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (G >= 2) v += dpp_row_move<0xB1>(v);    // quad_perm [1,0,3,2]
    if constexpr (G >= 4) v += dpp_row_move<0x4E>(v);    // quad_perm [2,3,0,1]
    if constexpr (G >= 8) v += dpp_row_move<0x141>(v);   // row_half_mirror
    if constexpr (G >= 16) v += dpp_row_move<0x140>(v);  // row_mirror
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}

// out_k[c] = sum over i of part[(i * K + k) * cols + c] for k < K: column sums that workgroups left in `parts` slabs, in a
// fixed order.  out[k] may be null.
static constexpr int kFoldMax = 2;
struct FoldOut { void *p[kFoldMax]; };
template <class T>
int launch_fold_columns(const float *part, int parts, int K, long cols, const FoldOut &out, hipStream_t s);

// layer normalisation (layer_norm.hip).  T: type of x, y and their gradients; W: of the weight, the bias and theirs.
static constexpr long kNormRegisterWidth = 16384;   // rows up to which a workgroup holds the whole row
template <class T, class W>
int launch_layer_norm_fwd(const T *x, long x_stride, const W *w, const W *b, T *y, float *mean, float *rstd, float eps, long rows,
                          int D, hipStream_t s);
template <class T, class W>
int launch_layer_norm_bwd(const T *dy, long dy_stride, const T *x, long x_stride, const W *w, const float *mean, const float *rstd,
                          T *gx, W *gw, W *gb, long rows, int D, float *part, hipStream_t s);
int layer_norm_bwd_parts(long rows, int D);   // slabs of 2 D floats that the backward's workspace holds

// the AdamW step (adamw.hip)
static constexpr int kAdamWBatchMax = ADDER_ADAMW_BATCH_MAX, kAdamW8BatchMax = ADDER_ADAMW_8BIT_BATCH_MAX;
static constexpr int kStateBlock = ADDER_STATE_BLOCK;
struct AdamWArgs {
    const float *lr_ptr, *corr;   // device: the rate; 1 / (1 - b1^t) and 1 / sqrt(1 - b2^t).  Null: the numbers below
    float lr, decay;              // decay: the factor 1 - lr * weight_decay
    float weight_decay, b1, b2, one_b1, one_b2, eps, c1, c2;
};
template <class T>
int launch_adamw(int count, void *const *p, const void *const *g, float *const *m, float *const *v, const long *n, const AdamWArgs &a,
                 hipStream_t s);
template <class T>
int launch_adamw_8bit(int count, void *const *p, const void *const *g, int8_t *const *m, uint8_t *const *v, float *const *ms,
                      float *const *vs, const long *n, const AdamWArgs &a, hipStream_t s);
int launch_adamw_advance(float *step, double ln_b1, double ln_b2, float *corr, hipStream_t s);
template <class T>
int launch_state_values(const void *codes, int is_signed, const float *scales, T *out, long n, hipStream_t s);

// linear layers (linear.hip)
enum class Act { none = ADDER_ACT_NONE, relu = ADDER_ACT_RELU, gelu = ADDER_ACT_GELU, silu = ADDER_ACT_SILU };
// out[m, n] = act(sum_k A(m, k) B(n, k) + bias[n]) + res[m, n].  An operand lies with k along its rows (its element (i, k) at
// i * ld + k) or across them (k * ld + i).  out and pre (nullable: the values before the activation) are dense.
struct Product {
    const void *a, *b;
    long lda, ldb;
    bool a_across, b_across;
    long M, N, K;
    const void *bias, *res;
    long ldr;
    void *out, *pre;
    Act act;
};
template <class T>
size_t product_workspace_bytes(long M, long N, long K);
template <class T>
int launch_product(const Product &p, void *ws, hipStream_t s);
template <class T>
int product_kernel(long M, long N, long K, bool a_across, bool b_across, bool aligned, int outputs);   // as adder_linear_kernel numbers them
// dz = dy * act'(z) (dense; not written where act is none) and part[i, n]: shares of its column sums (nullable)
template <class T>
int launch_act_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s);
int act_bwd_parts(long rows, long N);

}  // namespace adder
