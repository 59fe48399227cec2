// What a gated block, its 8-bit form and its training from a teacher are made of: the RMS norm (rms_norm.hip), e4m3 codes with block scales
// (fp8.hip) and their products (fp8_product.hip), the gated linear layer's backward (gated.hip), the loss against a teacher's top logits
// (distill.hip).
#pragma once
#include "product.hpp"

namespace adder {

// ---- e4m3 codes --------------------------------------------------------------------------------------------------------
// kCodeBlock neighbouring values share a scale: the largest magnitude among them (at least kCodeLeast) becomes 448, the largest code.
static constexpr int kCodeBlock = ADDER_CODE_BLOCK;
static constexpr float kCodeTop = 448.f, kCodeLeast = 0x1p-100f;
// four floats to nearest even (v_cvt_pk_fp8_f32); magnitudes up to 448 and what rounding adds to them
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
    return (uint32_t)u;
}
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint32_t u32x2_any1 __attribute__((ext_vector_type(2), aligned(1)));
__device__ __forceinline__ void store_codes(uint8_t *p, int valid, const float (&v)[4]) {
    const uint32_t u = pack_codes(v[0], v[1], v[2], v[3]);
    if (valid >= 4) {
        *reinterpret_cast<u32_any *>(p) = u;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < valid) p[e] = (uint8_t)(u >> (8 * e));
    }
}
__device__ __forceinline__ void store_codes(uint8_t *p, int valid, const float (&v)[8]) {
    const uint32_t lo = pack_codes(v[0], v[1], v[2], v[3]), hi = pack_codes(v[4], v[5], v[6], v[7]);
    if (valid >= 8) {
        *reinterpret_cast<u32x2_any1 *>(p) = u32x2_any1{lo, hi};
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < valid) p[e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
    }
}
// Largest over G neighbouring lanes, in every one of them
template <int G>
__device__ __forceinline__ float lanes_max(float v) {
    if constexpr (G >= 2) v = fmaxf(v, dpp_row_move<0xB1>(v));
    if constexpr (G >= 4) v = fmaxf(v, dpp_row_move<0x4E>(v));
    if constexpr (G >= 8) v = fmaxf(v, dpp_row_move<0x141>(v));
    if constexpr (G >= 16) v = fmaxf(v, dpp_row_move<0x140>(v));
    if constexpr (G >= 32) v = fmaxf(v, __shfl_xor(v, 16, 64));
    if constexpr (G >= 64) v = fmaxf(v, __shfl_xor(v, 32, 64));
    return v;
}

// ---- RMS norm (rms_norm.hip) ---------------------------------------------------------------------------------------------
struct RmsRows {   // of a call: s = x + r, y = s rstd w
    const void *x, *r, *w;
    long x_stride, r_stride;
    void *sum, *y;       // sum: nullable; y: values, or codes
    float *scale;        // of the codes; null: y are values
    float *rstd;         // nullable
    float eps;
    long rows;
    int D;
};
template <class T, class W>
int launch_rms_norm_fwd(const RmsRows &p, hipStream_t s);
template <class T, class W>
int launch_rms_norm_bwd(const T *dy, long dy_stride, const T *ds, long ds_stride, const T *x, long x_stride, const W *w, const float *rstd, T *gx,
                        W *gw, long rows, int D, float *part, hipStream_t s);
int rms_norm_bwd_parts(long rows, int D);   // slabs of D floats that the backward's workspace holds

// ---- codes (fp8.hip) and their products (fp8_product.hip) ---------------------------------------------------------------
// act: of a gated input (rows of 2 D values), else none and not gated
template <class T>
int launch_quantize(const T *x, long x_stride, bool gated, Act act, uint8_t *q, float *scale, long rows, int D, hipStream_t s);
template <class T>
int launch_quantize_weight(const T *w, long w_stride, uint8_t *q, float *scale, long rows, int D, hipStream_t s);
struct CodesProduct {
    const uint8_t *x, *w;
    const float *xs, *ws;
    long ldx, ldw;
    long M, N, K;
    const void *bias, *res;
    long ldr;
    void *out;
    Act act;
};
// T: type of the result
template <class T>
int codes_product_kernel(long M, long N, long K);   // as adder_linear_codes_kernel numbers them
template <class T>
size_t codes_product_workspace_bytes(long M, long N, long K, bool x_aligned, bool w_aligned);
template <class T>
int launch_codes_product(const CodesProduct &p, void *ws, hipStream_t s);

// ---- gated linear layer's backward (gated.hip) ---------------------------------------------------------------------------
// z: what the forward kept, rows of 2 N values; dz likewise (dense), part: shares of its column sums (nullable)
template <class T>
int launch_gated_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s);
int gated_bwd_parts(long rows, long N);

// ---- loss against a teacher (distill.hip) -----------------------------------------------------------------------------------
struct DistillArgs {
    const void *logits, *top;
    const long long *idx, *target;   // target: nullable
    long stride;                     // of the logits' rows
    float *loss, *stats;             // stats: kDistillStats floats a row, and as many behind the last
    void *grad;                      // nullable
    const float *grad_loss;          // the backward's
    float temperature, alpha;
    long long ignore;
    long rows;
    int classes, K;
    bool top_bf16, unit;             // unit: grad already holds the gradient for a grad_loss of one
};
static constexpr int kDistillStats = 8;
bool distill_in_rows(long rows, int classes, int type);   // whether the forward keeps a row in registers, and can write the gradient
size_t distill_workspace_bytes(long rows, int classes, int type);
template <class T>
int launch_distill_fwd(const DistillArgs &a, void *ws, hipStream_t s);
template <class T>
int launch_distill_bwd(const DistillArgs &a, hipStream_t s);

}  // namespace adder
