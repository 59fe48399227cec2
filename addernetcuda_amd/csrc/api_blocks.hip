// C ABI of what gated blocks, their 8-bit form and their training from a teacher are made of: argument validation and dispatch.  As in
// api.hip, every check that can fail does so before the first HIP call.
#include "blocks.hpp"
#include "layer_checks.hpp"

namespace adder {

static size_t blocks_of(size_t n) { return (n + kCodeBlock - 1) / kCodeBlock; }
static bool known_types(int type, int weight_type) { return known(type) && known(weight_type); }

// the RMS norm's forward; scales: null where y are values
static int rms_norm(const void *x, long x_row_stride, const void *residual, long residual_row_stride, const void *weight, void *sum, void *y, float *scales,
                    float *save_rstd, float eps, long rows, int width, int type, int weight_type, void *stream) {
    if (rows <= 0 || width <= 0 || !known_types(type, weight_type) || !(eps >= 0.f) || bad_stride(x_row_stride, rows, width) ||
        (residual && bad_stride(residual_row_stride, rows, width)))
        return ADDER_ERR_BAD_SHAPE;
    if (type == ADDER_TYPE_F32 && weight_type != type) return ADDER_ERR_UNSUPPORTED;
    if (width > kMaxWidth || wide(rows, width) || wide(rows, x_row_stride) || (residual && wide(rows, residual_row_stride))) return ADDER_ERR_TOO_LARGE;
    const size_t n = (size_t)rows * width, e = size_of(type);
    const Span outs[] = {{sum, e * n}, {y, scales ? n : e * n}, {scales, sizeof(float) * rows * blocks_of(width)}, {save_rstd, sizeof(float) * (size_t)rows}};
    const Span ins[] = {{x, span(rows, x_row_stride, width, type)}, {residual, span(rows, residual_row_stride, width, type)},
                        {weight, size_of(weight_type) * (size_t)width}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const RmsRows p{x, residual, weight, x_row_stride, residual_row_stride, sum, y, scales, save_rstd, eps, rows, width};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == ADDER_TYPE_F32) return launch_rms_norm_fwd<float, float>(p, s);
    return weight_type == ADDER_TYPE_F32 ? launch_rms_norm_fwd<bf16_t, float>(p, s) : launch_rms_norm_fwd<bf16_t, bf16_t>(p, s);
}

static size_t codes_bytes(long rows, int in, int out, int type, bool x_aligned, bool w_aligned) {
    return type == ADDER_TYPE_BF16 ? codes_product_workspace_bytes<bf16_t>(rows, out, in, x_aligned, w_aligned)
                                   : codes_product_workspace_bytes<float>(rows, out, in, x_aligned, w_aligned);
}

static int check_gated(long rows, int in, int hidden, int type) {
    if (rows <= 0 || in <= 0 || hidden <= 0 || !known(type)) return ADDER_ERR_BAD_SHAPE;
    if (hidden > kMaxWidth / 2 - 16) return ADDER_ERR_TOO_LARGE;
    return check_linear(rows, in, (int)gated_columns(hidden), type);
}
static Product gated_product(const void *x, long ldx, const void *w, const void *bias, void *y, void *pre, int act, long rows, int in, int hidden) {
    Product p{x, w, ldx, in, false, false, rows, gated_columns(hidden), in, bias, nullptr, 0, y, pre, static_cast<Act>(act)};
    p.half = hidden;
    return p;
}
// The backward's workspace: dz, the column sums' shares, and what the products need
struct GatedBwdSpace { size_t dz, part, product; };
static GatedBwdSpace gated_bwd_space(long rows, int in, int hidden, int type) {
    const size_t gx = product_bytes(rows, in, 2L * hidden, type), gw = product_bytes(2L * hidden, in, rows, type);
    return {whole(size_of(type) * (size_t)rows * 2 * hidden), whole(sizeof(float) * (size_t)gated_bwd_parts(rows, hidden) * 2 * hidden), whole(gx > gw ? gx : gw)};
}

static int check_distill(long rows, int classes, int K, int type, int top_type, long stride, float temperature, float alpha) {
    if (rows <= 0 || classes <= 0 || K <= 0 || !known_types(type, top_type) || bad_stride(stride, rows, classes)) return ADDER_ERR_BAD_SHAPE;
    if (!(temperature > 0.f && temperature <= 3e38f) || !(alpha >= 0.f && alpha <= 1.f)) return ADDER_ERR_BAD_SHAPE;
    if (K > ADDER_DISTILL_TOP_MAX) return ADDER_ERR_UNSUPPORTED;
    return classes > kMaxWidth || wide(rows, classes) || wide(rows, stride) ? ADDER_ERR_TOO_LARGE : ADDER_OK;
}

}  // namespace adder

using namespace adder;

extern "C" {

int adder_rms_norm_fwd(const void *x, long x_row_stride, const void *residual, long residual_row_stride, const void *weight, void *sum, void *y,
                       float *save_rstd, float eps, long rows, int width, int type, int weight_type, void *stream) {
    if (!x || !y) return ADDER_ERR_NULL_POINTER;
    return rms_norm(x, x_row_stride, residual, residual_row_stride, weight, sum, y, nullptr, save_rstd, eps, rows, width, type, weight_type, stream);
}

int adder_rms_norm_fwd_codes(const void *x, long x_row_stride, const void *residual, long residual_row_stride, const void *weight, void *sum,
                             unsigned char *codes, float *scales, float eps, long rows, int width, int type, int weight_type, void *stream) {
    if (!x || !codes || !scales) return ADDER_ERR_NULL_POINTER;
    return rms_norm(x, x_row_stride, residual, residual_row_stride, weight, sum, codes, scales, nullptr, eps, rows, width, type, weight_type, stream);
}

int adder_rms_norm_bwd_workspace_bytes(long rows, int width, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type)) return ADDER_ERR_BAD_SHAPE;
    if (width > kMaxWidth || wide(rows, width)) return ADDER_ERR_TOO_LARGE;
    *bytes = whole(sizeof(float) * (size_t)rms_norm_bwd_parts(rows, width) * width);
    return ADDER_OK;
}

int adder_rms_norm_bwd(const void *dy, long dy_row_stride, const void *dsum, long dsum_row_stride, const void *x, long x_row_stride, const void *weight,
                       const float *save_rstd, void *gx, void *gweight, long rows, int width, int type, int weight_type, void *ws, size_t ws_bytes,
                       void *stream) {
    if (!dy || !x || !save_rstd || (!gx && !gweight)) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known_types(type, weight_type) || bad_stride(x_row_stride, rows, width) || bad_stride(dy_row_stride, rows, width) ||
        (dsum && bad_stride(dsum_row_stride, rows, width)))
        return ADDER_ERR_BAD_SHAPE;
    if (type == ADDER_TYPE_F32 && weight_type != type) return ADDER_ERR_UNSUPPORTED;
    if (width > kMaxWidth || wide(rows, width) || wide(rows, x_row_stride) || wide(rows, dy_row_stride) || (dsum && wide(rows, dsum_row_stride)))
        return ADDER_ERR_TOO_LARGE;
    size_t need = 0;
    if (int rc = adder_rms_norm_bwd_workspace_bytes(rows, width, type, &need)) return rc;
    if (!gweight) need = 0;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const size_t nw = size_of(weight_type) * (size_t)width;
    const Span outs[] = {{gx, size_of(type) * (size_t)rows * width}, {gweight, nw}, {ws, need}};
    const Span ins[] = {{dy, span(rows, dy_row_stride, width, type)}, {dsum, span(rows, dsum_row_stride, width, type)},
                        {x, span(rows, x_row_stride, width, type)}, {weight, nw}, {save_rstd, sizeof(float) * (size_t)rows}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float *part = static_cast<float *>(ws);
#define ADDER_RMS_BWD(T, W)                                                                                                                          \
    launch_rms_norm_bwd(static_cast<const T *>(dy), dy_row_stride, static_cast<const T *>(dsum), dsum_row_stride, static_cast<const T *>(x),         \
                        x_row_stride, static_cast<const W *>(weight), save_rstd, static_cast<T *>(gx), static_cast<W *>(gweight), rows, width, part, s)
    if (type == ADDER_TYPE_F32) return ADDER_RMS_BWD(float, float);
    return weight_type == ADDER_TYPE_F32 ? ADDER_RMS_BWD(bf16_t, float) : ADDER_RMS_BWD(bf16_t, bf16_t);
#undef ADDER_RMS_BWD
}

int adder_quantize(const void *x, long x_row_stride, int act, unsigned char *codes, float *scales, long rows, int width, int type, void *stream) {
    if (!x || !codes || !scales) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type) || (act >= 0 && !known_act(act))) return ADDER_ERR_BAD_SHAPE;
    const long in = act >= 0 ? 2L * width : width;
    if (bad_stride(x_row_stride, rows, in)) return ADDER_ERR_BAD_SHAPE;
    if (in > kMaxWidth || wide(rows, in) || wide(rows, x_row_stride)) return ADDER_ERR_TOO_LARGE;
    const Span outs[] = {{codes, (size_t)rows * width}, {scales, sizeof(float) * rows * blocks_of(width)}};
    const Span ins[] = {{x, span(rows, x_row_stride, in, type)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const Act a = act >= 0 ? static_cast<Act>(act) : Act::none;
    return type == ADDER_TYPE_BF16 ? launch_quantize(static_cast<const bf16_t *>(x), x_row_stride, act >= 0, a, codes, scales, rows, width, s)
                                   : launch_quantize(static_cast<const float *>(x), x_row_stride, act >= 0, a, codes, scales, rows, width, s);
}

int adder_quantize_weight(const void *w, long w_row_stride, unsigned char *codes, float *scales, long rows, int width, int type, void *stream) {
    if (!w || !codes || !scales) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type) || bad_stride(w_row_stride, rows, width)) return ADDER_ERR_BAD_SHAPE;
    if (width > kMaxWidth || rows > kCodeBlock * 65535L || wide(rows, w_row_stride)) return ADDER_ERR_TOO_LARGE;   // (a launch's rows of workgroups)
    const Span outs[] = {{codes, (size_t)rows * width}, {scales, sizeof(float) * blocks_of(rows) * blocks_of(width)}};
    const Span ins[] = {{w, span(rows, w_row_stride, width, type)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_quantize_weight(static_cast<const bf16_t *>(w), w_row_stride, codes, scales, rows, width, s)
                                   : launch_quantize_weight(static_cast<const float *>(w), w_row_stride, codes, scales, rows, width, s);
}

int adder_linear_codes_workspace_bytes(long rows, int in_features, int out_features, int type, int x_aligned, int w_aligned, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    *bytes = whole(codes_bytes(rows, in_features, out_features, type, x_aligned != 0, w_aligned != 0));
    return ADDER_OK;
}

int adder_linear_codes(const unsigned char *x, long x_row_stride, const float *x_scales, const unsigned char *w, long w_row_stride, const float *w_scales,
                       const void *bias, const void *residual, long residual_row_stride, void *y, int act, long rows, int in_features, int out_features,
                       int type, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !x_scales || !w || !w_scales || !y) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    if (!known_act(act) || bad_stride(x_row_stride, rows, in_features) || bad_stride(w_row_stride, out_features, in_features) ||
        (residual && bad_stride(residual_row_stride, rows, out_features)))
        return ADDER_ERR_BAD_SHAPE;
    // (a tile's rows lie within 2^32 bytes of each other)
    if (wide(rows, x_row_stride) || wide(out_features, w_row_stride) || x_row_stride >= ADDER_CODES_STRIDE_MAX ||
        w_row_stride >= ADDER_CODES_STRIDE_MAX || in_features >= ADDER_CODES_STRIDE_MAX || (residual && wide(rows, residual_row_stride)))
        return ADDER_ERR_TOO_LARGE;
    const auto aligned = [](const void *p, long ld) { return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)ld) & 15); };
    const size_t need = codes_bytes(rows, in_features, out_features, type, aligned(x, x_row_stride), aligned(w, w_row_stride));
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const size_t blocks = blocks_of(in_features), e = size_of(type);
    const Span outs[] = {{y, e * (size_t)rows * out_features}, {ws, need}};
    const Span ins[] = {{x, (size_t)(rows - 1) * (rows > 1 ? x_row_stride : 0) + in_features}, {x_scales, sizeof(float) * rows * blocks},
                        {w, (size_t)(out_features - 1) * (out_features > 1 ? w_row_stride : 0) + in_features}, {w_scales, sizeof(float) * blocks_of(out_features) * blocks},
                        {bias, e * (size_t)out_features}, {residual, span(rows, residual_row_stride, out_features, type)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const CodesProduct p{x, w, x_scales, w_scales, x_row_stride, w_row_stride, rows, out_features, in_features, bias, residual, residual_row_stride, y,
                         static_cast<Act>(act)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_codes_product<bf16_t>(p, ws, s) : launch_codes_product<float>(p, ws, s);
}

int adder_linear_codes_kernel(long rows, int in_features, int out_features, int type, int *kernel) {
    if (!kernel) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    *kernel = type == ADDER_TYPE_BF16 ? codes_product_kernel<bf16_t>(rows, out_features, in_features) : codes_product_kernel<float>(rows, out_features, in_features);
    return ADDER_OK;
}

int adder_gated_fwd_workspace_bytes(long rows, int in_features, int hidden, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_gated(rows, in_features, hidden, type)) return rc;
    *bytes = whole(product_bytes(rows, gated_columns(hidden), in_features, type, true));
    return ADDER_OK;
}

int adder_gated_fwd(const void *x, long x_row_stride, const void *w, const void *bias, void *y, void *pre, int act, long rows, int in_features, int hidden,
                    int type, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !w || !y) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_gated(rows, in_features, hidden, type)) return rc;
    if (!known_act(act) || bad_stride(x_row_stride, rows, in_features)) return ADDER_ERR_BAD_SHAPE;
    if (wide(rows, x_row_stride)) return ADDER_ERR_TOO_LARGE;
    const size_t need = product_bytes(rows, gated_columns(hidden), in_features, type, true), e = size_of(type), ny = e * (size_t)rows * hidden;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const Span outs[] = {{y, ny}, {pre, 2 * ny}, {ws, need}};
    const Span ins[] = {{x, span(rows, x_row_stride, in_features, type)}, {w, e * 2 * (size_t)hidden * in_features}, {bias, e * 2 * (size_t)hidden}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    return product(gated_product(x, x_row_stride, w, bias, y, pre, act, rows, in_features, hidden), type, ws, static_cast<hipStream_t>(stream));
}

int adder_gated_bwd_workspace_bytes(long rows, int in_features, int hidden, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_gated(rows, in_features, hidden, type)) return rc;
    const GatedBwdSpace n = gated_bwd_space(rows, in_features, hidden, type);
    *bytes = n.dz + n.part + n.product;
    return ADDER_OK;
}

int adder_gated_bwd(const void *dy, long dy_row_stride, const void *pre, const void *x, long x_row_stride, const void *w, void *gx, void *gw, void *gbias,
                    int act, long rows, int in_features, int hidden, int type, void *ws, size_t ws_bytes, void *stream) {
    if (!dy || !pre || (!gx && !gw && !gbias) || (gw && !x) || (gx && !w)) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_gated(rows, in_features, hidden, type)) return rc;
    if (!known_act(act) || bad_stride(dy_row_stride, rows, hidden) || (gw && bad_stride(x_row_stride, rows, in_features))) return ADDER_ERR_BAD_SHAPE;
    if (wide(rows, dy_row_stride) || (gw && wide(rows, x_row_stride))) return ADDER_ERR_TOO_LARGE;
    const GatedBwdSpace n = gated_bwd_space(rows, in_features, hidden, type);
    const size_t need = n.dz + n.part + n.product, e = size_of(type), nw = e * 2 * (size_t)hidden * in_features;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const Span outs[] = {{gx, e * (size_t)rows * in_features}, {gw, nw}, {gbias, e * 2 * (size_t)hidden}, {ws, need}};
    const Span ins[] = {{dy, span(rows, dy_row_stride, hidden, type)}, {pre, e * 2 * (size_t)rows * hidden},
                        {gw ? x : nullptr, span(rows, x_row_stride, in_features, type)}, {gx ? w : nullptr, nw}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    char *at = static_cast<char *>(ws);
    void *dz = gx || gw ? at : nullptr, *rest = at + n.dz + n.part;
    float *part = gbias ? reinterpret_cast<float *>(at + n.dz) : nullptr;
    const Act a = static_cast<Act>(act);
    if (int rc = type == ADDER_TYPE_BF16 ? launch_gated_bwd(static_cast<const bf16_t *>(dy), dy_row_stride, static_cast<const bf16_t *>(pre),
                                                            static_cast<bf16_t *>(dz), part, a, rows, hidden, s)
                                         : launch_gated_bwd(static_cast<const float *>(dy), dy_row_stride, static_cast<const float *>(pre),
                                                            static_cast<float *>(dz), part, a, rows, hidden, s))
        return rc;
    const long both = 2L * hidden;
    if (gbias) {
        const int parts = gated_bwd_parts(rows, hidden);
        const FoldOut out{{gbias, nullptr}};
        if (int rc = type == ADDER_TYPE_BF16 ? launch_fold_columns<bf16_t>(part, parts, 1, both, out, s) : launch_fold_columns<float>(part, parts, 1, both, out, s))
            return rc;
    }
    if (gx) {
        const Product p{dz, w, both, in_features, false, true, rows, in_features, both, nullptr, nullptr, 0, gx, nullptr, Act::none};
        if (int rc = product(p, type, rest, s)) return rc;
    }
    if (gw) {
        const Product p{dz, x, both, x_row_stride, true, true, both, in_features, rows, nullptr, nullptr, 0, gw, nullptr, Act::none};
        if (int rc = product(p, type, rest, s)) return rc;
    }
    return ADDER_OK;
}

int adder_gated_kernel(long rows, int in_features, int hidden, int type, int aligned, int outputs, int *kernel) {
    if (!kernel) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_gated(rows, in_features, hidden, type)) return rc;
    if (outputs < 1 || outputs > 2) return ADDER_ERR_BAD_SHAPE;
    const auto of = type == ADDER_TYPE_BF16 ? product_kernel<bf16_t> : product_kernel<float>;
    *kernel = of(rows, gated_columns(hidden), in_features, false, false, aligned != 0, outputs, true);
    return ADDER_OK;
}

int adder_distill_in_rows(long rows, int classes, int type) { return rows > 0 && classes > 0 && known(type) && distill_in_rows(rows, classes, type); }

int adder_distill_workspace_bytes(long rows, int classes, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_distill(rows, classes, 1, type, type, classes, 1.f, 1.f)) return rc;
    *bytes = whole(distill_workspace_bytes(rows, classes, type));
    return ADDER_OK;
}

int adder_distill_fwd(const void *logits, long logits_row_stride, const void *top, const long long *classes_of_top, const long long *labels, float *loss,
                      float *stats, void *grad, float temperature, float alpha, long long ignore, long rows, int classes, int K, int type, int top_type,
                      void *ws, size_t ws_bytes, void *stream) {
    if (!logits || !top || !classes_of_top || !loss || !stats) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_distill(rows, classes, K, type, top_type, logits_row_stride, temperature, alpha)) return rc;
    if (grad && !distill_in_rows(rows, classes, type)) return ADDER_ERR_UNSUPPORTED;
    const size_t need = distill_workspace_bytes(rows, classes, type);
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const Span outs[] = {{loss, sizeof(float)}, {stats, sizeof(float) * kDistillStats * (size_t)(rows + 1)}, {grad, size_of(type) * (size_t)rows * classes}, {ws, need}};
    const Span ins[] = {{logits, span(rows, logits_row_stride, classes, type)}, {top, size_of(top_type) * (size_t)rows * K},
                        {classes_of_top, sizeof(long long) * (size_t)rows * K}, {labels, sizeof(long long) * (size_t)rows}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const DistillArgs a{logits, top, classes_of_top, labels, logits_row_stride, loss, stats, grad, nullptr, temperature, alpha, ignore, rows, classes, K,
                        top_type == ADDER_TYPE_BF16, false};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_distill_fwd<bf16_t>(a, ws, s) : launch_distill_fwd<float>(a, ws, s);
}

int adder_distill_bwd(const void *logits, long logits_row_stride, const void *top, const long long *classes_of_top, const long long *labels,
                      const float *stats, const float *grad_loss, int unit, void *grad, float temperature, float alpha, long long ignore, long rows,
                      int classes, int K, int type, int top_type, void *stream) {
    if (!logits || !top || !classes_of_top || !stats || !grad_loss || !grad) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_distill(rows, classes, K, type, top_type, logits_row_stride, temperature, alpha)) return rc;
    const Span outs[] = {{grad, size_of(type) * (size_t)rows * classes}};
    const Span ins[] = {{logits, span(rows, logits_row_stride, classes, type)}, {top, size_of(top_type) * (size_t)rows * K},
                        {classes_of_top, sizeof(long long) * (size_t)rows * K}, {labels, sizeof(long long) * (size_t)rows},
                        {stats, sizeof(float) * kDistillStats * (size_t)(rows + 1)}, {grad_loss, sizeof(float)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const DistillArgs a{logits, top, classes_of_top, labels, logits_row_stride, nullptr, const_cast<float *>(stats), grad, grad_loss, temperature, alpha,
                        ignore, rows, classes, K, top_type == ADDER_TYPE_BF16, unit != 0};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_distill_bwd<bf16_t>(a, s) : launch_distill_bwd<float>(a, s);
}

}  // extern "C"
