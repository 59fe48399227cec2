// C ABI of the layers beside the adder layers: argument validation and dispatch.  As in api.hip, every check that can fail
// does so before the first HIP call.
#include "checks.hpp"
#include "layers.hpp"

#include <math.h>

namespace adder {

static const long kMaxElems = 0x7fffffffL;          // of a tensor that one kernel index of 32 bits walks over
static const double kMaxWide = 1099511627776.0;     // of the others: 2^40
static const int kMaxWidth = 1 << 26;               // of a row: the folds of columns are launches of 32 threads a column

static bool known(int type) { return type == ADDER_TYPE_F32 || type == ADDER_TYPE_BF16; }
static size_t size_of(int type) { return type == ADDER_TYPE_BF16 ? 2 : 4; }
static bool bad_stride(long stride, long rows, long width) { return rows > 1 && stride != 0 && stride < width; }
static size_t span(long rows, long stride, long width, int type) { return size_of(type) * ((size_t)(rows - 1) * (rows > 1 ? stride : 0) + width); }
static bool wide(double rows, double stride) { return rows * stride > kMaxWide; }
static size_t whole(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

static int check_workspace(const void *ws, size_t have, size_t need) {
    if (!need) return ADDER_OK;
    return !ws || (reinterpret_cast<uintptr_t>(ws) & 255) || have < need ? ADDER_ERR_WORKSPACE : ADDER_OK;
}

static int check_linear(long rows, int in, int out, int type) {
    if (rows <= 0 || in <= 0 || out <= 0 || !known(type)) return ADDER_ERR_BAD_SHAPE;
    if (wide(rows, in) || wide(rows, out) || wide(in, out) || in > kMaxWidth || out > kMaxWidth) return ADDER_ERR_TOO_LARGE;
    // (workgroups of 256 threads and at least 64 x 64 results; a launch has at most 2^32 threads)
    const double r = rows / 64 + 1, i = in / 64 + 1, o = out / 64 + 1, most = 16777216.0;
    return r * o > most || r * i > most || i * o > most ? ADDER_ERR_TOO_LARGE : ADDER_OK;
}
static bool known_act(int act) { return act >= ADDER_ACT_NONE && act <= ADDER_ACT_SILU; }

static size_t product_bytes(long M, long N, long K, int type) {
    return type == ADDER_TYPE_BF16 ? product_workspace_bytes<bf16_t>(M, N, K) : product_workspace_bytes<float>(M, N, K);
}
static int product(const Product &p, int type, void *ws, hipStream_t s) {
    return type == ADDER_TYPE_BF16 ? launch_product<bf16_t>(p, ws, s) : launch_product<float>(p, ws, s);
}

// The backward's workspace: dz where it is not dy, the column sums' shares, and what the products need
struct LinearBwdSpace { size_t dz, part, product; };
static LinearBwdSpace linear_bwd_space(long rows, int in, int out, int act, int type) {
    const size_t gx = product_bytes(rows, in, out, type), gw = product_bytes(out, in, rows, type);
    return {act == ADDER_ACT_NONE ? 0 : whole(size_of(type) * (size_t)rows * out), whole(sizeof(float) * (size_t)act_bwd_parts(rows, out) * out),
            whole(gx > gw ? gx : gw)};
}

static int adamw_args(AdamWArgs &a, const float *lr_device, double lr, double beta1, double beta2, double eps, double weight_decay, long step,
                      const float *corrections) {
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(weight_decay >= 0.0) || !(lr_device || lr >= 0.0))
        return ADDER_ERR_BAD_SHAPE;
    if (!corrections && step < 1) return ADDER_ERR_BAD_SHAPE;
    a.lr_ptr = lr_device;
    a.corr = corrections;
    a.lr = (float)lr;
    a.decay = (float)(1.0 - lr * weight_decay);
    a.weight_decay = (float)weight_decay;
    a.b1 = (float)beta1; a.b2 = (float)beta2; a.one_b1 = (float)(1.0 - beta1); a.one_b2 = (float)(1.0 - beta2);
    a.eps = (float)eps;
    a.c1 = corrections ? 0.f : (float)(1.0 / (1.0 - pow(beta1, (double)step)));
    a.c2 = corrections ? 0.f : (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    return ADDER_OK;
}

static int check_counts(int count, int most, const long *n) {
    if (count <= 0 || count > most) return ADDER_ERR_BAD_SHAPE;
    long blocks = 0;
    for (int t = 0; t < count; ++t) {
        if (n[t] <= 0) return ADDER_ERR_BAD_SHAPE;
        if (n[t] > kMaxElems) return ADDER_ERR_TOO_LARGE;
        blocks += (n[t] + 1023) / 1024;
    }
    return blocks > 16777215 ? ADDER_ERR_TOO_LARGE : ADDER_OK;   // (of 256 threads: a launch has at most 2^32)
}

}  // namespace adder

using namespace adder;

extern "C" {

int adder_linear_fwd_workspace_bytes(long rows, int in_features, int out_features, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    *bytes = whole(product_bytes(rows, out_features, in_features, type));
    return ADDER_OK;
}

int adder_linear_fwd(const void *x, long x_row_stride, const void *w, const void *bias, const void *residual, long residual_row_stride, void *y,
                     void *pre, int act, long rows, int in_features, int out_features, int type, void *ws, size_t ws_bytes, void *stream) {
    if (!x || !w || !y) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    if (!known_act(act) || bad_stride(x_row_stride, rows, in_features) || (residual && bad_stride(residual_row_stride, rows, out_features)))
        return ADDER_ERR_BAD_SHAPE;
    if (wide(rows, x_row_stride) || (residual && wide(rows, residual_row_stride))) return ADDER_ERR_TOO_LARGE;
    const size_t need = product_bytes(rows, out_features, in_features, type), ny = size_of(type) * (size_t)rows * out_features;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const Span outs[] = {{y, ny}, {pre, ny}, {ws, need}};
    const Span ins[] = {{x, span(rows, x_row_stride, in_features, type)}, {w, size_of(type) * (size_t)out_features * in_features},
                        {bias, size_of(type) * (size_t)out_features}, {residual, span(rows, residual_row_stride, out_features, type)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const Product p{x, w, x_row_stride, in_features, false, false, rows, out_features, in_features, bias, residual, residual_row_stride, y, pre,
                    static_cast<Act>(act)};
    return product(p, type, ws, static_cast<hipStream_t>(stream));
}

int adder_linear_bwd_workspace_bytes(long rows, int in_features, int out_features, int act, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    if (!known_act(act)) return ADDER_ERR_BAD_SHAPE;
    const LinearBwdSpace n = linear_bwd_space(rows, in_features, out_features, act, type);
    *bytes = n.dz + n.part + n.product;
    return ADDER_OK;
}

int adder_linear_bwd(const void *dy, long dy_row_stride, const void *pre, const void *x, long x_row_stride, const void *w, void *gx, void *gw,
                     void *gbias, int act, long rows, int in_features, int out_features, int type, void *ws, size_t ws_bytes, void *stream) {
    if (!dy || (!gx && !gw && !gbias) || (gw && !x) || (gx && !w)) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    if (!known_act(act) || bad_stride(dy_row_stride, rows, out_features) || (gw && bad_stride(x_row_stride, rows, in_features)))
        return ADDER_ERR_BAD_SHAPE;
    if (act != ADDER_ACT_NONE && !pre) return ADDER_ERR_NULL_POINTER;
    if (wide(rows, dy_row_stride) || wide(rows, x_row_stride)) return ADDER_ERR_TOO_LARGE;
    const LinearBwdSpace n = linear_bwd_space(rows, in_features, out_features, act, type);
    const size_t need = n.dz + n.part + n.product, e = size_of(type), nw = e * (size_t)out_features * in_features;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const Span outs[] = {{gx, e * (size_t)rows * in_features}, {gw, nw}, {gbias, e * (size_t)out_features}, {ws, need}};
    const Span ins[] = {{dy, span(rows, dy_row_stride, out_features, type)}, {act == ADDER_ACT_NONE ? nullptr : pre, e * (size_t)rows * out_features},
                        {gw ? x : nullptr, span(rows, x_row_stride, in_features, type)}, {gx ? w : nullptr, nw}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const Act a = static_cast<Act>(act);
    char *at = static_cast<char *>(ws);
    void *dz = n.dz && (gx || gw) ? at : nullptr;
    float *part = gbias ? reinterpret_cast<float *>(at + n.dz) : nullptr;
    void *rest = at + n.dz + n.part;
    if (a != Act::none || gbias) {
        const int rc = type == ADDER_TYPE_BF16 ? launch_act_bwd<bf16_t>(static_cast<const bf16_t *>(dy), dy_row_stride, static_cast<const bf16_t *>(pre),
                                                                        static_cast<bf16_t *>(dz), part, a, rows, out_features, s)
                                               : launch_act_bwd<float>(static_cast<const float *>(dy), dy_row_stride, static_cast<const float *>(pre),
                                                                       static_cast<float *>(dz), part, a, rows, out_features, s);
        if (rc) return rc;
    }
    if (gbias) {
        const int parts = act_bwd_parts(rows, out_features);
        const FoldOut out{{gbias, nullptr}};
        if (int rc = type == ADDER_TYPE_BF16 ? launch_fold_columns<bf16_t>(part, parts, 1, out_features, out, s)
                                             : launch_fold_columns<float>(part, parts, 1, out_features, out, s))
            return rc;
    }
    const void *d = dz ? dz : dy;
    const long ldd = dz ? out_features : dy_row_stride;
    if (gx) {
        const Product p{d, w, ldd, in_features, false, true, rows, in_features, out_features, nullptr, nullptr, 0, gx, nullptr, Act::none};
        if (int rc = product(p, type, rest, s)) return rc;
    }
    if (gw) {
        const Product p{d, x, ldd, x_row_stride, true, true, out_features, in_features, rows, nullptr, nullptr, 0, gw, nullptr, Act::none};
        if (int rc = product(p, type, rest, s)) return rc;
    }
    return ADDER_OK;
}

int adder_linear_kernel(long rows, int in_features, int out_features, int product, int type, int aligned, int outputs, int *kernel) {
    if (!kernel) return ADDER_ERR_NULL_POINTER;
    if (int rc = check_linear(rows, in_features, out_features, type)) return rc;
    if (product < 0 || product > 2 || outputs < 1 || outputs > (product ? 1 : 2)) return ADDER_ERR_BAD_SHAPE;
    const long M = product == 2 ? out_features : rows, N = product ? in_features : out_features, K = product == 0 ? in_features : product == 1 ? out_features : rows;
    const auto of = type == ADDER_TYPE_BF16 ? product_kernel<bf16_t> : product_kernel<float>;
    *kernel = of(M, N, K, product == 2, product != 0, aligned != 0, outputs);
    return ADDER_OK;
}

int adder_layer_norm_fwd(const void *x, long x_row_stride, const void *weight, const void *bias, void *y, float *save_mean, float *save_rstd,
                         float eps, long rows, int width, int type, int weight_type, void *stream) {
    if (!x || !y || (save_mean == nullptr) != (save_rstd == nullptr)) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type) || !known(weight_type) || !(eps >= 0.f) || bad_stride(x_row_stride, rows, width))
        return ADDER_ERR_BAD_SHAPE;
    if (type == ADDER_TYPE_F32 && weight_type != type) return ADDER_ERR_UNSUPPORTED;
    if (width > kMaxWidth || wide(rows, width) || wide(rows, x_row_stride)) return ADDER_ERR_TOO_LARGE;
    const size_t nw = size_of(weight_type) * (size_t)width, nr = sizeof(float) * (size_t)rows;
    const Span outs[] = {{y, size_of(type) * (size_t)rows * width}, {save_mean, nr}, {save_rstd, nr}};
    const Span ins[] = {{x, span(rows, x_row_stride, width, type)}, {weight, nw}, {bias, nw}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == ADDER_TYPE_F32)
        return launch_layer_norm_fwd(static_cast<const float *>(x), x_row_stride, static_cast<const float *>(weight), static_cast<const float *>(bias),
                                     static_cast<float *>(y), save_mean, save_rstd, eps, rows, width, s);
    if (weight_type == ADDER_TYPE_F32)
        return launch_layer_norm_fwd(static_cast<const bf16_t *>(x), x_row_stride, static_cast<const float *>(weight), static_cast<const float *>(bias),
                                     static_cast<bf16_t *>(y), save_mean, save_rstd, eps, rows, width, s);
    return launch_layer_norm_fwd(static_cast<const bf16_t *>(x), x_row_stride, static_cast<const bf16_t *>(weight), static_cast<const bf16_t *>(bias),
                                 static_cast<bf16_t *>(y), save_mean, save_rstd, eps, rows, width, s);
}

int adder_layer_norm_bwd_workspace_bytes(long rows, int width, int type, size_t *bytes) {
    if (!bytes) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type)) return ADDER_ERR_BAD_SHAPE;
    if (width > kMaxWidth || wide(rows, width)) return ADDER_ERR_TOO_LARGE;
    *bytes = whole(sizeof(float) * 2 * (size_t)layer_norm_bwd_parts(rows, width) * width);
    return ADDER_OK;
}

int adder_layer_norm_bwd(const void *dy, long dy_row_stride, const void *x, long x_row_stride, const void *weight, const float *save_mean,
                         const float *save_rstd, void *gx, void *gweight, void *gbias, long rows, int width, int type, int weight_type, void *ws,
                         size_t ws_bytes, void *stream) {
    if (!dy || !x || !save_mean || !save_rstd || (!gx && !gweight && !gbias)) return ADDER_ERR_NULL_POINTER;
    if (rows <= 0 || width <= 0 || !known(type) || !known(weight_type) || bad_stride(x_row_stride, rows, width) ||
        bad_stride(dy_row_stride, rows, width))
        return ADDER_ERR_BAD_SHAPE;
    if (type == ADDER_TYPE_F32 && weight_type != type) return ADDER_ERR_UNSUPPORTED;
    if (width > kMaxWidth || wide(rows, width) || wide(rows, x_row_stride) || wide(rows, dy_row_stride)) return ADDER_ERR_TOO_LARGE;
    const bool sums = gweight || gbias;
    size_t need = 0;
    if (int rc = adder_layer_norm_bwd_workspace_bytes(rows, width, type, &need)) return rc;
    if (!sums) need = 0;
    if (int rc = check_workspace(ws, ws_bytes, need)) return rc;
    const size_t nw = size_of(weight_type) * (size_t)width, nr = sizeof(float) * (size_t)rows;
    const Span outs[] = {{gx, size_of(type) * (size_t)rows * width}, {gweight, nw}, {gbias, nw}, {ws, need}};
    const Span ins[] = {{dy, span(rows, dy_row_stride, width, type)}, {x, span(rows, x_row_stride, width, type)}, {weight, nw}, {save_mean, nr},
                        {save_rstd, nr}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float *part = static_cast<float *>(ws);
    if (type == ADDER_TYPE_F32)
        return launch_layer_norm_bwd(static_cast<const float *>(dy), dy_row_stride, static_cast<const float *>(x), x_row_stride,
                                     static_cast<const float *>(weight), save_mean, save_rstd, static_cast<float *>(gx), static_cast<float *>(gweight),
                                     static_cast<float *>(gbias), rows, width, part, s);
    if (weight_type == ADDER_TYPE_F32)
        return launch_layer_norm_bwd(static_cast<const bf16_t *>(dy), dy_row_stride, static_cast<const bf16_t *>(x), x_row_stride,
                                     static_cast<const float *>(weight), save_mean, save_rstd, static_cast<bf16_t *>(gx), static_cast<float *>(gweight),
                                     static_cast<float *>(gbias), rows, width, part, s);
    return launch_layer_norm_bwd(static_cast<const bf16_t *>(dy), dy_row_stride, static_cast<const bf16_t *>(x), x_row_stride,
                                 static_cast<const bf16_t *>(weight), save_mean, save_rstd, static_cast<bf16_t *>(gx), static_cast<bf16_t *>(gweight),
                                 static_cast<bf16_t *>(gbias), rows, width, part, s);
}

int adder_adamw_step(int count, void *const *params, const void *const *grads, float *const *exp_avgs, float *const *exp_avg_sqs, const long *n,
                     const float *lr_device, double lr, double beta1, double beta2, double eps, double weight_decay, long step,
                     const float *corrections_device, int type, void *stream) {
    if (!params || !grads || !exp_avgs || !exp_avg_sqs || !n) return ADDER_ERR_NULL_POINTER;
    if (!known(type)) return ADDER_ERR_BAD_SHAPE;
    AdamWArgs a;
    if (int rc = adamw_args(a, lr_device, lr, beta1, beta2, eps, weight_decay, step, corrections_device)) return rc;
    if (int rc = check_counts(count, ADDER_ADAMW_BATCH_MAX, n)) return rc;
    for (int t = 0; t < count; ++t) {
        if (!params[t] || !grads[t] || !exp_avgs[t] || !exp_avg_sqs[t]) return ADDER_ERR_NULL_POINTER;
        const size_t np = size_of(type) * (size_t)n[t], nm = sizeof(float) * (size_t)n[t];
        const Span outs[] = {{params[t], np}, {exp_avgs[t], nm}, {exp_avg_sqs[t], nm}};
        const Span ins[] = {{grads[t], np}};
        if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_adamw<bf16_t>(count, params, grads, exp_avgs, exp_avg_sqs, n, a, s)
                                   : launch_adamw<float>(count, params, grads, exp_avgs, exp_avg_sqs, n, a, s);
}

int adder_adamw_step_8bit(int count, void *const *params, const void *const *grads, signed char *const *exp_avgs, unsigned char *const *exp_avg_sqs,
                          float *const *exp_avg_scales, float *const *exp_avg_sq_scales, const long *n, const float *lr_device, double lr,
                          double beta1, double beta2, double eps, double weight_decay, long step, const float *corrections_device, int type,
                          void *stream) {
    if (!params || !grads || !exp_avgs || !exp_avg_sqs || !exp_avg_scales || !exp_avg_sq_scales || !n) return ADDER_ERR_NULL_POINTER;
    if (!known(type)) return ADDER_ERR_BAD_SHAPE;
    AdamWArgs a;
    if (int rc = adamw_args(a, lr_device, lr, beta1, beta2, eps, weight_decay, step, corrections_device)) return rc;
    if (int rc = check_counts(count, ADDER_ADAMW_8BIT_BATCH_MAX, n)) return rc;
    for (int t = 0; t < count; ++t) {
        if (!params[t] || !grads[t] || !exp_avgs[t] || !exp_avg_sqs[t] || !exp_avg_scales[t] || !exp_avg_sq_scales[t]) return ADDER_ERR_NULL_POINTER;
        const size_t np = size_of(type) * (size_t)n[t], ns = sizeof(float) * (size_t)((n[t] + kStateBlock - 1) / kStateBlock);
        const Span outs[] = {{params[t], np}, {exp_avgs[t], (size_t)n[t]}, {exp_avg_sqs[t], (size_t)n[t]}, {exp_avg_scales[t], ns},
                             {exp_avg_sq_scales[t], ns}};
        const Span ins[] = {{grads[t], np}};
        if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    int8_t *const *m = reinterpret_cast<int8_t *const *>(exp_avgs);
    return type == ADDER_TYPE_BF16 ? launch_adamw_8bit<bf16_t>(count, params, grads, m, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, n, a, s)
                                   : launch_adamw_8bit<float>(count, params, grads, m, exp_avg_sqs, exp_avg_scales, exp_avg_sq_scales, n, a, s);
}

int adder_adamw_advance(float *step_device, double beta1, double beta2, float *corrections, void *stream) {
    if (!step_device || !corrections) return ADDER_ERR_NULL_POINTER;
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return ADDER_ERR_BAD_SHAPE;
    if (overlaps(step_device, sizeof(float), corrections, 2 * sizeof(float))) return ADDER_ERR_ALIAS;
    return launch_adamw_advance(step_device, log(beta1), log(beta2), corrections, static_cast<hipStream_t>(stream));
}

int adder_state_values(const void *codes, int is_signed, const float *scales, void *values, long n, int type, void *stream) {
    if (!codes || !scales || !values) return ADDER_ERR_NULL_POINTER;
    if (n <= 0 || !known(type)) return ADDER_ERR_BAD_SHAPE;
    if (n > 17179869184L - 1024) return ADDER_ERR_TOO_LARGE;   // (2^31 threads of eight each)
    const Span outs[] = {{values, size_of(type) * (size_t)n}};
    const Span ins[] = {{codes, (size_t)n}, {scales, sizeof(float) * (size_t)((n + kStateBlock - 1) / kStateBlock)}};
    if (any_alias(outs, ins)) return ADDER_ERR_ALIAS;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return type == ADDER_TYPE_BF16 ? launch_state_values(codes, is_signed, scales, static_cast<bf16_t *>(values), n, s)
                                   : launch_state_values(codes, is_signed, scales, static_cast<float *>(values), n, s);
}

}  // extern "C"
