// What the C entry points of the layers beside the adder layers check their arguments with, and how they call a product.
#pragma once
#include "checks.hpp"
#include "layers.hpp"

namespace adder {

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

static size_t product_bytes(long M, long N, long K, int type, bool gated = false) {
    return type == ADDER_TYPE_BF16 ? product_workspace_bytes<bf16_t>(M, N, K, gated) : product_workspace_bytes<float>(M, N, K, gated);
}
static int product(const Product &p, int type, void *ws, hipStream_t s) {
    return type == ADDER_TYPE_BF16 ? launch_product<bf16_t>(p, ws, s) : launch_product<float>(p, ws, s);
}

}  // namespace adder
