// What the kernels of the linear layers' products share: activations, the epilogue, the matrix instructions' operands.
#pragma once
#include "layers.hpp"

namespace adder {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---- activations ---------------------------------------------------------------------------------------------------
// EXACT: float32 results.  The others are rounded to bfloat16 behind this: 1 / (1 + exp) and the normal distribution's function
// from one exponential and one reciprocal instruction (Abramowitz and Stegun 7.1.26, 1.5e-7 off at most).  An epilogue of a
// large tile has nothing beside it to hide behind, and erff costs three times as much.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float x) {
    return EXACT ? expf(x) : __builtin_amdgcn_exp2f(x * 1.44269504f);
}
template <bool EXACT>
__device__ __forceinline__ float sigmoid(float z) {
    return EXACT ? 1.f / (1.f + expf(-z)) : __builtin_amdgcn_rcpf(1.f + exp_of<false>(-z));
}
// Phi(z), and exp(-z^2 / 2) on the way
template <bool EXACT>
__device__ __forceinline__ float normal_cdf(float z, float &bell) {
    bell = exp_of<EXACT>(-0.5f * z * z);
    if constexpr (EXACT) {
        return 0.5f * (1.f + erff(z * 0.70710678f));
    } else {
        const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.3275911f * 0.70710678f, 1.f));
        const float tail = 0.5f * t * bell * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        return z < 0.f ? tail : 1.f - tail;
    }
}
template <bool EXACT>
__device__ __forceinline__ float activate(float z, Act act) {
    float bell;
    switch (act) {
        case Act::relu: return relu_keep_nan(z);
        case Act::gelu: return z * normal_cdf<EXACT>(z, bell);
        case Act::silu: return z * sigmoid<EXACT>(z);
        default: return z;
    }
}
// the derivative of a GELU or SiLU
template <bool EXACT>
__device__ __forceinline__ float slope(float z, Act act) {
    switch (act) {
        case Act::gelu: {
            float bell;
            const float p = normal_cdf<EXACT>(z, bell);
            return fmaf(0.39894228f * z, bell, p);
        }
        case Act::silu: {
            const float s = sigmoid<EXACT>(z);
            return s * fmaf(z, 1.f - s, 1.f);
        }
        default: return 1.f;
    }
}
template <class T>
static constexpr bool kExactAct = sizeof(T) == 4;

// z as it is kept for the backward.  In bfloat16 a GELU's or SiLU's is an IEEE half, of 11 bits instead of 8: a derivative from z in
// bfloat16 alone would be 6e-4 off, beside the 1.6e-3 of rounding dz.  Rounded toward zero (v_cvt_pkrtz_f16_f32), so that no finite z
// becomes infinite: beyond 65504 the derivative is a constant.  A ReLU's has z's sign, in the layer's type.
__host__ __device__ constexpr bool keeps_half(size_t size, Act act) { return size == 2 && (act == Act::gelu || act == Act::silu); }
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(lo, hi)); }
__device__ __forceinline__ uint4 pack_half(const float (&v)[8]) {
    return make_uint4(pack_half(v[0], v[1]), pack_half(v[2], v[3]), pack_half(v[4], v[5]), pack_half(v[6], v[7]));
}
__device__ __forceinline__ void unpack_half(const uint4 &u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e / 2] >> (16 * (e & 1))));
}

// ---- products ------------------------------------------------------------------------------------------------------
struct ProductArgs {
    const void *a, *b, *bias, *res;
    void *out, *pre;
    float *part;          // splits > 1: (splits, M, N) sums without an epilogue
    long lda, ldb, ldr, M, N, K, k_share;
    int tiles_m, tiles_n, splits;
    Act act;
};

__device__ __forceinline__ void keep(float *p, float z, Act) { *p = z; }
__device__ __forceinline__ void keep(bf16_t *p, float z, Act act) { *p = keeps_half(2, act) ? (bf16_t)pack_half(z, 0.f) : round_bf16(z); }
__device__ __forceinline__ void keep4(float *p, const float (&z)[4], Act) { put4(p, z); }
__device__ __forceinline__ void keep4(bf16_t *p, const float (&z)[4], Act act) {
    if (!keeps_half(2, act)) return put4(p, z);
    const uint32_t lo = pack_half(z[0], z[1]), hi = pack_half(z[2], z[3]);
    *reinterpret_cast<u16x4_any *>(p) = u16x4_any{(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
}

// `cnt` <= 4 neighbouring sums of row m from column n on: the epilogue
template <class T>
__device__ __forceinline__ void finish(const ProductArgs &p, long m, long n, int cnt, const float (&sum)[4]) {
    const T *bias = static_cast<const T *>(p.bias), *res = static_cast<const T *>(p.res);
    T *out = static_cast<T *>(p.out), *pre = static_cast<T *>(p.pre);
    const long at = m * p.N + n;
    float b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f}, z[4], y[4];
    if (cnt == 4) {
        if (bias) ld_strip<4>(bias + n, b);
        if (res) ld_strip<4>(res + m * p.ldr + n, r);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e) {
            if (bias && e < cnt) b[e] = ldf(bias + n + e);
            if (res && e < cnt) r[e] = ldf(res + m * p.ldr + n + e);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = sum[e] + b[e];
    switch (p.act) {   // (outside the loop: one branch for four values)
        case Act::relu:
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = activate<kExactAct<T>>(z[e], Act::relu);
            break;
        case Act::gelu:
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = activate<kExactAct<T>>(z[e], Act::gelu);
            break;
        case Act::silu:
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = activate<kExactAct<T>>(z[e], Act::silu);
            break;
        default:
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = z[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] += r[e];
    if (cnt == 4) {
        put4(out + at, y);
        if (pre) keep4(pre + at, z, p.act);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < cnt) {
                put(out + at + e, y[e]);
                if (pre) keep(pre + at + e, z[e], p.act);
            }
    }
}

// The epilogue of a wave's tile that lies within the output: TM x TN tiles of 16 x 16.  A lane holds four neighbouring results of
// each; in bfloat16 lanes 16 apart exchange theirs between two tiles that lie side by side, so that each stores eight neighbours.
__device__ __forceinline__ void swap_rows(uint32_t &u, uint32_t &v) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, v, false, false);   // odd rows of sixteen lanes of u with the even ones of v
    u = r[0];
    v = r[1];
}
template <class T, int TM, int TN, Act ACT>
__device__ __forceinline__ void finish_tile(const ProductArgs &p, const f32x4 (&acc)[TM][TN], long m0, long n0, int lane) {
    constexpr int V = Chunk<T>::n, G = V / 4;   // tiles side by side that make a chunk
    const T *bias = static_cast<const T *>(p.bias), *res = static_cast<const T *>(p.res);
    T *out = static_cast<T *>(p.out), *pre = static_cast<T *>(p.pre);
    const int quad = lane >> 4;
    float b[TN][4];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[j][e] = 0.f;
        if (bias) ld_strip<4>(bias + n0 + j * 16 + quad * 4, b[j]);
    }
    // the first of a lane's columns in the first G tiles: as they stand, or after the exchange
    const long at = n0 + (G == 1 ? quad * 4 : (quad & 1) * 16 + (quad >> 1) * 8);
    auto exchange = [](uint4 &q) {
        if constexpr (G == 2) {
            swap_rows(q.x, q.z);
            swap_rows(q.y, q.w);
        }
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long m = m0 + i * 16 + (lane & 15);
        uint4 r[TN / G];
        if (res) {
#pragma unroll
            for (int j = 0; j < TN / G; ++j) r[j] = load_raw(res + m * p.ldr + at + j * (16 * G));
        }
#pragma unroll
        for (int j = 0; j < TN; j += G) {
            float z[V], y[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                z[e] = acc[i][j + e / 4][e % 4] + b[j + e / 4][e % 4];
                y[e] = activate<kExactAct<T>>(z[e], ACT);
            }
            if (res) {
                uint4 &q = r[j / G];
                exchange(q);
                float v[V];
                unpack(q, v);
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] += v[e];
            }
            uint4 o = pack(y);
            exchange(o);
            store_raw(out + m * p.N + at + j * 16, o);
            if (pre) {
                uint4 q;
                if constexpr (keeps_half(sizeof(T), ACT)) q = pack_half(z);
                else q = pack(z);
                exchange(q);
                store_raw(pre + m * p.N + at + j * 16, q);
            }
        }
    }
}

// A wave's results: the epilogue, or the sums of a share of k
template <class T, int TM, int TN>
__device__ __forceinline__ void finish_wave(const ProductArgs &p, const f32x4 (&acc)[TM][TN], long m0, long n0, int lane) {
    if (p.splits == 1 && m0 + TM * 16 <= p.M && n0 + TN * 16 <= p.N) {
        switch (p.act) {
            case Act::relu: finish_tile<T, TM, TN, Act::relu>(p, acc, m0, n0, lane); break;
            case Act::gelu: finish_tile<T, TM, TN, Act::gelu>(p, acc, m0, n0, lane); break;
            case Act::silu: finish_tile<T, TM, TN, Act::silu>(p, acc, m0, n0, lane); break;
            default: finish_tile<T, TM, TN, Act::none>(p, acc, m0, n0, lane);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long m = m0 + i * 16 + (lane & 15);
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const long n = n0 + j * 16 + (lane >> 4) * 4;
            if (n >= p.N) continue;
            const int cnt = p.N - n < 4 ? (int)(p.N - n) : 4;
            const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (p.splits > 1) {
                float *o = p.part + ((long)blockIdx.y * p.M + m) * p.N + n;
                if (cnt == 4) {
                    st_strip<4>(o, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (e < cnt) o[e] = v[e];
                }
            } else {
                finish<T>(p, m, n, cnt, v);
            }
        }
    }
}

template <bool V>
struct Flag { static constexpr bool value = V; };

// ---- operands in LDS -------------------------------------------------------------------------------------------------
// A tile of R rows (or columns, with k across the rows) by BK values of k in bfloat16.  Where rows lie a power of two apart, a bank
// conflict is avoided by the order of their 16-byte chunks:
//   k along the rows:   row r has BK / 8 chunks; chunk c at place c ^ (r & 7) (rows of 128 bytes) or c ^ (r / 2 & 3) (64 bytes)
//   k across the rows:  row k has R / 8 chunks, read in pairs by 32 lanes at once: rows 0 to 3 and 8 to 11 of sixteen, or 4 to 7 and 12 to
//                       15.  Chunk c at place c ^ 2 (k & 3 | k / 8 & 1 << 2), below 128 columns, where two rows lie beside each other in
//                       the 64 banks, c ^ 2 (k / 2 & 1 | k / 8 & 1 << 1)
template <int R, int BK, bool ACROSS>
struct LdsTile {
    static constexpr int bytes = R * BK * 2, row_bytes = ACROSS ? R * 2 : BK * 2, row_chunks = row_bytes / 16;
    static __device__ __forceinline__ int place(int row, int chunk) {
        if constexpr (ACROSS) return chunk ^ (R >= 128 ? (row & 3) << 1 | (row & 8) : (row & 2) | (row & 8) >> 1);
        else return BK == 64 ? chunk ^ (row & 7) : chunk ^ ((row >> 1) & 3);
    }
    // values k + 8 (lane / 16) .. + 7 of row (column) at + lane % 16, a matrix instruction's operand.  With k across the rows:
    // ds_read_b64_tr_b16 takes four rows of sixteen columns from sixteen lanes, four columns each, and gives each lane a column.
    static __device__ __forceinline__ bf16x8 fragment(const char *tile, int at, int k, int lane) {
        if constexpr (ACROSS) {
            typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
            const int i = lane & 15, row = k + (lane >> 4) * 8 + (i >> 2), c = at / 8 + ((i & 3) >> 1);
            const char *q = tile + row * row_bytes + (place(row, c) << 4) + ((i & 1) << 3);   // (four rows on: the same place)
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)q);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(q + 4 * row_bytes));
            struct Both { s16x4 lo, hi; };
            return __builtin_bit_cast(bf16x8, Both{lo, hi});
        } else {
            const int row = at + (lane & 15);
            return *reinterpret_cast<const bf16x8 *>(tile + row * row_bytes + (place(row, k / 8 + (lane >> 4)) << 4));
        }
    }
};

// Workgroup number -> tile.  Workgroups go to the eight dies in turn, each with its own L2: a die takes consecutive tiles, and those
// run down eight rows of tiles before they go to the next column, so that the operands' tiles stay in its L2.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int whole = tiles_m * tiles_n & ~7;
    if (id < whole) id = (id & 7) * (whole >> 3) + (id >> 3);
    const int strip = id / (8 * tiles_n), in = id - strip * 8 * tiles_n, high = tiles_m - strip * 8 < 8 ? tiles_m - strip * 8 : 8;
    tm = strip * 8 + in % high;
    tn = in / high;
}

// Launches of the tiled kernels; p has everything but its tiles
enum class StreamShape { big, wide, mid, small };   // 256 x 256, 128 x 256, 128 x 128, 64 x 64 results a workgroup
int launch_product_stream(ProductArgs p, bool a_across, bool b_across, StreamShape shape, hipStream_t s);
// 128 x 128, 64 x 64, and (float32) both by twice as many waves, for launches that leave a compute unit one workgroup
enum class StagedShape { large, small, alone, pair };
template <class T>
int launch_product_staged(const ProductArgs &p, bool a_across, bool b_across, StagedShape shape, hipStream_t s);
template <class T>
int launch_product_rows(const ProductArgs &p, hipStream_t s);   // both along; few rows
inline int product_rows_tiles(long M) { return M <= 16 ? 1 : M <= 32 ? 2 : 4; }   // of sixteen rows that a workgroup takes

}  // namespace adder
