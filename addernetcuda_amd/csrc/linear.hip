// Linear layers: y = act(x w' + b) + r and its gradients,
//     z = x w' + b,   dz = dy * act'(z),   gx = dz w,   gw = dz' x,   gb = sum over rows of dz.
// All three products are out[m, n] = sum_k A(m, k) B(n, k) with k along or across the rows of either operand.
#include "layers.hpp"

namespace adder {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- activations ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + expf(-z)); }
__device__ __forceinline__ float activate(float z, Act act) {
    switch (act) {
        case Act::relu: return relu_keep_nan(z);
        case Act::gelu: return 0.5f * z * (1.f + erff(z * 0.70710678f));
        case Act::silu: return z * sigmoid(z);
        default: return z;
    }
}
__device__ __forceinline__ float slope(float z, Act act) {
    switch (act) {
        case Act::relu: return z <= 0.f ? 0.f : 1.f;
        case Act::gelu: return 0.5f * (1.f + erff(z * 0.70710678f)) + 0.39894228f * z * expf(-0.5f * z * z);
        case Act::silu: {
            const float s = sigmoid(z);
            return s * (1.f + z * (1.f - s));
        }
        default: return 1.f;
    }
}

// ---- the product in tiles, for any sizes, strides and alignments -----------------------------------------------------
// A workgroup of four waves (2 x 2) computes BM x BN results.  Both operands' tiles hold 128 bytes of k a row -- 64 bfloat16
// or 32 floats -- in LDS, in 16-byte chunks that are exchanged by the row's low bits so that the sixteen rows of a matrix
// instruction's operand spread over the banks; they are double-buffered, the next tile's loads under way while this one is
// multiplied.  An operand with k across its rows is transposed in registers between its load and its store to LDS.  The
// matrix instruction takes B as its rows: a lane then holds four neighbouring results of one row of the output.
static constexpr int kTileThreads = 256, kTileBytes = 128, kTileChunks = kTileBytes / 16;

__device__ __forceinline__ int tile_at(int row, int chunk) { return row * kTileBytes + ((chunk ^ (row & 7)) << 4); }

template <class T>
__device__ __forceinline__ void transpose_chunks(const uint4 (&in)[Chunk<T>::n], uint4 (&out)[Chunk<T>::n]) {
    if constexpr (Chunk<T>::n == 4) {
        out[0] = make_uint4(in[0].x, in[1].x, in[2].x, in[3].x);
        out[1] = make_uint4(in[0].y, in[1].y, in[2].y, in[3].y);
        out[2] = make_uint4(in[0].z, in[1].z, in[2].z, in[3].z);
        out[3] = make_uint4(in[0].w, in[1].w, in[2].w, in[3].w);
    } else {
        uint32_t w[8][4];
#pragma unroll
        for (int k = 0; k < 8; ++k) { w[k][0] = in[k].x; w[k][1] = in[k].y; w[k][2] = in[k].z; w[k][3] = in[k].w; }
#pragma unroll
        for (int m = 0; m < 8; ++m) {
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t lo = w[2 * j][m / 2], hi = w[2 * j + 1][m / 2];
                o[j] = m & 1 ? (hi & 0xffff0000u) | (lo >> 16) : (hi << 16) | (lo & 0xffffu);
            }
            out[m] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// One operand's tile of R rows from row0 and k0 on: into registers, and from there to LDS.
template <class T, int R, bool ACROSS>
struct TileLoad {
    static constexpr int E = Chunk<T>::n, BK = kTileBytes / (int)sizeof(T);
    // along: chunks (row, c); across: blocks of E x E values (rows mb * E.., k kb * E..)
    static constexpr int units = ACROSS ? R / E * (BK / E) : R * kTileChunks;
    static constexpr int per = (units + kTileThreads - 1) / kTileThreads, regs = ACROSS ? per * E : per;
    uint4 v[regs];

    __device__ __forceinline__ void load(const T *p, long ld, long rows, long k_end, long row0, long k0) {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int u = threadIdx.x + i * kTileThreads;
            if constexpr (ACROSS) {
                const int mb = u % (R / E), kb = u / (R / E);
                const long r = row0 + mb * E, k = k0 + kb * E;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const long left = k + e < k_end && kb < BK / E ? rows - r : 0;
                    v[i * E + e] = load_raw_part(p + (k + e) * ld + r, left < E ? (int)left : E);
                }
            } else {
                const int c = u % kTileChunks, row = u / kTileChunks;
                const long k = k0 + c * E, left = row0 + row < rows ? k_end - k : 0;
                v[i] = load_raw_part(p + (row0 + row) * ld + k, left < 0 ? 0 : left < E ? (int)left : E);
            }
        }
    }
    __device__ __forceinline__ void store(char *tile) const {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int u = threadIdx.x + i * kTileThreads;
            if constexpr (ACROSS) {
                const int mb = u % (R / E), kb = u / (R / E);
                uint4 in[E], out[E];
#pragma unroll
                for (int e = 0; e < E; ++e) in[e] = v[i * E + e];
                transpose_chunks<T>(in, out);
                if (kb < BK / E)
#pragma unroll
                    for (int e = 0; e < E; ++e) *reinterpret_cast<uint4 *>(tile + tile_at(mb * E + e, kb)) = out[e];
            } else {
                *reinterpret_cast<uint4 *>(tile + tile_at(u / kTileChunks, u % kTileChunks)) = v[i];
            }
        }
    }
};

// acc += the products of one 16-byte chunk of each operand per lane: 32 bfloat16 or 16 floats of k
__device__ __forceinline__ void multiply(f32x4 &acc, const uint4 &b, const uint4 &a, float) {
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.x), __uint_as_float(a.x), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.y), __uint_as_float(a.y), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.z), __uint_as_float(a.z), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.w), __uint_as_float(a.w), acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(f32x4 &acc, const uint4 &b, const uint4 &a, bf16_t) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
}

struct ProductArgs {
    const void *a, *b, *bias, *res;
    void *out, *pre;
    float *part;          // splits > 1: (splits, M, N) sums without an epilogue
    long lda, ldb, ldr, M, N, K, k_share;
    int tiles_n, splits;
    Act act;
};

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
    for (int e = 0; e < 4; ++e) {
        z[e] = sum[e] + b[e];
        y[e] = activate(z[e], p.act) + r[e];
    }
    if (cnt == 4) {
        put4(out + at, y);
        if (pre) put4(pre + at, z);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < cnt) {
                put(out + at + e, y[e]);
                if (pre) put(pre + at + e, z[e]);
            }
    }
}

template <class T, int BM, int BN, bool AA, bool BA>
__global__ __launch_bounds__(kTileThreads) void product_tile_kernel(const ProductArgs p) {
    constexpr int BK = kTileBytes / (int)sizeof(T), TM = BM / 32, TN = BN / 32;   // tiles of 16 x 16 a wave
    __shared__ __align__(16) char lds[2][(BM + BN) * kTileBytes];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quad = lane >> 4, l16 = lane & 15;
    const int wm = (wave & 1) * (BM / 2), wn = (wave >> 1) * (BN / 2);
    const long m0 = (long)(blockIdx.x / p.tiles_n) * BM, n0 = (long)(blockIdx.x % p.tiles_n) * BN;
    const long k_begin = blockIdx.y * p.k_share, k_end = k_begin + p.k_share < p.K ? k_begin + p.k_share : p.K;
    const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    TileLoad<T, BM, AA> ta;
    TileLoad<T, BN, BA> tb;
    ta.load(a, p.lda, p.M, k_end, m0, k_begin);
    tb.load(b, p.ldb, p.N, k_end, n0, k_begin);
    int buf = 0;
    for (long k0 = k_begin; k0 < k_end; k0 += BK, buf ^= 1) {
        ta.store(lds[buf]);
        tb.store(lds[buf] + BM * kTileBytes);
        __syncthreads();   // (one barrier a tile: the other buffer was read before the one in front of this)
        if (k0 + BK < k_end) {
            ta.load(a, p.lda, p.M, k_end, m0, k0 + BK);
            tb.load(b, p.ldb, p.N, k_end, n0, k0 + BK);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 fa[TM], fb[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i)
                fa[i] = *reinterpret_cast<const uint4 *>(lds[buf] + tile_at(wm + i * 16 + l16, h * 4 + quad));
#pragma unroll
            for (int j = 0; j < TN; ++j)
                fb[j] = *reinterpret_cast<const uint4 *>(lds[buf] + BM * kTileBytes + tile_at(wn + j * 16 + l16, h * 4 + quad));
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) multiply(acc[i][j], fb[j], fa[i], T{});
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const long m = m0 + wm + i * 16 + l16;
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const long n = n0 + wn + j * 16 + quad * 4;
            if (n >= p.N) continue;
            const int cnt = p.N - n < 4 ? (int)(p.N - n) : 4;
            const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
            if (p.splits > 1) {
                float *o = p.part + ((long)blockIdx.y * p.M + m) * p.N + n;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < cnt) o[e] = v[e];
            } else {
                finish<T>(p, m, n, cnt, v);
            }
        }
    }
}

// The shares of the sums added up in their order, and the epilogue: four results a thread
template <class T>
__global__ __launch_bounds__(256) void product_join_kernel(const ProductArgs p) {
    const long groups = (p.N + 3) / 4, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.M * groups) return;
    const long m = i / groups, n = i % groups * 4;
    const int cnt = p.N - n < 4 ? (int)(p.N - n) : 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) {
        const float *q = p.part + ((long)s * p.M + m) * p.N + n;
        float t[4] = {0.f, 0.f, 0.f, 0.f};
        if (cnt == 4) {
            ld_strip<4>(q, t);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < cnt) t[e] = q[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
    }
    finish<T>(p, m, n, cnt, v);
}

// ---- which tiles ----------------------------------------------------------------------------------------------------
struct ProductPlan { int bm, bn, splits; long k_share; };
static constexpr int kCUs = 256;

template <class T>
static ProductPlan plan_product(long M, long N, long K) {
    constexpr int BK = kTileBytes / (int)sizeof(T);
    ProductPlan p{128, 128, 1, K};
    if (ceil_div_l(M, 128) * ceil_div_l(N, 128) < kCUs) p.bm = p.bn = 64;
    const long tiles = ceil_div_l(M, p.bm) * ceil_div_l(N, p.bn), steps = ceil_div_l(K, BK);
    long splits = tiles < kCUs ? kCUs / tiles : 1;
    if (splits > steps / 4) splits = steps / 4;   // (at least four tiles of k each: the join is a launch of its own)
    if (splits > 16) splits = 16;
    if (splits > 1) {
        p.k_share = ceil_div_l(steps, splits) * BK;
        p.splits = (int)ceil_div_l(K, p.k_share);
    }
    return p;
}

template <class T>
size_t product_workspace_bytes(long M, long N, long K) {
    const ProductPlan p = plan_product<T>(M, N, K);
    return p.splits > 1 ? sizeof(float) * (size_t)p.splits * M * N : 0;
}

template <class T, int BM, int BN>
static int launch_tiles(const Product &q, const ProductArgs &p, hipStream_t s) {
    const dim3 grid((unsigned)(ceil_div_l(p.M, BM) * p.tiles_n), p.splits);
    if (!q.a_across && !q.b_across) hipLaunchKernelGGL((product_tile_kernel<T, BM, BN, false, false>), grid, dim3(kTileThreads), 0, s, p);
    else if (!q.a_across) hipLaunchKernelGGL((product_tile_kernel<T, BM, BN, false, true>), grid, dim3(kTileThreads), 0, s, p);
    else hipLaunchKernelGGL((product_tile_kernel<T, BM, BN, true, true>), grid, dim3(kTileThreads), 0, s, p);
    return check_launch();
}

template <class T>
int launch_product(const Product &q, void *ws, hipStream_t s) {
    const ProductPlan plan = plan_product<T>(q.M, q.N, q.K);
    const ProductArgs p{q.a, q.b, q.bias, q.res, q.out, q.pre, static_cast<float *>(ws), q.lda, q.ldb, q.ldr, q.M, q.N, q.K, plan.k_share,
                        (int)ceil_div_l(q.N, plan.bn), plan.splits, q.act};
    const int rc = plan.bm == 128 ? launch_tiles<T, 128, 128>(q, p, s) : launch_tiles<T, 64, 64>(q, p, s);
    if (rc || plan.splits == 1) return rc;
    hipLaunchKernelGGL(product_join_kernel<T>, dim3((unsigned)ceil_div_l(q.M * ((q.N + 3) / 4), 256)), dim3(256), 0, s, p);
    return check_launch();
}

// ---- the activation's derivative and the bias's gradient ---------------------------------------------------------------
// A workgroup takes 64 lanes' chunks of columns and a share of the rows: its four waves walk over the rows, and their column
// sums are added through LDS into one slab per share.
template <class T>
__global__ __launch_bounds__(256) void act_bwd_kernel(const T *__restrict__ dy, long dy_stride, const T *__restrict__ z,
                                                      T *__restrict__ dz, float *__restrict__ part, Act act, long rows, long N) {
    constexpr int V = Chunk<T>::n;
    __shared__ float lds[4][64 * V];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n = ((long)blockIdx.x * 64 + lane) * V;
    const int left = N - n < V ? (int)(N - n < 0 ? 0 : N - n) : V;
    float sum[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sum[e] = 0.f;
    for (long m = (long)blockIdx.y * 4 + wave; m < rows; m += (long)gridDim.y * 4) {
        float g[V], v[V];
        load_part(dy + m * dy_stride + n, left, g);
        if (act != Act::none) {
            load_part(z + m * N + n, left, v);
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] *= slope(v[e], act);
            if (dz) store_part(dz + m * N + n, left, g);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) sum[e] += g[e];
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

int act_bwd_parts(long rows, long N) {
    const long columns = ceil_div_l(N, 256), need = ceil_div_l(rows, 16), most = ceil_div_l(1024, columns);
    return (int)(need < most ? need : most);
}

template <class T>
int launch_act_bwd(const T *dy, long dy_stride, const T *z, T *dz, float *part, Act act, long rows, long N, hipStream_t s) {
    hipLaunchKernelGGL(act_bwd_kernel<T>, dim3((unsigned)ceil_div_l(N, 64 * Chunk<T>::n), act_bwd_parts(rows, N)), dim3(256), 0, s, dy,
                       dy_stride, z, dz, part, act, rows, N);
    return check_launch();
}

#define ADDER_LINEAR_INSTANCE(T)                                                                                      \
    template size_t product_workspace_bytes<T>(long, long, long);                                                     \
    template int launch_product<T>(const Product &, void *, hipStream_t);                                            \
    template int launch_act_bwd<T>(const T *, long, const T *, T *, float *, Act, long, long, hipStream_t);
ADDER_LINEAR_INSTANCE(float)
ADDER_LINEAR_INSTANCE(bf16_t)

}  // namespace adder
