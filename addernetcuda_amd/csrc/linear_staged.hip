// The linear layers' products of float32 operands, and of bfloat16 ones that no load of 16 aligned bytes fits: any sizes, strides and
// alignments.
#include "product.hpp"

namespace adder {

// ---- tiles that pass through registers --------------------------------------------------------------------------------
// Four waves (2 x 2) compute BM x BN results, a wave TM x TN tiles of 16 x 16.  The next tiles of BK values of k are loaded into
// registers (zeros in place of what does not exist) while the ones in LDS are multiplied.
//
// float32: the matrix cores multiply floats at a sixteenth of the rate of bfloat16.  A float is the sum of three bfloat16 (hi = x
// rounded, mid = x - hi rounded, lo = x - hi - mid rounded: 8 bits each, 2^-27 of x is left), and of the nine products of two of
// them the six that matter, hi hi, hi mid, mid hi, mid mid, hi lo and lo hi, are summed in 32 bits: what is left out is 2^-26 of a
// product.  An operand that is infinite, not a number, or rounds up to infinity gives a sum that is not finite; a wave that finds some
// computes those again, in float32.
static constexpr int kStagedThreads = 256;
template <class T>
static constexpr int kStagedPlanes = sizeof(T) == 4 ? 3 : 1;
template <class T>
static constexpr int kStagedK = sizeof(T) == 4 ? 32 : 64;

__device__ __forceinline__ float low_f32(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high_f32(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
// two floats -> their hi, mid and lo, each pair as 32 bits
__device__ __forceinline__ void split(float x, float y, uint32_t (&o)[3]) {
    o[0] = pack_bf16(x, y);
    x -= low_f32(o[0]);
    y -= high_f32(o[0]);
    o[1] = pack_bf16(x, y);
    o[2] = pack_bf16(x - low_f32(o[1]), y - high_f32(o[1]));
}

// One operand's tile: loads of 16 bytes, of 4 floats or 8 bfloat16 that lie side by side
template <class T, int R, bool ACROSS>
struct Staged {
    static constexpr int E = Chunk<T>::n, BK = kStagedK<T>, P = kStagedPlanes<T>;
    typedef LdsTile<R, BK, ACROSS> Tile;
    static constexpr int row_loads = Tile::row_chunks * 8 / E, per = R * BK / E / kStagedThreads;
    uint4 v[per];

    __device__ __forceinline__ void load(const T *p, long ld, long rows, long k_end, long row0, long k0) {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int u = threadIdx.x + i * kStagedThreads, c = u % row_loads, r = u / row_loads;
            long left;
            const T *q;
            if constexpr (ACROSS) {
                left = k0 + r < k_end ? rows - row0 - c * E : 0;
                q = p + (k0 + r) * ld + row0 + c * E;
            } else {
                left = row0 + r < rows ? k_end - k0 - c * E : 0;
                q = p + (row0 + r) * ld + k0 + c * E;
            }
            v[i] = load_raw_part(q, left < 0 ? 0 : left < E ? (int)left : E);
        }
    }
    __device__ __forceinline__ void store(char *tile) const {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int u = threadIdx.x + i * kStagedThreads, c = u % row_loads, r = u / row_loads;
            if constexpr (P == 1) {
                *reinterpret_cast<uint4 *>(tile + r * Tile::row_bytes + (Tile::place(r, c) << 4)) = v[i];
            } else {
                uint32_t a[3], b[3];
                split(__uint_as_float(v[i].x), __uint_as_float(v[i].y), a);
                split(__uint_as_float(v[i].z), __uint_as_float(v[i].w), b);
                char *q = tile + r * Tile::row_bytes + (Tile::place(r, c >> 1) << 4) + ((c & 1) << 3);
#pragma unroll
                for (int k = 0; k < 3; ++k) *reinterpret_cast<uint2 *>(q + k * Tile::bytes) = make_uint2(a[k], b[k]);
            }
        }
    }
};

__device__ __forceinline__ f32x4 mfma(const bf16x8 &b, const bf16x8 &a, const f32x4 &acc) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, acc, 0, 0, 0);
}

// A wave's sums over its share of k that are not finite, with the float32 matrix instructions straight from memory
template <int TM, int TN, bool AA, bool BA>
__device__ __forceinline__ void sum_again(const ProductArgs &p, f32x4 (&acc)[TM][TN], long m0, long n0, long k_begin, long k_end, int lane) {
    const float *a = static_cast<const float *>(p.a), *b = static_cast<const float *>(p.b);
    f32x4 again[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) again[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (long k0 = k_begin; k0 < k_end; k0 += 4) {
        const long k = k0 + (lane >> 4);
        float fa[TM], fb[TN];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const long m = m0 + i * 16 + (lane & 15);
            fa[i] = k < k_end && m < p.M ? a[AA ? k * p.lda + m : m * p.lda + k] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const long n = n0 + j * 16 + (lane & 15);
            fb[j] = k < k_end && n < p.N ? b[BA ? k * p.ldb + n : n * p.ldb + k] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) again[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j], fa[i], again[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fabsf(acc[i][j][e]) < __builtin_inff() ? acc[i][j][e] : again[i][j][e];
}

// AHEAD: tiles in registers or on their way there.  Small tiles are multiplied faster than the next arrives.
template <class T, int TM, int TN, bool AA, bool BA>
__global__ __launch_bounds__(kStagedThreads, 2) void product_staged_kernel(const ProductArgs p) {
    constexpr int BM = TM * 32, BN = TN * 32, BK = kStagedK<T>, P = kStagedPlanes<T>, AHEAD = TM * TN <= 4 ? 3 : 1;
    typedef Staged<T, BM, AA> SA;
    typedef Staged<T, BN, BA> SB;
    __shared__ __align__(16) char lds[P * (SA::Tile::bytes + SB::Tile::bytes)];
    char *ta = lds, *tb = lds + P * SA::Tile::bytes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave & 1) * (TM * 16), wn = (wave >> 1) * (TN * 16);
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const long k_begin = blockIdx.y * p.k_share, k_end = k_begin + p.k_share < p.K ? k_begin + p.k_share : p.K;
    const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b);
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    SA sa[AHEAD];
    SB sb[AHEAD];
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
        sa[d].load(a, p.lda, p.M, k_end, m0, k_begin + d * BK);
        sb[d].load(b, p.ldb, p.N, k_end, n0, k_begin + d * BK);
    }
    auto step = [&](long k0, SA &na, SB &nb) {
        __syncthreads();
        na.store(ta);
        nb.store(tb);
        __syncthreads();
        if (k0 + AHEAD * BK < k_end) {
            na.load(a, p.lda, p.M, k_end, m0, k0 + AHEAD * BK);
            nb.load(b, p.ldb, p.N, k_end, n0, k0 + AHEAD * BK);
        }
#pragma unroll
        for (int k = 0; k < BK; k += 32) {
            bf16x8 fb[P][TN];
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[q][j] = SB::Tile::fragment(tb + q * SB::Tile::bytes, wn + j * 16, k, lane);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                bf16x8 fa[P];
#pragma unroll
                for (int q = 0; q < P; ++q) fa[q] = SA::Tile::fragment(ta + q * SA::Tile::bytes, wm + i * 16, k, lane);
#pragma unroll
                for (int u = P == 3 ? 2 : 0; u >= 0; --u)   // (the small products first)
#pragma unroll
                    for (int q = 0; q <= u; ++q)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = mfma(fb[u - q][j], fa[q], acc[i][j]);
            }
        }
    };
    for (long k0 = k_begin; k0 < k_end; k0 += AHEAD * BK)
#pragma unroll
        for (int d = 0; d < AHEAD; ++d)
            if (k0 + d * BK < k_end) step(k0 + d * BK, sa[d], sb[d]);
    if constexpr (P == 3) {
        bool finite = true;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) finite = finite && fabsf(acc[i][j][e]) < __builtin_inff();
        if (!__all(finite)) sum_again<TM, TN, AA, BA>(p, acc, m0 + wm, n0 + wn, k_begin, k_end, lane);
    }
    finish_wave<T, TM, TN>(p, acc, m0 + wm, n0 + wn, lane);
}

template <class T, int TM, int TN>
static int launch_staged(ProductArgs p, bool a_across, bool b_across, hipStream_t s) {
    p.tiles_m = (int)ceil_div_l(p.M, TM * 32);
    p.tiles_n = (int)ceil_div_l(p.N, TN * 32);
    const dim3 grid((unsigned)p.tiles_m * p.tiles_n, p.splits), threads(kStagedThreads);
    if (!a_across && !b_across) hipLaunchKernelGGL((product_staged_kernel<T, TM, TN, false, false>), grid, threads, 0, s, p);
    else if (!a_across) hipLaunchKernelGGL((product_staged_kernel<T, TM, TN, false, true>), grid, threads, 0, s, p);
    else hipLaunchKernelGGL((product_staged_kernel<T, TM, TN, true, true>), grid, threads, 0, s, p);
    return check_launch();
}
template <class T>
int launch_product_staged(ProductArgs p, bool a_across, bool b_across, bool small, hipStream_t s) {
    return small ? launch_staged<T, 2, 2>(p, a_across, b_across, s) : launch_staged<T, 4, 4>(p, a_across, b_across, s);
}
template int launch_product_staged<float>(ProductArgs, bool, bool, bool, hipStream_t);
template int launch_product_staged<bf16_t>(ProductArgs, bool, bool, bool, hipStream_t);

}  // namespace adder
