// The linear layers' forward for few rows: a single token's, a small batch's.
#include "product.hpp"

namespace adder {

// ---- few rows of x: the time is that of reading w ---------------------------------------------------------------------
// A workgroup takes sixteen rows of w (columns of the output) and up to 16 MT rows of x.  Its waves take turns along k, 128
// bytes of every row at a time, straight from memory into the matrix instructions' operands -- a lane 32 of a row's 128
// bytes, so that lines are used whole -- and add their sums through LDS.  No tile of w is read twice by a workgroup, nothing waits
// for a barrier before the end, and no second launch joins anything.  One row, 4096 x 4096 in bfloat16: 7.4 us in a graph (4.5 TB/s)
// with everything around it; 64 rows 11.5 us; one float32 row 14 us.  float32 stays float32: the matrix cores' rate for it is enough
// beside the loads.
template <int MT>
static constexpr int kRowsWaves = MT == 4 ? 8 : 16;   // (four tiles of x and what arrives behind them take more than 128 registers)

__device__ __forceinline__ void multiply(f32x4 &acc, const uint4 &b, const uint4 &a, float) {
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.x), __uint_as_float(a.x), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.y), __uint_as_float(a.y), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.z), __uint_as_float(a.z), acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b.w), __uint_as_float(a.w), acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(f32x4 &acc, const uint4 &b, const uint4 &a, bf16_t) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, b), __builtin_bit_cast(bf16x8, a), acc, 0, 0, 0);
}

template <class T, int MT>
__global__ __launch_bounds__(kRowsWaves<MT> * 64) void product_rows_kernel(const ProductArgs p) {
    constexpr int E = Chunk<T>::n, BK = 8 * E, U = MT == 1 ? 2 : 1;   // blocks that a wave multiplies while as many arrive
    extern __shared__ __align__(16) char lds[];
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, l16 = lane & 15;
    const long n0 = (long)blockIdx.x * 16, m0 = (long)blockIdx.y * (16 * MT);
    const T *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b);
    const int mine = (lane >> 4) * E;   // of half a block's values of k
    // (rows past the last: that one again; their results are not stored)
    const T *pb = b + (n0 + l16 < p.N ? n0 + l16 : p.N - 1) * p.ldb + mine, *pa[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long m = m0 + i * 16 + l16;
        pa[i] = a + (m < p.M ? m : p.M - 1) * p.lda + mine;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Blocks { uint4 b[U][2], a[U][MT][2]; };
    auto load = [&](Blocks &t, long kb) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const long k = (kb + u * waves) * BK + h * (4 * E);
                t.b[u][h] = load_raw(pb + k);
#pragma unroll
                for (int i = 0; i < MT; ++i) t.a[u][i][h] = load_raw(pa[i] + k);
            }
    };
    auto add = [&](const Blocks &t) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < MT; ++i) multiply(acc[i], t.b[u][h], t.a[u][i][h], T{});
    };
    const long whole = p.K / BK, turn = U * waves, last = whole - (U - 1) * waves;   // (a turn begins below `last`)
    long kb = wave;
    if (kb < last) {
        Blocks t[2];
        load(t[0], kb);
        for (;;) {   // (two turns a pass: a copy of what is on its way would wait for it)
            if (kb + turn < last) load(t[1], kb + turn);
            add(t[0]);
            kb += turn;
            if (kb >= last) break;
            if (kb + turn < last) load(t[0], kb + turn);
            add(t[1]);
            kb += turn;
            if (kb >= last) break;
        }
    }
    for (; kb * BK < p.K; kb += waves) {
        const long k = kb * BK, left = p.K - k - mine;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long rest = left - h * (4 * E);
            const int valid = rest < 0 ? 0 : rest < E ? (int)rest : E;
            const uint4 fb = load_raw_part(pb + k + h * (4 * E), valid);
#pragma unroll
            for (int i = 0; i < MT; ++i) multiply(acc[i], fb, load_raw_part(pa[i] + k + h * (4 * E), valid), T{});
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[(wave * MT + i) * 64 + lane] = acc[i];
    __syncthreads();
    for (int t = threadIdx.x; t < MT * 64; t += blockDim.x) {
        f32x4 s = sums[t];
        for (int w = 1; w < waves; ++w) s += sums[w * MT * 64 + t];
        const long m = m0 + t / 64 * 16 + (t & 15), n = n0 + (t >> 4 & 3) * 4;
        if (m < p.M && n < p.N) {
            const float v[4] = {s[0], s[1], s[2], s[3]};
            finish<T>(p, m, n, p.N - n < 4 ? (int)(p.N - n) : 4, v);
        }
    }
}

template <class T, int MT>
static int launch_rows(const ProductArgs &p, hipStream_t s) {
    const long blocks = ceil_div_l(p.K, 8 * Chunk<T>::n);
    const int waves = (int)(blocks < kRowsWaves<MT> ? blocks : kRowsWaves<MT>);
    hipLaunchKernelGGL((product_rows_kernel<T, MT>), dim3((unsigned)ceil_div_l(p.N, 16), (unsigned)ceil_div_l(p.M, 16 * MT)), dim3(waves * 64),
                       waves * MT * 1024, s, p);
    return check_launch();
}
template <class T>
int launch_product_rows(const ProductArgs &p, hipStream_t s) {
    switch (product_rows_tiles(p.M)) {
        case 1: return launch_rows<T, 1>(p, s);
        case 2: return launch_rows<T, 2>(p, s);
        default: return launch_rows<T, 4>(p, s);
    }
}
template int launch_product_rows<float>(const ProductArgs &, hipStream_t);
template int launch_product_rows<bf16_t>(const ProductArgs &, hipStream_t);

}  // namespace adder
