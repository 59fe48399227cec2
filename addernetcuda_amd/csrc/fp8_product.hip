// Products of e4m3 codes with block scales:
//     out[m, n] = act(sum over blocks b of 128 values of k  xs[m, b] ws[n / 128, b] (sum_{k in b} x[m, k] w[n, k]) + bias[n]) + res[m, n]
// The matrix cores multiply the codes as they are: the 16 x 16 sums of a block start from zero, and one multiply-add a value adds them,
// scaled, to the result's sums in 32 bits.
#include "blocks.hpp"
#include "stream.hpp"

namespace adder {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct CodesArgs : ProductArgs {
    const float *xs, *ws;
    int blocks;   // of K
};

// A lane's 32 codes of a row as an operand, and a block's sums of the products of two.  The 8-bit instructions line their products up with the
// largest and keep some 14 bits of it: 1.6e-5 off, a hundredth of what rounding to bfloat16 changes.  A float32 result has the products of the
// codes as bfloat16, exact and summed in 32 bits, at half the rate.
template <class T>
struct Operand {
    i32x8 codes;
    __device__ __forceinline__ void set(const i32x8 &u) { codes = u; }
};
template <>
struct Operand<float> {
    bf16x8 values[4];
    __device__ __forceinline__ void set(const i32x8 &u) {
        typedef __bf16 pair __attribute__((ext_vector_type(2)));
        struct Eight { pair p[4]; };
#pragma unroll
        for (int i = 0; i < 4; ++i)
            values[i] = __builtin_bit_cast(bf16x8, Eight{{__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)u[2 * i], 1.f, false),
                                                          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)u[2 * i], 1.f, true),
                                                          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)u[2 * i + 1], 1.f, false),
                                                          __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)u[2 * i + 1], 1.f, true)}});
    }
};
__device__ __forceinline__ f32x4 block_sums(const Operand<bf16_t> &b, const Operand<bf16_t> &a) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.codes, a.codes, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);   // (both e4m3, no scales of its own)
}
__device__ __forceinline__ f32x4 block_sums(const Operand<float> &b, const Operand<float> &a) {
    f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.values[i], a.values[i], t, 0, 0, 0);
    return t;
}
// the first `valid` of sixteen codes; zeros in place of the others, whatever they are
__device__ __forceinline__ i32x4 keep_codes(i32x4 u, long valid) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const long left = valid - 4 * j;
        u[j] &= left >= 4 ? -1 : left <= 0 ? 0 : (1 << (8 * (int)left)) - 1;
    }
    return u;
}
__device__ __forceinline__ i32x8 join(const i32x4 &lo, const i32x4 &hi) {
    struct Both { i32x4 lo, hi; };
    return __builtin_bit_cast(i32x8, Both{lo, hi});
}

// ---- tiles that stream through LDS ------------------------------------------------------------------------------------------
// As the bfloat16 products' (linear_stream.hip), a tile's row being a block of 128 bytes.  8192 x 4096 to 4096 and a shortcut 153 us, 1800 TFLOP/s: 64
// steps of some 2.07 us a compute unit.  Nothing is busy all that time: a step's 24 reads of 1 KB a wave out of LDS alone take 0.35 us (4.6 cycles each), its products alone
// 1.05 (0.88 on zeros, for which the card keeps its clock), both with the multiply-adds and a barrier 1.33.  The rest is waiting, behind the barrier that all waves
// leave together, for the next block's loads and, once they are there, for the first operands (without 14 of the 24 reads it takes 133 us, without the
// multiply-adds 152, without the loads behind the first 128; further reads ahead, tiles that follow each other in one workgroup, and a higher
// priority for waves that multiply changed nothing).  With every stage come the scales of the tile's
// rows and columns, a float each, by one load more a wave.  A lane's 32 codes of a row are its chunks q and q + 4 (q = lane / 16): the
// instruction adds the products of all 128, so any order does that is the same for both operands.
__device__ __forceinline__ void stream4(const i32x4 &d, unsigned offset, unsigned to) {   // 4 bytes a lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "memory", "m0");
}

template <class T, int WM, int WN, int TM, int TN, int STAGES>
__global__ __launch_bounds__(WM *WN * 64, 2) void codes_stream_kernel(const CodesArgs p) {
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    typedef Stream<BM, 64, false, WAVES> SA;   // (rows of 64 bfloat16, or 128 codes)
    typedef Stream<BN, 64, false, WAVES> SB;
    constexpr int SCALES = SA::bytes + SB::bytes, STAGE = SCALES + (BM + BN) * 4, LOADS = SA::loads + SB::loads + 1;
    static_assert((BM + BN) / 64 <= WAVES && 128 % (TN * 16) == 0, "a wave's load of scales; a wave's columns share theirs");
    extern __shared__ __align__(1024) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave % WM) * TM * 16, wn = (wave / WM) * TN * 16;
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const long k_begin = blockIdx.y * p.k_share, k_end = k_begin + p.k_share < p.K ? k_begin + p.k_share : p.K;   // (shares of whole blocks)
    const char *a = static_cast<const char *>(p.a) + m0 * p.lda + k_begin, *b = static_cast<const char *>(p.b) + n0 * p.ldb + k_begin;
    long left_a = (p.M - 1 - m0) * p.lda + p.K - k_begin, left_b = (p.N - 1 - n0) * p.ldb + p.K - k_begin;
    SA sa;
    SB sb;
    sa.setup(p.lda / 2, wave, lane);
    sb.setup(p.ldb / 2, wave, lane);
    // this wave's load of scales: of 64 rows, or of 64 columns
    const int part = wave % ((BM + BN) / 64);
    const bool rows = part < BM / 64;
    const long first = rows ? m0 * p.blocks : 0, all = (rows ? p.M : (p.N + kCodeBlock - 1) / kCodeBlock) * p.blocks;
    const char *scales = reinterpret_cast<const char *>((rows ? p.xs : p.ws) + first + k_begin / kCodeBlock);
    long left_s = (all - first - k_begin / kCodeBlock) * 4;
    const unsigned offset_s = (unsigned)(rows ? (part * 64 + lane) * (long)p.blocks * 4 : (n0 + (part - BM / 64) * 64 + lane) / kCodeBlock * p.blocks * 4);
    const int steps = (int)((k_end - k_begin + kCodeBlock - 1) / kCodeBlock);
    const unsigned at_lds = (unsigned)(size_t)(__attribute__((address_space(3))) char *)lds;
    int next = 0;   // the stage's buffer that the next loads go to
    auto load = [&]() {
        sa.load(descriptor(a, left_a), at_lds + next * STAGE, wave);
        sb.load(descriptor(b, left_b), at_lds + next * STAGE + SA::bytes, wave);
        stream4(descriptor(scales, left_s), offset_s, at_lds + next * STAGE + SCALES + part * 256);
        a += kCodeBlock;
        b += kCodeBlock;
        scales += 4;
        left_a -= kCodeBlock;
        left_b -= kCodeBlock;
        left_s -= 4;
        next = next + 1 == STAGES ? 0 : next + 1;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load();
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int buf = 0;
    auto multiply = [&](auto masked, long k0) {
        const char *ta = lds + buf * STAGE, *tb = ta + SA::bytes;
        const float *xs = reinterpret_cast<const float *>(ta + SCALES) + wm + (lane & 15);
        const float by = reinterpret_cast<const float *>(ta + SCALES)[BM + wn];
        Operand<T> fb[TN];
        float s[TM];
        const auto fragment = [&](const char *tile, int at) {
            i32x4 lo = __builtin_bit_cast(i32x4, SA::Tile::fragment(tile, at, 0, lane)), hi = __builtin_bit_cast(i32x4, SA::Tile::fragment(tile, at, 32, lane));
            if constexpr (decltype(masked)::value) {
                const long valid = k_end - k0 - (lane >> 4) * 16;
                lo = keep_codes(lo, valid);
                hi = keep_codes(hi, valid - 64);
            }
            return join(lo, hi);
        };
        Operand<T> fa[2];
        f32x4 t[2][TN];
        const auto add = [&](int i, int j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(t[i & 1][j][e], s[i], acc[i][j][e]);
        };
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[j].set(fragment(tb, wn + j * 16));
        fa[0].set(fragment(ta, wm));
#pragma unroll
        for (int i = 0; i < TM; ++i) s[i] = xs[i * 16] * by;
        // A row of tiles is multiplied while the one before it is scaled and the next one's operand is read, in this order
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if (i + 1 < TM) fa[(i + 1) & 1].set(fragment(ta, wm + (i + 1) * 16));
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                __builtin_amdgcn_sched_barrier(0);
                t[i & 1][j] = block_sums(fb[j], fa[i & 1]);
                if (i > 0) add(i - 1, j);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) add(TM - 1, j);
    };
    const int full = (int)((k_end - k_begin) / kCodeBlock);
    for (int s = 0; s < full; ++s) {
        arrive<(STAGES - 2) * LOADS>();
        load();   // (past the end: descriptors of no bytes; the count of loads under way stays the same)
        multiply(Flag<false>{}, 0);
        buf = buf + 1 == STAGES ? 0 : buf + 1;
    }
    if (full < steps) {
        arrive<(STAGES - 2) * LOADS>();
        multiply(Flag<true>{}, k_begin + (long)full * kCodeBlock);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load into LDS outlives the workgroup)
    finish_wave<T, false, TM, TN>(p, acc, m0 + wm, n0 + wn, lane);
}

template <class T, int WM, int WN, int TM, int TN, int STAGES>
static int launch_stream(CodesArgs p, hipStream_t s) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16, bytes = (BM + BN) * (kCodeBlock + 4) * STAGES;
    p.tiles_m = (int)ceil_div_l(p.M, BM);
    p.tiles_n = (int)ceil_div_l(p.N, BN);
    if (int rc = allow_dynamic_lds<&codes_stream_kernel<T, WM, WN, TM, TN, STAGES>>(bytes)) return rc;
    hipLaunchKernelGGL((codes_stream_kernel<T, WM, WN, TM, TN, STAGES>), dim3((unsigned)p.tiles_m * p.tiles_n, p.splits), dim3(WM * WN * 64), bytes, s, p);
    return check_launch();
}

// ---- few rows of x: the time is that of reading w -------------------------------------------------------------------------
// As the other layers' (linear_rows.hip): sixteen rows of w and up to 16 MT rows of x a workgroup, whose waves take turns along the blocks
// of k, straight from memory, and add their sums through LDS.  Any strides and alignment.  One row, 4096 to 8192: 9.4 us (3.6 TB/s), of which launch, one
// way to memory and back, and the waves' sums are some 4; sixteen waves, or four blocks of each under way, take as long.
static constexpr int kCodesWaves = 8;
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ i32x4 load_codes(const uint8_t *p) { return *reinterpret_cast<const i32x4_any *>(p); }
__device__ __forceinline__ i32x4 load_codes_part(const uint8_t *p, long valid) {
    if (valid >= 16) return load_codes(p);
    i32x4 u = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 15; ++e)
        if (e < valid) u[e / 4] |= (int)p[e] << (8 * (e & 3));
    return u;
}

template <class T, int MT>
__global__ __launch_bounds__(kCodesWaves * 64) void codes_rows_kernel(const CodesArgs p) {
    constexpr int U = MT == 1 ? 2 : 1;   // blocks that a wave multiplies while as many arrive
    extern __shared__ __align__(16) char lds[];
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, l16 = lane & 15, mine = (lane >> 4) * 16;
    const long n0 = (long)blockIdx.x * 16, m0 = (long)blockIdx.y * (16 * MT);
    // (rows past the last: that one again; their results are not stored)
    const uint8_t *pb = static_cast<const uint8_t *>(p.b) + (n0 + l16 < p.N ? n0 + l16 : p.N - 1) * p.ldb + mine, *pa[MT];
    const float *xs[MT], *ws = p.ws + n0 / kCodeBlock * p.blocks;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long m = m0 + i * 16 + l16 < p.M ? m0 + i * 16 + l16 : p.M - 1;
        pa[i] = static_cast<const uint8_t *>(p.a) + m * p.lda + mine;
        xs[i] = p.xs + m * p.blocks;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct Blocks {
        i32x4 b[U][2], a[U][MT][2];
        float xs[U][MT], ws[U];
    };
    auto load = [&](Blocks &t, long kb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long at = kb + u * waves, k = at * kCodeBlock;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                t.b[u][h] = load_codes(pb + k + h * 64);
#pragma unroll
                for (int i = 0; i < MT; ++i) t.a[u][i][h] = load_codes(pa[i] + k + h * 64);
            }
            t.ws[u] = ws[at];
#pragma unroll
            for (int i = 0; i < MT; ++i) t.xs[u][i] = xs[i][at];
        }
    };
    auto add_one = [&](f32x4 &to, const i32x8 &b, const i32x8 &a, float by) {
        Operand<T> u, v;
        u.set(b);
        v.set(a);
        const f32x4 t = block_sums(u, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = fmaf(t[e], by, to[e]);
    };
    auto add = [&](const Blocks &t) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) add_one(acc[i], join(t.b[u][0], t.b[u][1]), join(t.a[u][i][0], t.a[u][i][1]), t.xs[u][i] * t.ws[u]);
    };
    const long whole = p.K / kCodeBlock, turn = U * waves, last = whole - (U - 1) * waves;   // (a turn begins below `last`)
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
    for (; kb * kCodeBlock < p.K; kb += waves) {
        const long k = kb * kCodeBlock, left = p.K - k - mine;
        const i32x8 b = join(load_codes_part(pb + k, left), load_codes_part(pb + k + 64, left - 64));
#pragma unroll
        for (int i = 0; i < MT; ++i) add_one(acc[i], b, join(load_codes_part(pa[i] + k, left), load_codes_part(pa[i] + k + 64, left - 64)), xs[i][kb] * ws[kb]);
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
static int launch_rows(const CodesArgs &p, hipStream_t s) {
    const int waves = p.blocks < kCodesWaves ? p.blocks : kCodesWaves;
    hipLaunchKernelGGL((codes_rows_kernel<T, MT>), dim3((unsigned)ceil_div_l(p.N, 16), (unsigned)ceil_div_l(p.M, 16 * MT)), dim3(waves * 64),
                       waves * MT * 1024, s, p);
    return check_launch();
}

// ---- operands whose rows are not 16 aligned bytes: copies that are, one or both in a launch ------------------------------------
struct AlignArgs {
    const uint8_t *from[2];
    uint4 *to[2];
    long ld[2], chunks_of[2];   // chunks_of: all of an operand's, none where it is aligned
    int K, chunks;              // chunks: a row's
};
__global__ __launch_bounds__(256) void align_codes_kernel(const AlignArgs p) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < p.chunks_of[0] + p.chunks_of[1]; i += (long)gridDim.x * 256) {
        const int o = i >= p.chunks_of[0];
        const long c = o ? i - p.chunks_of[0] : i, row = c / p.chunks;
        const int at = (int)(c - row * p.chunks) * 16;
        const i32x4 u = load_codes_part((o ? p.from[1] : p.from[0]) + row * (o ? p.ld[1] : p.ld[0]) + at, p.K - at);
        (o ? p.to[1] : p.to[0])[c] = make_uint4((uint32_t)u[0], (uint32_t)u[1], (uint32_t)u[2], (uint32_t)u[3]);
    }
}
static long padded(long K) { return (K + 15) & ~15L; }
static size_t copy_bytes(long rows, long K) { return ((size_t)rows * padded(K) + 255) & ~(size_t)255; }

// ---- which kernel ---------------------------------------------------------------------------------------------------------------
// (the estimate: product.hpp; a step is a block of 128 values of k.  Measured as 8192 x 4096 -> 4096, 8192 x 1024 -> 8192 and, alone, as 64 and 128
// workgroups.  256 x 256 results of float32 would not fit the registers beside their operands.)
template <class T>
static constexpr Shape kCodesShapes[] = {   // 8192 x 4096 -> 4096, TFLOP/s
    {128, 128, 2, 2.f, 1.1f, 4.f},          //  886
    {64, 64, 2, 0.755f, 0.5f, 1.9f},        //  653
};
template <>
constexpr Shape kCodesShapes<bf16_t>[] = {
    {128, 128, 2, 1.3f, 0.655f, 3.25f},     // 1501
    {64, 64, 2, 0.6f, 0.33f, 1.6f},         //  817
    {256, 256, 1, 2.07f, 2.07f, 5.9f},      // 1864
};
// The kernel for few rows likewise: workgroups of 16 columns whose waves take turns along the blocks of k, us each; more rows of x are more to read
// from the second-level caches (one row, 4096 to 4096, 8192 to 8192 and 8192 to 1024: 6.6, 16.6, 7.9 us, the small tiles 9.9, 18.7, 8.7; sixteen
// rows 8.3, 25, 12.4 and 10.3, 19.9, 9.2).  With 33 to 64 rows it was behind them (64 x 4096 -> 4096 in 16.5 us instead of 11.4).
static constexpr long kCodesRowsMost = 32;
static float codes_rows_us(long M, long N, long K) {
    const float groups = (float)ceil_div_l(N, 16), turns = (float)ceil_div_l(ceil_div_l(K, kCodeBlock), kCodesWaves);
    return 3.f + ceilf(groups / kCUs) * (0.75f + turns * (0.72f + 0.035f * (float)M));
}
// The one choice that a launch and the queries make; shape -1: the kernel for few rows
template <class T>
static ProductPlan plan_codes(long M, long N, long K) {
    const ProductPlan plan = plan_product(kCodesShapes<T>, kCodeBlock, M, N, K, 1);
    return M <= kCodesRowsMost && codes_rows_us(M, N, K) < plan.us ? ProductPlan{-1, 1, K, 0.f} : plan;
}
static size_t split_bytes(const ProductPlan &plan, long M, long N) { return plan.splits > 1 ? (sizeof(float) * (size_t)plan.splits * M * N + 255) & ~(size_t)255 : 0; }

template <class T>
size_t codes_product_workspace_bytes(long M, long N, long K, bool x_aligned, bool w_aligned) {
    const ProductPlan plan = plan_codes<T>(M, N, K);
    if (plan.shape < 0) return 0;
    return split_bytes(plan, M, N) + (x_aligned ? 0 : copy_bytes(M, K)) + (w_aligned ? 0 : copy_bytes(N, K));
}

template <class T>
int codes_product_kernel(long M, long N, long K) {
    const ProductPlan plan = plan_codes<T>(M, N, K);
    if (plan.shape < 0) return 10000 + 100 * (M <= 16 ? 1 : 2) + 1;
    return 20000 + 100 * plan.shape + plan.splits;
}

template <class T>
int launch_codes_product(const CodesProduct &q, void *ws, hipStream_t s) {
    CodesArgs p{};
    p.a = q.x; p.b = q.w; p.bias = q.bias; p.res = q.res; p.out = q.out;
    p.lda = q.ldx; p.ldb = q.ldw; p.ldr = q.ldr;
    p.M = q.M; p.N = q.N; p.K = q.K;
    p.splits = 1;
    p.act = q.act;
    p.xs = q.xs; p.ws = q.ws;
    p.blocks = (int)ceil_div_l(q.K, kCodeBlock);
    const ProductPlan plan = plan_codes<T>(q.M, q.N, q.K);
    if (plan.shape < 0) return q.M <= 16 ? launch_rows<T, 1>(p, s) : launch_rows<T, 2>(p, s);
    char *at = static_cast<char *>(ws);
    p.part = reinterpret_cast<float *>(at);
    at += split_bytes(plan, q.M, q.N);
    p.splits = plan.splits;
    p.k_share = plan.k_share;
    AlignArgs g{{}, {}, {}, {}, (int)q.K, (int)(padded(q.K) / 16)};
    const auto align = [&](int i, const void *&from, long &ld, long rows) {
        if (!((reinterpret_cast<uintptr_t>(from) | (uintptr_t)ld) & 15)) return;
        g.from[i] = static_cast<const uint8_t *>(from);
        g.ld[i] = ld;
        g.to[i] = reinterpret_cast<uint4 *>(at);
        g.chunks_of[i] = rows * g.chunks;
        from = at;
        ld = padded(q.K);
        at += copy_bytes(rows, q.K);
    };
    align(0, p.a, p.lda, q.M);
    align(1, p.b, p.ldb, q.N);
    if (const long all = g.chunks_of[0] + g.chunks_of[1]) {
        const long groups = ceil_div_l(all, 256);
        hipLaunchKernelGGL(align_codes_kernel, dim3((unsigned)(groups < 16384 ? groups : 16384)), dim3(256), 0, s, g);
        if (int rc = check_launch()) return rc;
    }
    int rc = ADDER_ERR_UNSUPPORTED;
    if (plan.shape == 0) rc = launch_stream<T, 2, 2, 4, 4, 2>(p, s);
    else if (plan.shape == 1) rc = launch_stream<T, 2, 2, 2, 2, 4>(p, s);
    else if constexpr (sizeof(T) == 2) rc = launch_stream<T, 2, 4, 8, 4, 2>(p, s);
    if (rc || plan.splits == 1) return rc;
    return launch_product_join<T>(p, s);
}
#define ADDER_CODES_PRODUCT_INSTANCE(T)                                                     \
    template size_t codes_product_workspace_bytes<T>(long, long, long, bool, bool);          \
    template int codes_product_kernel<T>(long, long, long);                                  \
    template int launch_codes_product<T>(const CodesProduct &, void *, hipStream_t);
ADDER_CODES_PRODUCT_INSTANCE(float)
ADDER_CODES_PRODUCT_INSTANCE(bf16_t)

}  // namespace adder
