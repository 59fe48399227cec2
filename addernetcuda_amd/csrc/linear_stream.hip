// The linear layers' products of large aligned bfloat16 operands.
#include "stream.hpp"

namespace adder {

// ---- tiles that stream through LDS ----------------------------------------------------------------------------------
// A workgroup of WM x WN waves computes BM x BN results, a wave TM x TN tiles of 16 x 16.  The operands' tiles of BK values of k go
// from memory to LDS without passing through registers, STAGES of them in flight: a wave waits for its own loads of the oldest
// stage, the barrier makes that every wave's, and behind it the buffer read last is free for the next loads.  One barrier a
// stage, and no wait for loads that are under way.
//
// The matrix cores decide, with what the LDS reads leave them: 8192 x 4096 to 1024 values and a residual 62.9 us, 1093 TFLOP/s, the matrix
// cores busy for 61 % of the cycles (the rates of all shapes stand beside the choice among them).  8192 x 1024 to 4096 with a GELU and the
// values before it as a second output takes 97 us: 51 for the products, the rest for 17 vector instructions a result and 134 MB of
// stores, which two workgroups a compute unit overlap in part; to start them apart from each other changed nothing.
//
// A load instruction of a wave fills 1024 consecutive bytes of LDS, 16 a lane: the lanes fetch the chunks in the order in which the
// tile keeps them.  Loads past a tensor's end return nothing: the buffer descriptor ends with the tensor, or with the word that its last value
// shares (a word that reaches beyond the end is not loaded at all; what lies beside the value in it belongs to a column that is not stored).
// What lies past a row's end (k beyond K in the last tile) is masked in registers, results of rows past M or N are not stored.
// the first `valid` of eight values; zeros in place of the others, whatever they are
__device__ __forceinline__ bf16x8 keep_first(const bf16x8 &v, int valid) {
    i32x4 u = __builtin_bit_cast(i32x4, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] &= valid >= 2 * j + 2 ? -1 : valid == 2 * j + 1 ? 0xffff : 0;
    return __builtin_bit_cast(bf16x8, u);
}

template <int WM, int WN, int TM, int TN, int BK, int STAGES, bool AA, bool BA, bool GATED, int OCC>
__global__ __launch_bounds__(WM *WN * 64, OCC) void product_stream_kernel(const ProductArgs p) {
    constexpr int WAVES = WM * WN, BM = WM * TM * 16, BN = WN * TN * 16;
    typedef Stream<BM, BK, AA, WAVES> SA;
    typedef Stream<BN, BK, BA, WAVES, GATED> SB;
    static_assert(!GATED || (!AA && !BA), "gated: a forward's product");
    constexpr int STAGE = SA::bytes + SB::bytes, LOADS = SA::loads + SB::loads;
    extern __shared__ __align__(1024) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave % WM) * TM * 16, wn = (wave / WM) * TN * 16;
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const long m0 = (long)tm * BM, n0 = (long)tn * BN;
    const long k_begin = blockIdx.y * p.k_share, k_end = k_begin + p.k_share < p.K ? k_begin + p.k_share : p.K;
    const long step_a = AA ? p.lda * BK * 2 : BK * 2, step_b = BA ? p.ldb * BK * 2 : BK * 2;
    // from the tile's first value to the tensor's end
    const char *a = static_cast<const char *>(p.a), *b = static_cast<const char *>(p.b);
    const long from_a = (AA ? k_begin * p.lda + m0 : m0 * p.lda + k_begin) * 2, from_b = (BA ? k_begin * p.ldb + n0 : (GATED ? n0 / 2 : n0) * p.ldb + k_begin) * 2;
    long left_a = (AA ? (p.K - 1) * p.lda + p.M : (p.M - 1) * p.lda + p.K) * 2 - from_a;
    long left_b = (BA ? (p.K - 1) * p.ldb + p.N : ((GATED ? 2 * p.half : p.N) - 1) * p.ldb + p.K) * 2 - from_b;
    a += from_a;
    b += from_b;
    SA sa;
    SB sb;
    sa.setup(p.lda, wave, lane);
    sb.setup(p.ldb, wave, lane, p.half);
    const int steps = (int)((k_end - k_begin + BK - 1) / BK);
    const unsigned at_lds = (unsigned)(size_t)(__attribute__((address_space(3))) char *)lds;
    int next = 0;   // the stage's buffer that the next loads go to
    auto load = [&]() {
        sa.load(descriptor(a, left_a), at_lds + next * STAGE, wave);
        sb.load(descriptor(b, left_b), at_lds + next * STAGE + SA::bytes, wave);
        a += step_a;
        b += step_b;
        left_a -= step_a;
        left_b -= step_b;
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
#pragma unroll
        for (int k = 0; k < BK; k += 32) {
            bf16x8 fa[TM], fb[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[j] = SB::Tile::fragment(tb, wn + j * 16, k, lane);
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[i] = SA::Tile::fragment(ta, wm + i * 16, k, lane);
            if constexpr (decltype(masked)::value) {
                const long at = k_end - k0 - k - (lane >> 4) * 8;
                const int valid = at < 0 ? 0 : at < 8 ? (int)at : 8;
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[j] = keep_first(fb[j], valid);
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[i] = keep_first(fa[i], valid);
            }
            // (with two stages a wave that multiplies goes before those that read: 2 to 3 % at 8192^3; with more it lost as much)
            if constexpr (STAGES == 2) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
            if constexpr (STAGES == 2) __builtin_amdgcn_s_setprio(0);
        }
    };
    const int full = (int)((k_end - k_begin) / BK);
    for (int s = 0; s < full; ++s) {
        arrive<(STAGES - 2) * LOADS>();
        load();   // (past the end: descriptors of no bytes; the count of loads under way stays the same)
        multiply(Flag<false>{}, 0);
        buf = buf + 1 == STAGES ? 0 : buf + 1;
    }
    if (full < steps) {
        arrive<(STAGES - 2) * LOADS>();
        multiply(Flag<true>{}, k_begin + (long)full * BK);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load into LDS outlives the workgroup)
    finish_wave<bf16_t, GATED, TM, TN>(p, acc, m0 + wm, n0 + wn, lane);
}

template <int WM, int WN, int TM, int TN, int BK, int STAGES, bool AA, bool BA, bool GATED>
static int launch_stream(ProductArgs p, hipStream_t s) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16, bytes = (BM + BN) * BK * 2 * STAGES;
    p.tiles_m = (int)ceil_div_l(p.M, BM);
    p.tiles_n = (int)ceil_div_l(p.N, BN);
    if (int rc = allow_dynamic_lds<&product_stream_kernel<WM, WN, TM, TN, BK, STAGES, AA, BA, GATED, 2>>(bytes)) return rc;
    hipLaunchKernelGGL((product_stream_kernel<WM, WN, TM, TN, BK, STAGES, AA, BA, GATED, 2>), dim3((unsigned)p.tiles_m * p.tiles_n, p.splits),
                       dim3(WM * WN * 64), bytes, s, p);
    return check_launch();
}
template <bool AA, bool BA, bool GATED>
static int launch_stream_shape(const ProductArgs &p, StreamShape shape, hipStream_t s) {
    switch (shape) {
        case StreamShape::big: return launch_stream<2, 4, 8, 4, 64, 2, AA, BA, GATED>(p, s);
        case StreamShape::wide: return launch_stream<2, 4, 4, 4, 64, 3, AA, BA, GATED>(p, s);
        case StreamShape::mid: return launch_stream<2, 2, 4, 4, 64, 2, AA, BA, GATED>(p, s);
        default: return launch_stream<2, 2, 2, 2, 64, 4, AA, BA, GATED>(p, s);
    }
}
int launch_product_stream(ProductArgs p, bool a_across, bool b_across, StreamShape shape, hipStream_t s) {
    if (p.half) return launch_stream_shape<false, false, true>(p, shape, s);
    if (!a_across && !b_across) return launch_stream_shape<false, false, false>(p, shape, s);
    return a_across ? launch_stream_shape<true, true, false>(p, shape, s) : launch_stream_shape<false, true, false>(p, shape, s);
}

}  // namespace adder
