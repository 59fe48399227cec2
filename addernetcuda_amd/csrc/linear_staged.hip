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
//
// 8192 x 1024 x 4096: 312 us, 220 TFLOP/s (float32 matrix instructions: 155 at their best); 1024^3 20 us, 105 TFLOP/s; 1531 x 515 x 1027 22 us.
// Where the tiles fill the card, LDS bounds it: 32 values of k of a 64 x 64 tile are 24 KB written and 48 KB read, 576 cycles, beside
// 384 of the matrix cores and 350 of the splitting; where they do not, each of those waits for the other.
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

// One operand's tile: loads of 16 bytes, of 4 floats or 8 bfloat16 that lie side by side.  The loads of the main loop have no branch
// around them (a wait behind one would have to be for all that is under way): rows and columns that do not exist are other ones
// again, whose results are not stored; with k across the rows, the chunk that ends beyond the last column is read as the last whole
// chunk and shifted on its way to LDS (EDGE; below a chunk's columns: NARROW, no main loop).  Only the last tile of a k that is no whole
// number of tiles holds zeros, and is read on its own.
template <class T, int R, bool ACROSS, int THREADS, bool GATED = false>
struct Staged {
    static constexpr int E = Chunk<T>::n, BK = kStagedK<T>, P = kStagedPlanes<T>;
    typedef LdsTile<R, BK, ACROSS> Tile;
    static constexpr int row_loads = Tile::row_chunks * 8 / E, per = R * BK / E / THREADS;
    struct Values { uint4 v[per]; };
    const T *at[per];   // of the next tile
    int shift[per];     // across: how many columns before its place a chunk was read
    long step;

    // chunk i of this thread: its row (across: of k) and its first column (along: of k) in the tile
    static __device__ __forceinline__ int row_of(int i) { return (threadIdx.x % THREADS + i * THREADS) / row_loads; }
    static __device__ __forceinline__ int column_of(int i) { return (threadIdx.x % THREADS + i * THREADS) % row_loads * E; }
    static __device__ __forceinline__ bool edge(long all, long row0) { return ACROSS && row0 + R > all; }
    static __device__ __forceinline__ bool narrow(long all) { return ACROSS && all < E; }

    __device__ __forceinline__ void setup(const T *p, long ld, long all, long row0, long k_begin, long half = 0) {
        step = ACROSS ? BK * ld : BK;
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int r = row_of(i), c = column_of(i);
            if constexpr (ACROSS) {
                const long col = row0 + c + E <= all ? row0 + c : all - E;
                at[i] = p + (k_begin + r) * ld + col;
                shift[i] = row0 + c < all ? (int)(row0 + c - col) : 0;
            } else {
                at[i] = p + (GATED ? gated_row(row0 + r, half) : row0 + r < all ? row0 + r : all - 1) * ld + k_begin + c;
            }
        }
    }
    __device__ __forceinline__ void load(Values &t, bool more) {
#pragma unroll
        for (int i = 0; i < per; ++i) t.v[i] = load_raw(at[i]);
        const long go = more ? step : 0;   // (past the last whole tile: that one again, unused)
#pragma unroll
        for (int i = 0; i < per; ++i) at[i] += go;
    }
    // the tile from k on, of which `left` values of k exist
    static __device__ __forceinline__ void load_last(Values &t, const T *p, long ld, long all, long row0, long k, int left, long half = 0) {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int r = row_of(i), c = column_of(i);
            const long rows = all - row0 - (ACROSS ? c : r);
            if constexpr (ACROSS) t.v[i] = load_raw_part(p + (k + r) * ld + row0 + c, r >= left || rows <= 0 ? 0 : rows < E ? (int)rows : E);
            else if constexpr (GATED) t.v[i] = load_raw_part(p + gated_row(row0 + r, half) * ld + k + c, gated_exists(row0 + r, half) ? left - c : 0);
            else t.v[i] = load_raw_part(p + (row0 + r) * ld + k + c, rows <= 0 ? 0 : left - c);
        }
    }
    static __device__ __forceinline__ uint4 shifted(uint4 v, int by) {   // values by.. in the first places
        if constexpr (E == 8) {
            v.x = by & 1 ? (v.x >> 16) | (v.y << 16) : v.x;
            v.y = by & 1 ? (v.y >> 16) | (v.z << 16) : v.y;
            v.z = by & 1 ? (v.z >> 16) | (v.w << 16) : v.z;
            v.w = by & 1 ? v.w >> 16 : v.w;
            by >>= 1;
        }
        if (by & 1) v = make_uint4(v.y, v.z, v.w, v.w);
        if (by & 2) v = make_uint4(v.z, v.w, v.w, v.w);
        return v;
    }
    template <bool EDGE>
    __device__ __forceinline__ void store(char *tile, Values t) const {
        if constexpr (EDGE && ACROSS)
#pragma unroll
            for (int i = 0; i < per; ++i) t.v[i] = shifted(t.v[i], shift[i]);
        put(tile, t);
    }
    static __device__ __forceinline__ void put(char *tile, const Values &t) {
#pragma unroll
        for (int i = 0; i < per; ++i) {
            const int r = row_of(i), c = column_of(i) / E;
            if constexpr (P == 1) {
                *reinterpret_cast<uint4 *>(tile + r * Tile::row_bytes + (Tile::place(r, c) << 4)) = t.v[i];
            } else {
                uint32_t a[3], b[3];
                split(__uint_as_float(t.v[i].x), __uint_as_float(t.v[i].y), a);
                split(__uint_as_float(t.v[i].z), __uint_as_float(t.v[i].w), b);
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
template <int TM, int TN, bool AA, bool BA, bool GATED>
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
            if constexpr (GATED) fb[j] = k < k_end && gated_exists(n, p.half) ? b[gated_row(n, p.half) * p.ldb + k] : 0.f;
            else fb[j] = k < k_end && n < p.N ? b[BA ? k * p.ldb + n : n * p.ldb + k] : 0.f;
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

// WM x WN waves of TM x TN tiles of 16 x 16.  AHEAD: tiles of k in registers or on their way there (small ones are multiplied faster than the
// next arrives).  BUFFERS = 2: one barrier a tile, and the next is split and stored while this one is multiplied.  KG: groups of so many
// waves that share the tiles of k, each with buffers of its own; their sums are added through LDS.
template <class T, int WM, int WN, int TM, int TN, int AHEAD, int BUFFERS, int KG, bool AA, bool BA, bool GATED>
__global__ __launch_bounds__(WM *WN * 64 * KG, KG == 1 ? 2 : 1) void product_staged_kernel(const ProductArgs p) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16, BK = kStagedK<T>, P = kStagedPlanes<T>, THREADS = WM * WN * 64;
    typedef Staged<T, BM, AA, THREADS> SA;
    typedef Staged<T, BN, BA, THREADS, GATED> SB;
    static_assert(!GATED || (!AA && !BA), "gated: a forward's product");
    constexpr int BYTES = P * (SA::Tile::bytes + SB::Tile::bytes);
    extern __shared__ __align__(16) char all_lds[];
    const int lane = threadIdx.x & 63, wave = (threadIdx.x % THREADS) >> 6, group = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    char *lds = all_lds + group * (BUFFERS * BYTES);
    const int wm = (wave % WM) * (TM * 16), wn = (wave / WM) * (TN * 16);
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
    // One tile.  `between`, the next tile's splitting and stores, runs once the last two rows of matrix instructions are left to hide it (four
    // rows a wave: in front of the first row the gradients of 4096 x 1024 x 4096 took 397 us instead of 345)
    auto multiply = [&](const char *ta, auto between) {
        const char *tb = ta + P * SA::Tile::bytes;
#pragma unroll
        for (int k = 0; k < BK; k += 32) {
            bf16x8 fb[P][TN], fa[2][P];
            auto read = [&](int i) {
#pragma unroll
                for (int q = 0; q < P; ++q) fa[i & 1][q] = SA::Tile::fragment(ta + q * SA::Tile::bytes, wm + i * 16, k, lane);
            };
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[q][j] = SB::Tile::fragment(tb + q * SB::Tile::bytes, wn + j * 16, k, lane);
            read(0);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                if (i + 1 < TM) read(i + 1);
                if (k == 0 && i == TM - 2) between();
#pragma unroll
                for (int u = P == 3 ? 2 : 0; u >= 0; --u)   // (the small products first)
#pragma unroll
                    for (int q = 0; q <= u; ++q)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = mfma(fb[u - q][j], fa[i & 1][q], acc[i][j]);
            }
        }
    };
    const int full = (int)((k_end - k_begin) / BK), left = (int)(k_end - k_begin - (long)full * BK);
    // this group's whole tiles: `mine` of them from `first` on, in `turns` turns of all groups
    const int turns = (full + KG - 1) / KG, first = group * turns < full ? group * turns : full - 1;
    const int mine = full - group * turns < 0 ? 0 : full - group * turns < turns ? full - group * turns : turns;
    auto walk = [&](auto edge) {   // over the whole tiles of k
        constexpr bool EDGE = decltype(edge)::value;
        SA sa;
        SB sb;
        sa.setup(a, p.lda, p.M, m0, k_begin + (long)first * BK);
        sb.setup(b, p.ldb, p.N, n0, k_begin + (long)first * BK, p.half);
        typename SA::Values va[AHEAD];
        typename SB::Values vb[AHEAD];
        int next = 0;
        auto load = [&](int d) {
            ++next;
            sa.load(va[d], next < mine);
            sb.load(vb[d], next < mine);
        };
        auto store = [&](char *tile, int d) {
            sa.template store<EDGE>(tile, va[d]);
            sb.template store<EDGE>(tile + P * SA::Tile::bytes, vb[d]);
        };
#pragma unroll
        for (int d = 0; d < AHEAD; ++d) {
            load(d);
            asm volatile("" ::: "memory");   // (in this order: the loop waits for the oldest)
        }
        if constexpr (BUFFERS == 2) {
            store(lds, 0);
            load(0);
            asm volatile("" ::: "memory");
            int buf = 0;
            for (int t = 0; t < turns; t += AHEAD)
#pragma unroll
                for (int d = 0; d < AHEAD; ++d) {
                    if (t + d >= turns) break;
                    __syncthreads();   // this tile is there; the other buffer has been read
                    if (KG == 1 || t + d < mine)
                        multiply(lds + buf * BYTES, [&]() {
                            store(lds + (buf ^ 1) * BYTES, (d + 1) % AHEAD);
                            load((d + 1) % AHEAD);
                        });
                    buf ^= 1;
                }
        } else {
            for (int t = 0; t < turns; ++t) {
                __syncthreads();
                store(lds, 0);
                __syncthreads();
                load(0);
                multiply(lds, [] {});
            }
        }
    };
    auto single = [&](long k, int left) {   // one tile on its own, by the last group
        typename SA::Values va;
        typename SB::Values vb;
        if (group == KG - 1) {
            SA::load_last(va, a, p.lda, p.M, m0, k, left);
            SB::load_last(vb, b, p.ldb, p.N, n0, k, left, p.half);
        }
        __syncthreads();
        if (group == KG - 1) {
            SA::put(lds, va);
            SB::put(lds + P * SA::Tile::bytes, vb);
        }
        __syncthreads();
        if (group == KG - 1) multiply(lds, [] {});
    };
    if (SA::narrow(p.M) || SB::narrow(p.N)) {
        for (int t = 0; t < full; ++t) single(k_begin + (long)t * BK, BK);
    } else if (full) {
        if (SA::edge(p.M, m0) || SB::edge(p.N, n0)) walk(Flag<true>{});
        else walk(Flag<false>{});
    }
    if (left) single(k_begin + (long)full * BK, left);
    if constexpr (KG > 1) {
        static_assert((KG - 1) * WM * WN * TM * TN * 64 * sizeof(f32x4) <= KG * BUFFERS * BYTES, "the groups' sums fit");
        f32x4 *sums = reinterpret_cast<f32x4 *>(all_lds) + ((group - 1) * WM * WN + wave) * (TM * TN * 64) + lane;
        __syncthreads();
        if (group > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) sums[(i * TN + j) * 64] = acc[i][j];
        }
        __syncthreads();
        if (group > 0) return;
#pragma unroll
        for (int g = 1; g < KG; ++g)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] += sums[(g * WM * WN * TM * TN + i * TN + j) * 64];
    }
    if constexpr (P == 3) {
        bool finite = true;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) finite = finite && fabsf(acc[i][j][e]) < __builtin_inff();
        if (!__all(finite)) sum_again<TM, TN, AA, BA, GATED>(p, acc, m0 + wm, n0 + wn, k_begin, k_end, lane);
    }
    finish_wave<T, GATED, TM, TN>(p, acc, m0 + wm, n0 + wn, lane);
}

template <class T, int WM, int WN, int TM, int TN, int AHEAD, int BUFFERS, int KG, bool AA, bool BA, bool GATED>
static int launch_staged_layout(ProductArgs p, hipStream_t s) {
    constexpr int BM = WM * TM * 16, BN = WN * TN * 16, bytes = KG * BUFFERS * kStagedPlanes<T> * (BM + BN) * kStagedK<T> * 2;
    p.tiles_m = (int)ceil_div_l(p.M, BM);
    p.tiles_n = (int)ceil_div_l(p.N, BN);
    if (int rc = allow_dynamic_lds<&product_staged_kernel<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, AA, BA, GATED>>(bytes)) return rc;
    hipLaunchKernelGGL((product_staged_kernel<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, AA, BA, GATED>), dim3((unsigned)p.tiles_m * p.tiles_n, p.splits),
                       dim3(WM * WN * 64 * KG), bytes, s, p);
    return check_launch();
}
template <class T, int WM, int WN, int TM, int TN, int AHEAD, int BUFFERS, int KG = 1>
static int launch_staged(const ProductArgs &p, bool a_across, bool b_across, hipStream_t s) {
    if (p.half) return launch_staged_layout<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, false, false, true>(p, s);
    if (a_across) return launch_staged_layout<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, true, true, false>(p, s);
    return b_across ? launch_staged_layout<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, false, true, false>(p, s)
                    : launch_staged_layout<T, WM, WN, TM, TN, AHEAD, BUFFERS, KG, false, false, false>(p, s);
}
template <>
int launch_product_staged<float>(const ProductArgs &p, bool a_across, bool b_across, StagedShape shape, hipStream_t s) {
    switch (shape) {
        case StagedShape::large: return launch_staged<float, 2, 2, 4, 4, 1, 1>(p, a_across, b_across, s);
        case StagedShape::small: return launch_staged<float, 2, 2, 2, 2, 3, 2>(p, a_across, b_across, s);
        case StagedShape::alone: return launch_staged<float, 2, 4, 4, 2, 1, 2>(p, a_across, b_across, s);
        default: return launch_staged<float, 2, 2, 2, 2, 3, 2, 2>(p, a_across, b_across, s);
    }
}
template <>
int launch_product_staged<bf16_t>(const ProductArgs &p, bool a_across, bool b_across, StagedShape shape, hipStream_t s) {
    return shape == StagedShape::large ? launch_staged<bf16_t, 2, 2, 4, 4, 1, 1>(p, a_across, b_across, s)
                                       : launch_staged<bf16_t, 2, 2, 2, 2, 3, 2>(p, a_across, b_across, s);
}

}  // namespace adder
