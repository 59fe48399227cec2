// Tiles that go from memory to LDS without passing through registers, for the products whose operands have rows of 16 aligned bytes.
#pragma once
#include "product.hpp"

namespace adder {

struct Descriptor { uint64_t base; uint32_t bytes, flags; };
__device__ __forceinline__ i32x4 descriptor(const char *p, long left) {
    const long words = (left + 3) & ~3L;
    const Descriptor d{reinterpret_cast<uint64_t>(p), left <= 0 ? 0u : words < 0xffffffffL ? (uint32_t)words : 0xffffffffu, 0x00027000u};
    return __builtin_bit_cast(i32x4, d);
}
// 16 bytes a lane from base + offset to the 1024 bytes of LDS at `to` (a wave's); no register is written
__device__ __forceinline__ void stream(const i32x4 &d, unsigned offset, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(offset), "s"(d) : "memory", "m0");
}
// All but the `N` newest loads of this wave done, and its LDS reads; then the workgroup's waves meet.
template <int N>
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One operand's tile: R rows (or columns, with k across) of BK
template <int R, int BK, bool ACROSS, int WAVES, bool GATED = false>
struct Stream {
    typedef LdsTile<R, BK, ACROSS> Tile;
    static constexpr int bytes = Tile::bytes, loads = bytes / 1024 / WAVES;
    static_assert(bytes % (1024 * WAVES) == 0, "whole loads for every wave");
    unsigned offset[loads];

    __device__ __forceinline__ void setup(long ld, int wave, int lane, long half = 0) {
#pragma unroll
        for (int i = 0; i < loads; ++i) {
            const int chunk = (wave * loads + i) * 64 + lane, row = chunk / Tile::row_chunks;   // as it lies in LDS
            const long at = GATED ? (row >> 5) * 16 + (row & 15) + (row & 16 ? half : 0) : row;
            offset[i] = (unsigned)(at * ld * 2 + Tile::place(row, chunk % Tile::row_chunks) * 16);   // (the order is its own inverse)
        }
    }
    __device__ __forceinline__ void load(const i32x4 &d, unsigned to, int wave) const {
#pragma unroll
        for (int i = 0; i < loads; ++i) stream(d, offset[i], to + (wave * loads + i) * 1024);
    }
};

}  // namespace adder
