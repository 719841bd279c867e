// K/V tiles of the 32-row flash forms: 64 rows of 256 f16 straight from memory into LDS, for four waves.
#pragma once
#include "common.h"

namespace it {

constexpr int KV_HD = 256;   // head_dim

// LDS tiles are unpadded 512-byte rows of 32 16-byte chunks; logical chunk j of row r lives at
// physical chunk j ^ swz32(r). With 512-byte rows a chunk's bank group is (chunk mod 16), so swz32
// gives 16 consecutive rows 16 distinct values (K operand reads: one row per lane) and 4
// consecutive rows distinct chunk pairs (V transpose reads: 4 rows x 2 chunks per 16 lanes).
__device__ __forceinline__ int swz32(int r) { return ((r & 3) << 1) | ((r >> 2) & 1) | (((r >> 3) & 1) << 3); }

// Issue the direct-to-LDS loads of one 64-row tile: wave w moves rows 16w..16w+15, two rows
// (64 lanes x 16 bytes) per instruction, each lane fetching the logical chunk that belongs at its
// physical slot. Rows past kend-1 repeat row kend-1 (a tile issued past the end only refetches it).
// Addresses are a uniform row base plus a 32-bit lane offset, so each instruction needs two VALU
// ops; the chunk part of the offsets (cj, including the head's column) is computed once.
struct TileSrc {
    const char* base;   // the tile's first row, clamped
    int rmax;           // last row to read, from there
    unsigned rowb;      // bytes per row
};
__device__ __forceinline__ TileSrc tile_src(const uint16_t* __restrict__ src, int kvd, int kb, int kend) {
    const int ts = min(kb, kend - 1);
    return {(const char*)(src + (size_t)ts * kvd), kend - 1 - ts, 2u * (unsigned)kvd};
}
// load i of the wave's eight
__device__ __forceinline__ void tile_piece32(const TileSrc& t, const int (&cj)[8], _Float16* lds, int w, int l, int i) {
    typedef __attribute__((address_space(3))) void lds_void;
    const int r = 16 * w + 2 * i + (l >> 5);
    const unsigned off = (unsigned)min(r, t.rmax) * t.rowb + (unsigned)cj[i];
    __builtin_amdgcn_global_load_lds((const void*)(t.base + off), (lds_void*)(lds + (16 * w + 2 * i) * KV_HD), 16, 0, 0);
}
__device__ __forceinline__ void tile_to_lds32(const uint16_t* __restrict__ src, int kvd, int kb, int kend,
                                            const int (&cj)[8], _Float16* lds, int w, int l) {
    const TileSrc t = tile_src(src, kvd, kb, kend);
#pragma unroll
    for (int i = 0; i < 8; ++i) tile_piece32(t, cj, lds, w, l, i);
}

// acc *= a for an MFMA accumulator tile held in AGPRs, element by element in place (read to a VGPR,
// multiply, write back). Written out so the accumulators never need a VGPR home: with a plain
// multiply in the (rare) rescale branch the register allocator keeps them in VGPRs at the branch
// merge and the common path copies all of them to VGPRs and back on every tile.
__device__ __forceinline__ void scale_acc(f16v& acc, float a) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x = acc[i], t;
        asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32_e32 %1, %2, %1\n\tv_accvgpr_write_b32 %0, %1"
                     : "+a"(x), "=&v"(t)
                     : "v"(a));
        acc[i] = x;
    }
}

}  // namespace it
