// Index and split arithmetic of the paged 8-bit cache, shared by its kernels and compiled for the host by the tests.
#pragma once
#include <stdint.h>

#ifdef __HIP__
#define IT_HD __host__ __device__ __forceinline__
#else
#define IT_HD inline
#endif

namespace it {
namespace kv8 {

constexpr int PAGE = 64, BLOCK = 16;   // rows of a page, rows that share a scale

// Element of a page and KV head that holds (row, dim), for the codes (bytes) and the open rows (f16) alike. The order is that of
// the matrix operands: a wave's lane l reads 16 codes at 16 l of each KiB.
//   K: KiB (row / 16, dim / 64); lane = 16 (dim / 8 % 4) + row % 16; then two runs of 8 dims, 32 apart
//   V: KiB (dim / 16); lane = 16 (row / 4 % 4) + dim % 16; then four rows of each of the four blocks
IT_HD int k_elem(int hd, int row, int dim) {
    return (((row >> 4) * (hd >> 6) + (dim >> 6)) * 64 + ((dim >> 3) & 3) * 16 + (row & 15)) * 16 + ((dim >> 5) & 1) * 8 +
           (dim & 7);
}
IT_HD int v_elem(int row, int dim) {
    return ((dim >> 4) * 64 + ((row >> 2) & 3) * 16 + (dim & 15)) * 16 + (row >> 4) * 4 + (row & 3);
}

// Pages per split of an attention call: `work` is the sum over sequences and KV heads of row blocks times pages, shared
// out to about `wgs` workgroups; each of the `groups` row blocks may leave one split that is not full, which the count allows
// for while they are few. Half of the workgroups if there is more than a FEW row blocks and they need take no more than SHORT
// pages: those pages are then quicker than the records of twice the splits (us, 16 heads, 2 KV heads, hd 256: 64 tokens after
// 4032 28.4 / 30.0, 12 after 8180 21.2 / 23.1, but the 18 pages of 64 after 8128 36.7 / 33.8, and the four row blocks of 4
// tokens after 8190, 24 heads, 20.0 / 19.4). Between: 11 pages 26.3 / 27.5, 14 29.8 / 30.3, 16 32.7 / 31.9; the two row blocks of a
// token after 8191 12.8 / 12.2. The same in the partial and the merge kernel.
constexpr int FEW = 4, SHORT = 10;
IT_HD float reciprocal(float x) {   // (to a rounding or two; the splits need not be exact, only alike)
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_rcpf(x);
#else
    return 1.0f / x;
#endif
}
IT_HD int pages_each(float work, float groups, float wgs) {
    const float room = wgs - groups, c = work * reciprocal(room < 0.5f * wgs ? 0.5f * wgs : room);
    if (!(c < 33554432.0f)) return 33554432;   // no sequence has more pages
    const int i = (int)c;
    return (float)i < c ? i + 1 : i < 1 ? 1 : i;
}
IT_HD int chunk_pages(float work, float groups, int wgs) {
    if (groups > (float)FEW) {
        const int half = pages_each(work, groups, 0.5f * (float)wgs);
        if (half <= SHORT) return half;
    }
    return pages_each(work, groups, (float)wgs);
}
// Batches rarely leave that much: fewer pages per split, which a call takes if its splits are then no more than wgs (about_splits
// of each row block added up: a count that is off by one where page counts lie near a multiple costs nothing but time).
// 64 sequences of 4096 rows, a token each, 58.3 / 61.5 us, 8 of 32 tokens after 8160 80 / 90.
constexpr int TRIES = 4;
IT_HD int fewer_pages(float work, float groups, int wgs, int k) { return pages_each(work, 0.25f * (float)k * groups, (float)wgs); }
IT_HD float about_splits(int pages, float rcp_chunk) { return __builtin_ceilf((float)pages * rcp_chunk - 0.001f); }
IT_HD int splits(int pages, int chunk) { return (int)(((unsigned)pages + (unsigned)chunk - 1u) / (unsigned)chunk); }   // (both at most 2^25)
// Record of (split, row block, KV head) among a sequence's, and how many blocks of records all split sequences can
// need: splits(p, c) <= 2 p / c where p > c, so at most 2 wgs and what f32 sums round off.
IT_HD int record(int split, int nrb, int rb, int nkv, int kh) { return (split * nrb + rb) * nkv + kh; }
IT_HD int max_records(int wgs) { return 2 * wgs + 16; }

}  // namespace kv8
}  // namespace it
