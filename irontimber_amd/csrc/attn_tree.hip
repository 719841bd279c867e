// Attention of a drafted tree's nodes: every node sees the pos0 context rows, and its own ancestors and
// itself among the tree's rows (cache rows pos0 + j, bit j of anc[t]). The softmax over both sets is a merge:
//   context   no mask at all, so it is split over the keys into the decode partials' records {m, l, o[256]}
//             (kernels/src/lib.rs:753-798), each key read once for all rows of its KV head;
//   own path  at most 64 keys a node, each one's record is {score, 1, V row}: the merge makes them itself,
//             from the path's rows alone. A row that the mask hides is never read, so whatever it holds (an
//             unused row, the infinities of another branch) reaches no output.
// out = sum_i e^(m_i - M) o_i / sum_i e^(m_i - M) l_i * sigmoid(gate), M = max m_i (kernels/src/lib.rs:722-740).
#include <algorithm>
#include <cfloat>

#include "common.h"
#include "internal.h"
#include "kv_tile.h"

namespace it {

namespace {
constexpr int HD = 256;
constexpr int PART = idx::PART;
constexpr int SPL = 8;   // context records a lane loads per batch
constexpr int BM = 64, BN = 64;          // rows per workgroup and keys per tile of the row-block form
constexpr float P_BITS = 7.0f;           // weights up to 2^15 of the reference: see the softmax
constexpr float LN2_F = 0.6931471805599453f;
}  // namespace

// The context's records for many rows or long contexts (plan(), below): workgroup = 64 rows r = t*G + g
// of one KV head x one key split, four waves of 32 rows x half of each 64-key tile's keys: wave w takes rows
// 32 (w & 1) .. +31 and keys 32 (w >> 1) .. +31, with a running maximum, sum and O of its own that are joined at the
// end. The transposed products of the flash form (S^T = K q^T, O^T += V^T P^T, 32x32x16, one query row a lane
// pair), twice each: q (scaled) and P go in as f16 pairs hi + lo, so K and V, exact in f16, meet f32 operands to 2^-22 and the
// f32 records keep f32's accuracy. A tile takes a wave 64 matrix ops of 32 cycles.
// Splitting rows and keys between the waves halves what a wave reads from LDS against four waves of 16 rows: 1024
// cycles of LDS a tile and workgroup beside 2048 of the matrix cores.
// Measured, 64 nodes, 16/2 heads: 131072 keys 236-272 us = 1.01-1.17 PFLOP/s of matrix work (the pairs double the 137.5
// GFLOP of the call; a large f16 product runs at 1.15 here). 2 / 4 / 8 / 16 / 32 / 128 tiles a workgroup take 17.3 / 20.0 / 26.4 /
// 38.7 / 67.7 / 245 us at best: 1.5 us a tile in short runs, 1.85 in long ones, and 14 us beside the tiles (in the workgroup q 2,
// its conversion 1.2, the first tile 2, the join of the key halves 2.4, the records 2; the rest outside it). For its 2,048 cycles
// of matrix ops a tile takes 2,700 cycles in short runs and 3,240 in long ones, where the clock falls to 1.75 GHz; what the
// cycles without a matrix op are is not known (without its loads, exponentials, operand reads or rescaling a tile is 3 %
// shorter each).
__global__ __launch_bounds__(256) void attn_tree_ctx_kernel(const float* __restrict__ q, int qts,
                                                            const uint16_t* __restrict__ kc,
                                                            const uint16_t* __restrict__ vc, int kvd, int n, int nh,
                                                            int nkv, int nt, float scale, float* __restrict__ part,
                                                            int chunk, int smax, int nrb) {
    __shared__ __align__(16) _Float16 K0[BN * HD];
    __shared__ __align__(16) _Float16 K1[BN * HD];
    __shared__ __align__(16) _Float16 V0[BN * HD];
    __shared__ __align__(16) _Float16 V1[BN * HD];
    __shared__ float ms[2][BM], ls[2][BM];   // per key half
    __shared__ f2 rowml[BM];
    __shared__ int rowex[BM];   // power of two that a q row was multiplied with

    // Row blocks of one (split, KV head) read the same keys: their ids differ by multiples of 8, which puts
    // them on one XCD and its L2.
    const int G = nh / nkv, R = nt * G;
    const int grp = (int)blockIdx.x / (8 * nrb) * 8 + (int)blockIdx.x % 8, rb = (int)blockIdx.x / 8 % nrb;
    if (grp >= smax * nkv) return;   // whole workgroup (the id count is rounded up to multiples of 8)
    const int s = grp / nkv, kh = grp % nkv;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, hh = l >> 5, c = l & 31;
    const int wr = w & 1, wk = w >> 1;
    const int kb0 = s * chunk, kend = min(kb0 + chunk, n);
    const size_t head_off = (size_t)kh * HD;
    const float neg1 = in_register(-1.0f);
    int cj[8];   // byte offset of the chunk each lane's tile loads bring, plus the KV head's column
#pragma unroll
    for (int i = 0; i < 8; ++i) cj[i] = 2 * (int)head_off + 16 * ((l & 31) ^ swz32(16 * w + 2 * i + (l >> 5)));

    // ---- q: wave w reads rows 16w .. 16w+15 of the block whole, and the operand layout comes out of hi and lo planes
    // in the second K and V buffers, which the first tile does not use. Rows past R read the last row.
    h8 qh[16], ql[16];
    {
        f4 qx[16];
        const int r0 = min(rb * BM + 16 * w, R - 1);
        const int t0 = __builtin_amdgcn_readfirstlane(r0 / G);
        int g0 = r0 - t0 * G;   // the row's head in its group; its floats start at `at`
        size_t at = uniform_off((size_t)t0 * qts + (size_t)(kh * G + g0) * 2 * HD);
        const int wrap = qts - G * 2 * HD;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            qx[i] = ld_f4(q + at + 4 * l);
            const bool more = r0 + i + 1 < R, last = g0 + 1 == G;
            at += more ? 2 * HD + (last ? wrap : 0) : 0;
            g0 = !more ? g0 : last ? 0 : g0 + 1;
        }
        tile_to_lds32(kc, kvd, kb0, kend, cj, K0, w, l);
        tile_to_lds32(vc, kvd, kb0, kend, cj, V0, w, l);
        // Each row times the power of two that takes its largest value to 2^13 .. 2^14, so that the pairs hold every value to
        // 2^-22 of itself or 2^-39 of the row's largest, whatever q's size. The maxima: rows i and i + 8 in the half-waves, i and
        // i + 4 in their 16-lane rows, then over those 16 lanes.
        float mx[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            mx[i] = fmaxf(fmaxf(fabsf(qx[i][0]), fabsf(qx[i][1])), fmaxf(fabsf(qx[i][2]), fabsf(qx[i][3])));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            swap32(mx[i], mx[i + 8]);
            mx[i] = fmaxf(mx[i], mx[i + 8]);
        }
        int ex[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            swap16(mx[i], mx[i + 4]);
            float m = fmaxf(mx[i], mx[i + 4]);
            m = fmaxf(m, dppc<0xB1>(m));
            m = fmaxf(m, dppc<0x4E>(m));
            m = fmaxf(m, dppc<0x141>(m));
            m = fmaxf(m, dppc<0x140>(m));
            ex[i] = 14 - __builtin_amdgcn_frexp_expf(m);   // of row i + 4 (16-lane row & 1) + 8 (half-wave)
            if ((l & 15) == 0) rowex[16 * w + i + 4 * ((l >> 4) & 1) + 8 * (l >> 5)] = ex[i];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 16 * w + i, e = __builtin_amdgcn_readlane(ex[i & 3], 16 * ((i >> 2) & 1) + 32 * (i >> 3));
            h2 h0, h1, l0, l1;
            split2(f2{__builtin_amdgcn_ldexpf(qx[i][0], e), __builtin_amdgcn_ldexpf(qx[i][1], e)}, neg1, h0, l0);
            split2(f2{__builtin_amdgcn_ldexpf(qx[i][2], e), __builtin_amdgcn_ldexpf(qx[i][3], e)}, neg1, h1, l1);
            const h4 hi = {h0[0], h0[1], h1[0], h1[1]}, lo = {l0[0], l0[1], l1[0], l1[1]};
            const int to = row * HD + 8 * ((l >> 1) ^ (row & 31)) + 4 * (l & 1);
            *(h4*)(K1 + to) = hi;
            *(h4*)(V1 + to) = lo;
        }
        __syncthreads();
#pragma unroll
        for (int ks = 0; ks < 16; ++ks) {
            const int at = (32 * wr + c) * HD + 8 * ((2 * ks + hh) ^ c);
            qh[ks] = ld_h8(K1 + at);
            ql[ks] = ld_h8(V1 + at);
        }
    }
    const float back = __builtin_amdgcn_ldexpf(scale * LOG2E, -rowex[32 * wr + c]);   // from products to log2 units
    f16v o[8];
#pragma unroll
    for (int db = 0; db < 8; ++db) o[db] = f16v{};
    float m_run = -INFINITY, l_run = 0.f;   // log2 units; l over this lane half's keys

    // LDS offsets of the K operand (row 32 wk + c) and of the V transpose reads (rows 32 wk + 16 ks + 4 hh + vrow and 8
    // further), as in the flash form
    int koff[8], voff[4][2];
#pragma unroll
    for (int k2 = 0; k2 < 8; ++k2) koff[k2] = (32 * wk + c) * HD + 8 * ((2 * k2 + hh) ^ swz32(c));
    {
        const int vrow = (l & 15) >> 2, vcol = 16 * ((l >> 4) & 1) + 4 * (l & 3);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = 4 * hh + vrow + 8 * half;
#pragma unroll
            for (int par = 0; par < 4; ++par)
                voff[par][half] = (32 * wk + r) * HD + 8 * ((4 * par + (vcol >> 3)) ^ swz32(r)) + (vcol & 7);
        }
    }

    // Operand reads: K rows as the A operand of k-step ks, V as that of (k-step, dim block) j = 8 ks + db.
    auto k_op = [&](const _Float16* K, int ks) { return ld_h8(K + koff[ks & 7] + 128 * (ks >> 3)); };
    auto v_op = [&](const _Float16* V, int j) {
        const _Float16* v = V + (16 * (j >> 3)) * HD + 128 * ((j & 7) >> 2);
        return cat_h4(lds_tr4(v + voff[j & 3][0]), lds_tr4(v + voff[j & 3][1]));
    };
    // Online softmax in log2 units. The weights are 2^(s - m_run) with m_run 7 below the maximum seen when it was last
    // raised, and it is raised when a row's maximum passes m_run + 15: weights stay below 2^15, inside f16, and the pair
    // hi + lo resolves 2^-24 of them, 2^-31 of a fresh maximum, so that many small weights still count.
    float minus = 0.f;     // -m_run, 0 while a row has seen no key
    f16v sc;               // the tile's exponents
    h8 ph[2], pl[2];       // its weights, hi and lo
    auto settle = [&](float mx) __attribute__((always_inline)) {   // mx: the largest exponent
        mx = max_xor32(mx);
        const bool grow = mx > 2 * P_BITS + 1 || (m_run == -INFINITY && mx > -INFINITY);
        if (__any(grow)) {
            const float up = grow ? mx - P_BITS : 0.0f;
            const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(-up);
            const float mnew = m_run == -INFINITY ? up : m_run + up;
            l_run *= alpha;
            // wait states between the last matrix ops' writes of O and scale_acc's reads, as in the flash form
            asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7\n\ts_nop 7");
#pragma unroll
            for (int db = 0; db < 8; ++db) scale_acc(o[db], alpha);
            if (grow) m_run = mnew;
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[i] -= up;
            minus = m_run == -INFINITY ? 0.0f : -m_run;
        }
    };
    // keys at or past kend: exponent -inf; returns the largest of the rest
    auto mask = [&](int kb) __attribute__((always_inline)) {
        const int lim = kend - kb - 32 * wk - 4 * hh;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (8 * (i >> 2) + (i & 3) >= lim) sc[i] = -INFINITY;
            mx = fmaxf(mx, sc[i]);
        }
        return mx;
    };
    auto weight2 = [&](int i) {   // weights i and i + 1
        const f2 p = {__builtin_amdgcn_exp2f(sc[i]), __builtin_amdgcn_exp2f(sc[i + 1])};
        h2 hi, lo;
        split2(p, neg1, hi, lo);
        l_run += p[0];
        l_run += p[1];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            ph[i >> 3][(i & 7) + e] = hi[e];
            pl[i >> 3][(i & 7) + e] = lo[e];
        }
    };
    // Tile loads in flight: offsets of this lane's rows from the tile's first, clamped anew for the last, partial tiles
    unsigned offk[8], offv[8];
    const unsigned rowb = 2u * (unsigned)kvd;
    auto offsets = [&](unsigned (&off)[8], int kb) __attribute__((always_inline)) {
        const int rmax = max(kend - 1 - kb, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) off[i] = (unsigned)min(16 * w + 2 * i + (l >> 5), rmax) * rowb + (unsigned)cj[i];
    };
    auto row_base = [&](const uint16_t* src, int kb) { return (const char*)(src + (size_t)min(kb, kend - 1) * kvd); };
    auto piece = [&](const char* base, const unsigned (&off)[8], _Float16* lds, int i) {
        typedef __attribute__((address_space(3))) void lds_void;
        __builtin_amdgcn_global_load_lds((const void*)(base + off[i]), (lds_void*)(lds + (16 * w + 2 * i) * HD), 16, 0, 0);
    };
#define IT_FENCE __builtin_amdgcn_sched_barrier(0)
    // One tile and the next one's scores, in 32 steps of two dependent matrix ops (hi, lo). One wave a SIMD issues in order,
    // so what is to run in the shadow of the matrix ops stands between them: the score steps hold this tile's 16
    // exponentials with their conversions and the 16 loads of coming tiles, the value steps the next tile's maximum;
    // operands are read four steps ahead. K runs a tile ahead of V: at the start K of the next tile (Kn) and V of this
    // one have landed, and K of the one after (into Kf) and V of the next (into Vn) go out.
    auto tile = [&](int kb, const _Float16* Kn, const _Float16* V, _Float16* Kf, _Float16* Vn) __attribute__((always_inline)) {
        IT_WAIT_VMCNT(0);
        __syncthreads();   // landed for every wave, and every wave is done with the buffers written now
        if (kb + 3 * BN > kend) offsets(offk, kb + 2 * BN);   // (a tile past the end: its last row again, unused)
        if (kb + 2 * BN > kend) offsets(offv, kb + BN);
        const char *kbase = row_base(kc, kb + 2 * BN), *vbase = row_base(vc, kb + BN);
        f16v sa = f16v{};
        h8 k[16], v[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = k_op(Kn, i);
        IT_FENCE;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i < 12) k[i + 4] = k_op(Kn, i + 4);
            else v[i - 12] = v_op(V, i - 12);
            sa = mfma32x32x16(k[i], qh[i], sa);
            if (i & 1) weight2(i - 1);
            IT_FENCE;
            sa = mfma32x32x16(k[i], ql[i], sa);
            if (i < 8) piece(kbase, offk, Kf, i);
            else piece(vbase, offv, Vn, i - 8);
            IT_FENCE;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            if (j < 12) v[j + 4] = v_op(V, j + 4);
            o[j & 7] = mfma32x32x16(v[j], ph[j >> 3], o[j & 7]);
            if (j >= 4 && j < 12) {   // (the last score op's result takes the first steps)
                sc[2 * j - 8] = __builtin_fmaf(sa[2 * j - 8], back, minus);
                sc[2 * j - 7] = __builtin_fmaf(sa[2 * j - 7], back, minus);
                mx = fmaxf(fmaxf(mx, sc[2 * j - 8]), sc[2 * j - 7]);
            }
            IT_FENCE;
            o[j & 7] = mfma32x32x16(v[j], pl[j >> 3], o[j & 7]);
            IT_FENCE;
        }
        if (kb + 2 * BN > kend) mx = mask(kb + BN);
        settle(mx);
    };
    offsets(offk, kb0 + BN);
    offsets(offv, kb0 + BN);
    // first tile's scores: K0, V0 hold it; its successor's K goes to K1 once q has been read from there
    {
        IT_WAIT_VMCNT(0);
        __syncthreads();
        if (kb0 + BN < kend) {
            const char* kbase = row_base(kc, kb0 + BN);
#pragma unroll
            for (int i = 0; i < 8; ++i) piece(kbase, offk, K1, i);
        }
        sc = f16v{};
        h8 k[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = k_op(K0, i);
        IT_FENCE;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i < 8) k[i + 8] = k_op(K0, i + 8);
            sc = mfma32x32x16(k[i], qh[i], sc);
            sc = mfma32x32x16(k[i], ql[i], sc);
            IT_FENCE;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] *= back;
        const float mx = max_xor32(mask(kb0));
        if (mx > -INFINITY) m_run = mx - P_BITS;   // (O and l are zero: nothing to rescale)
        const float up = mx > -INFINITY ? m_run : 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] -= up;
        minus = -up;
    }
    int kb = kb0;
    for (; kb + 2 * BN < kend; kb += 2 * BN) {   // two tiles whose successors exist
        tile(kb, K1, V0, K0, V1);
        tile(kb + BN, K0, V1, K1, V0);
    }
    const bool even = kb + BN >= kend;   // the last tile's V is in V0, else one more tile precedes it
    if (!even) tile(kb, K1, V0, K0, V1);
    IT_WAIT_VMCNT(0);
    __syncthreads();
    {
        const _Float16* V = even ? V0 : V1;
#pragma unroll
        for (int i = 0; i < 16; i += 2) weight2(i);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const h8 v = v_op(V, j);
            o[j & 7] = mfma32x32x16(v, ph[j >> 3], o[j & 7]);
            o[j & 7] = mfma32x32x16(v, pl[j >> 3], o[j & 7]);
        }
    }
#undef IT_FENCE
    // ---- join the two key halves of each row: a wave keeps the 128 dims 128 wk .. +127 and hands the others to its
    // partner (O^T of row c at dims 32 db + 8 i4 + 4 hh .. +3, 16-byte chunks XOR-swizzled by row, in one pair of
    // buffers), the joined rows go out through the other pair, whole rows a store
    IT_WAIT_VMCNT(0);   // the loads issued past the end land in the buffers
    __syncthreads();
    l_run = sum_xor32(l_run);
    float* give = (float*)(wr ? K1 : K0);
    const auto chunk_at = [&](int db, int i4) { return c * HD + 4 * ((8 * db + 2 * i4 + hh) ^ c); };
    const auto part_of = [&](int db, int i4) {
        return f4{o[db][4 * i4], o[db][4 * i4 + 1], o[db][4 * i4 + 2], o[db][4 * i4 + 3]};
    };
    if (wk == 0) {   // (static register indexes)
#pragma unroll
        for (int db = 4; db < 8; ++db)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) *(f4*)(give + chunk_at(db, i4)) = part_of(db, i4);
    } else {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) *(f4*)(give + chunk_at(db, i4)) = part_of(db, i4);
    }
    if (hh == 0) { ms[wk][32 * wr + c] = m_run; ls[wk][32 * wr + c] = l_run; }
    __syncthreads();
    float* joined = (float*)(wr ? V1 : V0);
    {
        const float m2 = ms[wk ^ 1][32 * wr + c], l2 = ls[wk ^ 1][32 * wr + c], m = fmaxf(m_run, m2);
        const float a1 = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run - m);
        const float a2 = m2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m2 - m);
        f4 got[16];   // (all read before any is written: the compiler does not know that the buffers differ)
#pragma unroll
        for (int i = 0; i < 16; ++i) got[i] = *(const f4*)(give + chunk_at(4 * wk + i / 4, i & 3)) * a2;
        if (wk == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) got[i] += part_of(i / 4, i & 3) * a1;
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) got[i] += part_of(4 + i / 4, i & 3) * a1;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) *(f4*)(joined + chunk_at(4 * wk + i / 4, i & 3)) = got[i];
        if (wk == 0 && hh == 0) rowml[32 * wr + c] = f2{m * LN2_F, l_run * a1 + l2 * a2};
    }
    __syncthreads();
    {
        const float* src = (const float*)(w < 2 ? V0 : V1);
        const int r0 = rb * BM + 16 * w;
        int tq = __builtin_amdgcn_readfirstlane(r0 / G), gq = r0 - tq * G;
#pragma unroll
        for (int i0 = 0; i0 < 16; i0 += 8) {
            f4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = 16 * w + i0 + i;
                v[i] = *(const f4*)(src + (row & 31) * HD + 4 * (l ^ (row & 31)));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (r0 + i0 + i < R) {
                    float* rec = part + idx::rec(tq * nh + kh * G + gq, s, smax) * PART;
                    *(f4*)(rec + 4 + 4 * l) = v[i];
                    if (l == 0) *(f4*)rec = f4{rowml[16 * w + i0 + i][0], rowml[16 * w + i0 + i][1], 0.f, 0.f};
                }
                if (++gq == G) { gq = 0; ++tq; }
            }
        }
    }
}

// Four cache values
template <class KVT> struct Kv4 { typedef h4 T; };
template <> struct Kv4<float> { typedef f4 T; };

// One workgroup per (256 / SL * 4 dims, head, node); nr: the tree's rows in the cache. Thread = (split lane sg of SL, dim lane
// of 256 / SL, 4 dims each): split lane sg takes the context's records sg, sg + SL, ... and the path's keys likewise.
// KVT: the cache's values, uint16_t (f16) or float.
// Bound by two dependent round trips (the mask, then the path's rows) and by the records' bytes: 5 nodes, 16 heads, 10
// records 4.4 us; 64 nodes with 16 records each, 17 MB, 7.6 us.
template <int SL, class KVT>
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(const float* __restrict__ q, int qts,
                                                              const KVT* __restrict__ kc,
                                                              const KVT* __restrict__ vc, int kvd, int pos0,
                                                              int nh, int nkv, int nr,
                                                              const uint64_t* __restrict__ anc, float scale,
                                                              const float* __restrict__ part, int smax,
                                                              float* __restrict__ out, int ots) {
    typedef typename Kv4<KVT>::T V4;
    constexpr int DLN = 256 / SL, DW = 4 * DLN;   // dim lanes, dims per workgroup
    constexpr int NK = 64 / SL;                   // path keys per split lane
    __shared__ int node[64];                      // the path's nodes in order
    __shared__ float score[64];
    __shared__ float red_m[SL], red_d[SL];
    __shared__ f4 red_o[SL][DLN];
    const int dq = blockIdx.x, h = blockIdx.y, t = blockIdx.z, tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    const int sg = tid / DLN, dl = tid % DLN, d0 = DW * dq + 4 * dl;
    float* dst = out + (size_t)t * ots + (size_t)h * HD + d0;
    // What does not hang on the mask goes out first: the first batch of the context's records, q and the gate. Lanes
    // past the last record reload it and count nothing.
    const float* base = part + idx::rec(t * nh + h, 0, smax) * PART;
    f2 hv[SPL];
    f4 ov[SPL];
    auto load = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            hv[j] = f2{-INFINITY, 0.f};
            ov[j] = f4{0.f, 0.f, 0.f, 0.f};
            if (s0 + SL * j < smax) {   // (the same for every lane)
                const float* rec = base + (size_t)min(s0 + sg + SL * j, smax - 1) * PART;
                hv[j] = *(const f2*)rec;
                ov[j] = ld_f4(rec + 4 + d0);
            }
        }
    };
    load(0);
    const float* qrow = q + (size_t)t * qts + (size_t)h * 2 * HD;
    const f4 qv = ld_f4(qrow + 4 * l), gt = ld_f4(qrow + HD + d0);
    const uint64_t mask = anc[t] & (~(uint64_t)0 >> (64 - nr));
    const int np = (int)__popcll(mask);
    if (np == 0) {   // a padding node
        if (sg == 0) *(f4*)dst = f4{0.f, 0.f, 0.f, 0.f};
        return;
    }
    if (tid < 64 && (mask >> tid & 1)) node[__popcll(mask & (((uint64_t)1 << tid) - 1))] = tid;
    __syncthreads();
    // ---- the path: this lane's V pieces go out first, then the scores, a key a wave
    const size_t head = (size_t)(h / (nh / nkv)) * HD;
    V4 pv[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j)
        if (SL * j < np) pv[j] = *(const V4*)(vc + (size_t)(pos0 + node[min(sg + SL * j, np - 1)]) * kvd + head + d0);
    for (int j0 = w; j0 < np; j0 += 16) {
        V4 kv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            kv[j] = *(const V4*)(kc + (size_t)(pos0 + node[min(j0 + 4 * j, np - 1)]) * kvd + head + 4 * l);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float s = wave_sum((qv[0] * (float)kv[j][0] + qv[1] * (float)kv[j][1]) +
                                     (qv[2] * (float)kv[j][2] + qv[3] * (float)kv[j][3]));
            if (l == 0 && j0 + 4 * j < np) score[j0 + 4 * j] = s * scale;
        }
    }
    auto batch_max = [&]() {
        float m = hv[0][0];
#pragma unroll
        for (int j = 1; j < SPL; ++j) m = fmaxf(m, hv[j][0]);
        return m;
    };
    if (dl == 0) red_m[sg] = batch_max();
    __syncthreads();
    // ---- the path and the first batch of records (no reference below the type's range, so that keys of score -inf weigh 0)
    float M = wave_max(l < np ? score[l] : -FLT_MAX);
#pragma unroll
    for (int j = 0; j < SL; ++j) M = fmaxf(M, red_m[j]);
    float den = 0.f;
    f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NK; ++j) {
        if (sg + SL * j < np) {
            const float e = __expf(score[sg + SL * j] - M);
            den += e;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += e * (float)pv[j][i];
        }
    }
    auto add_batch = [&](int s0) {
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            if (s0 + sg + SL * j < smax) {
                const float wgt = __expf(hv[j][0] - M);
                den += hv[j][1] * wgt;
                o += ov[j] * wgt;
            }
        }
    };
    add_batch(0);
    // ---- the other records
    for (int s0 = SL * SPL; s0 < smax; s0 += SL * SPL) {
        load(s0);
        __syncthreads();   // every lane has read the last batch's maxima
        if (dl == 0) red_m[sg] = batch_max();
        __syncthreads();
        float Mn = M;
#pragma unroll
        for (int j = 0; j < SL; ++j) Mn = fmaxf(Mn, red_m[j]);
        const float r = __expf(M - Mn);
        den *= r;
        o *= r;
        M = Mn;
        add_batch(s0);
    }
    red_o[sg][dl] = o;
    if (dl == 0) red_d[sg] = den;
    __syncthreads();
    if (sg == 0) {
        float dd = red_d[0];
#pragma unroll
        for (int j = 1; j < SL; ++j) { o += red_o[j][dl]; dd += red_d[j]; }
        f4 res;
#pragma unroll
        for (int j = 0; j < 4; ++j) res[j] = o[j] / dd * sigmoidf_(gt[j]);
        *(f4*)dst = res;
    }
}

// The context's form and keys per split, with R = nt * nh / nkv rows a KV head. The decode partials take 8 or 16 rows a
// workgroup: 8 where one 64-key tile each is at most one round of the CUs, else 16 (8 if there are no more), with as many
// tiles one after the other as make one round. A workgroup of 16 rows takes 8.5 us and 2.1 a tile of a whole call; those of 64
// rows take 19 and 0.8 to 1.6, share a tile among four times the rows and stream the next ones while they compute. So
// up to 5 tiles a workgroup go to the partials. Up to 16 rows both forms read each key once, and the partials stay ahead as
// long as the call is not at the bytes (12 tiles, 16 with 8 rows).
// Whole calls in us, 16/2 heads, 8 rows / 16: 5 nodes at 600 keys 8.8 / 9.7 (32 rows: 12.1), 8 at 1000 9.5 / 10.2, 12 at 1000
// 11.2 / 10.2, 4 at 3000 13.5 / 11.3. 16 rows / 64: 4 nodes 8155 keys (2 tiles) 14.4 / 20.9, 20443 (5) 21.1 / 21.6, 24539
// (6) 23.4 / 22.8; 8 nodes 4059 (2) 13.6 / 20.2, 8155 (4) 18.3 / 23.5, 10203 (5) 20.6 / 21.7, 12251 (6) 22.8 / 22.0; 64
// nodes 731 (3) 16.4 / 21.6, 1499 (6) 23.0 / 23.2, 2011 (8) 27.6 / 25.8; 2 nodes 65499 (8) 35.7 / 36.0, 131035 (16) 60.0 /
// 59.9; 8 rows / 64, 1 node 32731 (4) 18.5 / 22.2, 131035 (16) 52.4 / 58.8.
// Where the tiles do not divide evenly (3 or more a workgroup for one round, though one tile each is two rounds), two
// workgroups share a CU instead: 26 nodes at 1200 keys 14.7 us, in splits of three tiles 16.1.
constexpr int CUS = 256;   // MI355X compute units
struct TreePlan { int rows, chunk; };   // rows: 8 or 16 (decode partials), or 64
static TreePlan plan(int pos0, int nt, int nh, int nkv) {
    const long tiles = ((long)pos0 + 63) / 64, R = (long)nt * (nh / nkv);
    const auto groups = [&](long rows) { return nkv * ((R + rows - 1) / rows); };
    const auto one_round = [&](long g) {   // tiles a split
        const long splits = std::max(1L, CUS / g);
        return (tiles + splits - 1) / splits;
    };
    if (tiles * groups(8) <= CUS) return {8, 64};
    const int rows = R <= 8 ? 8 : 16;
    const long g = groups(rows);
    long k = one_round(g);
    if (k > 2 && tiles * g <= 2 * CUS) k = 1;
    const long rounds = (g + CUS - 1) / CUS;   // (more than one with more KV heads and rows than CUs)
    if (k * rounds <= (R <= 8 ? 16 : R <= 16 ? 12 : 5)) return {rows, 64 * (int)k};
    return {BM, 64 * (int)one_round(groups(BM))};
}
int attn_tree_chunk(int pos0, int nt, int nh, int nkv) { return plan(pos0, nt, nh, nkv).chunk; }

template <class KVT>
static hipError_t launch_merge(const float* q, int qts, const KVT* kc, const KVT* vc, int kvd, int pos0, int nh, int nkv,
                               int nt, int nr, const uint64_t* anc, float scale, float* out, int ots, const float* part,
                               int smax, hipStream_t st) {
    // A quarter of the dims and 16 split lanes a workgroup where a few rows have many records (1 node, 16/2 heads, 8128 keys
    // in 127 splits: 10.5 us the call against 14.2), else whole rows and 4 split lanes (26 nodes at 600 keys 14.2 against
    // 19.0, from the path's keys that every workgroup of a row scores).
    if (smax > 32 && nt * nh <= 192)
        attn_tree_merge_kernel<16, KVT><<<dim3(4, nh, nt), 256, 0, st>>>(q, qts, kc, vc, kvd, pos0, nh, nkv, nr, anc, scale,
                                                                       part, smax, out, ots);
    else
        attn_tree_merge_kernel<4, KVT><<<dim3(1, nh, nt), 256, 0, st>>>(q, qts, kc, vc, kvd, pos0, nh, nkv, nr, anc, scale,
                                                                      part, smax, out, ots);
    return hipGetLastError();
}

hipError_t launch_attn_tree(const float* q, int qts, const uint16_t* kc, const uint16_t* vc, int kvd, int pos0,
                            int nh, int nkv, int nt, int nr, const uint64_t* anc, float scale, float* out, int ots,
                            float* part, int chunk, hipStream_t st) {
    int smax = 0;
    if (pos0 > 0) {
        smax = idx::split_count(pos0, chunk);
        hipError_t e;
        const int rows = plan(pos0, nt, nh, nkv).rows;
        if (rows == BM) {
            const int nrb = (nt * (nh / nkv) + BM - 1) / BM;
            const unsigned grid = (unsigned)((smax * nkv + 7) / 8 * 8 * nrb);
            attn_tree_ctx_kernel<<<grid, 256, 0, st>>>(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, scale, part, chunk, smax, nrb);
            e = hipGetLastError();
        } else {
            e = launch_attn_all_partials(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, scale, part, chunk, rows, st);
        }
        if (e != hipSuccess) return e;
    }
    return launch_merge(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, nr, anc, scale, out, ots, part, smax, st);
}

hipError_t launch_attn_tree_f32kv(const float* q, int qts, const float* kc, const float* vc, int kvd, int pos0,
                                  int nh, int nkv, int nt, int nr, const uint64_t* anc, float scale, float* out, int ots,
                                  float* part, int chunk, hipStream_t st) {
    int smax = 0;
    if (pos0 > 0) {
        smax = idx::split_count(pos0, chunk);
        const hipError_t e =
            launch_attn_f32kv_all_partials(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, scale, part, chunk, st);
        if (e != hipSuccess) return e;
    }
    return launch_merge(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, nr, anc, scale, out, ots, part, smax, st);
}

}  // namespace it
