// Causal GQA attention with sigmoid gate over the paged 8-bit cache, for one token a sequence up to whole prompts:
//   out = sigmoid(gate) * sum_j p_j v_j / sum_j p_j,  p_j = e^(scale q.k_j), j <= len + t.
//
// A unit of work is (sequence, KV head, block of ROWS query rows r = t*G + g, split of the pages). Its workgroup takes a
// page a step, the four waves sharing it:
//   S^T = K q^T    wave w has the page's block w: 16 keys, all query rows
//   softmax        a running reference per row, common to the waves; P^T goes through LDS
//   O^T += V^T P^T wave w has a quarter of the dims, all 64 keys and rows
// K's codes are integers already, so K q^T is integer products with q in signed 8-bit digits, fixed point in its row's largest
// value: three digits (2^-23 of it) for an f32 output, two (2^-15) for most f16 ones. A digit more costs a product of 16 x 16 x 64
// a key block, where converting K would cost the vector units 6 operations for 4 codes, and they are what is short here. V's
// codes become f16 times their scale, exactly; P goes in as an f16 pair for an f32 output, as one f16 for an f16 one. What an f16
// output, whose own rounding is 2.1e-4, loses by that and what it would cost (error against 64 bits, us; as said / with pairs / and
// three digits): 8192-token prompt 2.7e-4 628, 2.1e-4 786, 2.1e-4 900; 512 tokens after 32256 383, 481, 573; in blocks of 16 rows, 32
// ragged sequences of a token each, 2.3e-4 19.5, 2.1e-4 20.2, 2.1e-4 20.3. So blocks of 16 rows are as for an f32 output
// (PAIRS), larger ones not.
// The open page (f16 rows) comes first, with q as f16 pairs.
//
// The page's element order is that of the matrix operands. Each wave copies the 4 hd bytes that it alone needs straight into its
// part of LDS, a page or two ahead, and reads them back without a barrier; one barrier a page, for P.
//
// What bounds it (MI355X, hd 256): few tokens, the bytes of the codes: a token after 65535, 131071, 262143 and 524287 rows takes 25.3,
// 35.6, 57.4 and 104 us in a graph over inputs that no cache holds, so 6.5, 6.1 and 5.7 TB/s from each to the next, behind 6 us to a
// launch's first page, 1.4 for its records and 4 for the join of the splits. Whole prompts, the vector units beside the matrix ones: of a wave's
// instructions for 48 rows and a page 235 are vector ones (softmax, 96 for V, 16 for K's sign) and 48 matrix ones, vector issue is
// busy 63 % of the cycles, matrix units 40 %: 0.89 PFLOP/s.
//
// The lengths are on the device, so every workgroup finds its unit by itself: pages per split from the total work, a prefix sum over
// the sequences' unit counts. Sequences of one split are finished in place, the others' records {m, l, o} are joined by
// the second kernel.
#include <algorithm>

#include "internal.h"
#include "kv8.h"

namespace it {
namespace {

constexpr float P_BITS = 7.0f;   // weights up to 2^15 of the reference: see `settle`

// The loads that copy a wave's share of a page from memory into LDS stay in flight over barriers and other loads' waits, so they and
// their waits are written out (the compiler waits for all of them at every barrier). They have no result register; LDS is
// read behind `landed`.
//
// A barrier that orders LDS traffic only.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
// Waits until at most N loads are still in flight; they land in the order that they were issued in.
template <int N> __device__ __forceinline__ void landed() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// N KiB from `from` (each lane 16 bytes at off + 1024 i) to LDS from `to` on (lane l at 16 l + 1024 i: the instruction's offset
// counts on both sides). What stood there has been read when they go out. m0 holds the LDS address: the compiler reserves it, and no
// instruction of its own here uses it (tests/test_kv8_asm.py).
template <int N> __device__ __forceinline__ void kib_to_lds(const uint8_t* from, unsigned off, uint8_t* to) {
    typedef __attribute__((address_space(3))) uint8_t lds_u8;
    const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_u8*)to);
    static_assert(N == 1 || N == 2 || N == 4, "a wave's share of a page");
    if constexpr (N == 4)
        asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\t"
                     "global_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400\n\t"
                     "global_load_lds_dwordx4 %1, %2 offset:0x800\n\tglobal_load_lds_dwordx4 %1, %2 offset:0xC00"
                     ::"s"(at), "v"(off), "s"(from) : "memory");
    else if constexpr (N == 2)
        asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\t"
                     "global_load_lds_dwordx4 %1, %2\n\tglobal_load_lds_dwordx4 %1, %2 offset:0x400"
                     ::"s"(at), "v"(off), "s"(from) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_waitcnt lgkmcnt(0)\n\tglobal_load_lds_dwordx4 %1, %2"
                     ::"s"(at), "v"(off), "s"(from) : "memory");
}
// Inclusive, over the wave: within rows of 16 lanes, then the rows before (by lane moves; through LDS the batch's 32 lengths
// were 1,500 cycles of the way to a page)
__device__ __forceinline__ int prefix_sum(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // lane 15 to the next row: rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // lane 31 to rows 2 and 3
    return v;
}

// x / d for 0 <= x < 2^21, inv = rcp(d): (x + 1/2) / d is off by less than 1/2d. (Indices by full divisions were 1,700 of
// the 12,800 cycles of a one-page workgroup.)
__device__ __forceinline__ int div_small(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// Pages per split of this call (the same in both kernels; sums in a fixed order)
template <int ROWS>
__device__ __forceinline__ int call_chunk(const Kv8Batch& b, const Kv8Seq& s0, int G, int nkv, int wgs, int l) {
    if (b.nseq == 1) {   // (the sum of one, without the exchanges)
        const float blocks = (float)((__builtin_amdgcn_readfirstlane(s0.n) * G + ROWS - 1) / ROWS);
        return kv8::chunk_pages(blocks * (float)__builtin_amdgcn_readfirstlane(s0.pages) * (float)nkv, blocks * (float)nkv, wgs);
    }
    float sum = 0.f, blocks = 0.f;
    for (int i0 = 0; i0 < b.nseq; i0 += 64) {
        const Kv8Seq s = i0 == 0 ? s0 : kv8_seq(b, i0 + l);
        const float nrb = (float)((s.n * G + ROWS - 1) / ROWS);
        sum += wave_sum(nrb * (float)s.pages);
        blocks += wave_sum(nrb);
    }
    const float work = readlane_f(sum, 0) * (float)nkv, groups = readlane_f(blocks, 0) * (float)nkv;
    int chunk = kv8::chunk_pages(work, groups, wgs);
    // (of fewer, the count costs more than it gives: us, counted / not, ten pages, 16 sequences of 4096 rows 27.8 / 24.6, 32 of four
    // tokens after 4096 47.7 / 45.5; of 22 pages, 64 sequences of 4096 rows 60.8 / 62.6, 8 of 32 tokens after 4096 54.2 / 58.5)
    if (chunk > (ROWS == 16 ? 12 : 18) && groups <= (float)wgs) {
        float rcp[kv8::TRIES], units[kv8::TRIES] = {};
#pragma unroll
        for (int k = 0; k < kv8::TRIES; ++k) rcp[k] = __builtin_amdgcn_rcpf((float)kv8::fewer_pages(work, groups, wgs, k));
        for (int i0 = 0; i0 < b.nseq; i0 += 64) {
            const Kv8Seq s = i0 == 0 ? s0 : kv8_seq(b, i0 + l);
            const float nrb = (float)((s.n * G + ROWS - 1) / ROWS);
#pragma unroll
            for (int k = 0; k < kv8::TRIES; ++k) units[k] += wave_sum(nrb * kv8::about_splits(s.pages, rcp[k]));
        }
#pragma unroll
        for (int k = kv8::TRIES - 1; k >= 0; --k)
            if (readlane_f(units[k], 0) * (float)nkv <= (float)wgs) chunk = kv8::fewer_pages(work, groups, wgs, k);
    }
    return chunk;
}

// What is found for a workgroup, in scalar registers: its sequence, the index of its unit (main kernel) or of its row block that
// was split (merge) among the sequence's, a KV head's alone, and the first record of the sequence.
struct Found {
    int seq, t0, n, len, pages, nrb, ns, at, rec;
    bool any, bad;
};
template <int ROWS, bool GROUPS>
__device__ __forceinline__ Found find(const Kv8Batch& b, const Kv8Seq& s0, int G, int nkv, int chunk, int id, int l) {
    Found f;
    if (b.nseq == 1) {
        f = {0, 0, 0, 0, 0, 0, 0, id, 0, false, false};
        f.t0 = __builtin_amdgcn_readfirstlane(s0.t0);
        f.n = __builtin_amdgcn_readfirstlane(s0.n);
        f.len = __builtin_amdgcn_readfirstlane(s0.len);
        f.pages = __builtin_amdgcn_readfirstlane(s0.pages);
        f.bad = __builtin_amdgcn_readfirstlane((int)s0.bad) != 0;
        f.nrb = (f.n * G + ROWS - 1) / ROWS;
        f.ns = kv8::splits(f.pages, chunk);
        f.any = id < f.nrb * (GROUPS ? (f.ns > 1 ? 1 : 0) : f.ns);
        return f;
    }
    f.any = false;
    int base = 0, rbase = 0;
    for (int i0 = 0; i0 < b.nseq; i0 += 64) {
        const Kv8Seq s = i0 == 0 ? s0 : kv8_seq(b, i0 + l);
        const int nrb = (s.n * G + ROWS - 1) / ROWS, ns = kv8::splits(s.pages, chunk);
        const int recs = ns > 1 ? nrb * ns * nkv : 0, units = GROUPS ? (ns > 1 ? nrb : 0) : nrb * ns;
        const int pu = prefix_sum(units), pr = prefix_sum(recs);
        const unsigned long long hit = __ballot(base + pu > id);
        if (hit) {
            const int src = __builtin_ctzll(hit);
            f.seq = i0 + src;
            f.t0 = __builtin_amdgcn_readlane(s.t0, src);
            f.n = __builtin_amdgcn_readlane(s.n, src);
            f.len = __builtin_amdgcn_readlane(s.len, src);
            f.pages = __builtin_amdgcn_readlane(s.pages, src);
            f.bad = __builtin_amdgcn_readlane((int)s.bad, src) != 0;
            f.nrb = __builtin_amdgcn_readlane(nrb, src);
            f.ns = __builtin_amdgcn_readlane(ns, src);
            f.at = id - base - __builtin_amdgcn_readlane(pu - units, src);
            f.rec = rbase + __builtin_amdgcn_readlane(pr - recs, src);
            f.any = true;
            return f;
        }
        base += __builtin_amdgcn_readlane(pu, 63);
        rbase += __builtin_amdgcn_readlane(pr, 63);
    }
    return f;
}

__device__ __forceinline__ void store4(float* p, f4 v) { *(f4*)p = v; }
__device__ __forceinline__ void store4(_Float16* p, f4 v) { st4(p, v); }

typedef int i4 __attribute__((ext_vector_type(4)));
// D = A(16x64) B(64x16) + C in 8-bit integers; lane l holds A row / B column l & 15 with 16 consecutive bytes of the group l >> 4,
// D as mfma16x16x32's.
__device__ __forceinline__ i4 mfma_i8(u4 a, u4 b, i4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i4, a), __builtin_bit_cast(i4, b), c, 0, 0, 0);
}
// Byte k of four words, as a word each.
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int k) {
    const uint32_t pair = 0x04000400u + 0x0101u * k * 0x10001u;   // per 16 bits: byte k of the second, byte k of the first
    const uint32_t ab = __builtin_amdgcn_perm(b, a, pair), cd = __builtin_amdgcn_perm(d, c, pair);
    return __builtin_amdgcn_perm(cd, ab, 0x05040100u);
}

// Records: {m, l} [record][ROWS] (m in log2 units), then o [record][ROWS][HD].
//
// Wave w takes key block w of a page for the scores and weights, and dim blocks ND * w .. + ND-1 for O.
template <int HD, int RB, bool PAIRS, class OutT>
__global__ __launch_bounds__(256, 2) void attn_kv8_kernel(Kv8 c, Kv8Batch b, const float* __restrict__ q, int qts, int G,
                                                          float scale, OutT* __restrict__ out, int ots,
                                                          float* __restrict__ part, int wgs) {
    constexpr int ROWS = 16 * RB, NP = PAIRS ? 2 : 1, NJ = HD / 64, NK = HD / 32, ND = HD / 64, DG = PAIRS ? 3 : 2;
    constexpr int KIB = 1024, QUARTER = 16 * HD;   // a wave's share of a page's codes
    // Forms of many rows keep a part of q's digits in LDS, and one page of V in place of two: 256 registers and half of a
    // CU's LDS, so that two workgroups share a CU.
    constexpr int KB = RB == 1 ? 2 : 1, VB = RB == 4 || (RB == 3 && PAIRS) ? 1 : 2;   // pages of K and of V
    constexpr int QL = HD < 256 || VB == 2 ? 0 : RB - 2, NR = NJ - QL;    // of q's NJ groups of 64 dims: in LDS, in registers
    __shared__ __align__(16) uint8_t kbuf[KB][4 * QUARTER], vbuf[VB][4 * QUARTER];
    __shared__ __align__(16) u4 qlast[QL ? RB : 1][QL ? QL : 1][DG][QL ? 64 : 1];
    __shared__ __align__(16) _Float16 pbuf[2][RB][2][NP][64 * 8];   // P^T operands: [parity][rows][keys][hi, lo]
    __shared__ __align__(16) float mbuf[ROWS][4];                   // row maxima by key block
    __shared__ __align__(16) int over[2][4];                        // whether a wave's weights are too large
    __shared__ __align__(16) float lbuf[ROWS][4];                   // row sums by key block; at first q's maxima by dims
    __shared__ int qlim[ROWS];                                      // the last key that a row sees

    const int nkv = c.nkv;   // G: query heads of a KV head
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, lr = l & 15;
    const Kv8Seq s0 = kv8_seq(b, l);
    const int chunk = call_chunk<ROWS>(b, s0, G, nkv, wgs, l);
    const Found u = find<ROWS, false>(b, s0, G, nkv, chunk, (int)(blockIdx.z * gridDim.y + blockIdx.y), l);
    if (!u.any) return;
    // the heaviest row blocks first; heads and row blocks of a split side by side
    const int kh = blockIdx.x;
    int rb = 0, split = u.at, tmin = 0, tmax = u.n - 1;
    const int R = u.n * G;
    if (u.nrb > 1) {
        split = (unsigned)u.at / (unsigned)u.nrb;
        rb = u.nrb - 1 - (u.at - split * u.nrb);
        tmin = (unsigned)(rb * ROWS) / (unsigned)G;
        tmax = (unsigned)(min(R, rb * ROWS + ROWS) - 1) / (unsigned)G;
    }
    // row r0 + i of the block: its token, and by that its query head
    const int r0 = rb * ROWS, over0 = r0 - tmin * G;
    const float rcp_G = __builtin_amdgcn_rcpf((float)G);
    auto token = [&](int i) __attribute__((always_inline)) { return tmin + div_small(over0 + i, rcp_G); };

    if (u.bad) {   // a sequence whose length cannot be: NaN
        for (int i = tid; i < ROWS * (HD / 4); i += 256) {
            const int r = r0 + i / (HD / 4), t = token(i / (HD / 4));
            if (r < R)
                store4(out + (size_t)(u.t0 + t) * ots + (size_t)(kh * G + r - t * G) * HD + 4 * (i % (HD / 4)), f4{NAN, NAN, NAN, NAN});
        }
        return;
    }
    const int total = u.len + u.n, closed = total / kv8::PAGE;          // full pages; the open rows are page `closed`
    const int p0 = (int)min((long)split * chunk, (long)u.pages);
    const int p1 = (int)min((long)p0 + chunk, (long)(u.len + tmax) / kv8::PAGE + 1);
    const bool tail = p1 > closed && p1 > p0;                            // the last page of the range is the open one
    const int np = max(min(p1, closed) - p0, 0);                         // full pages of the range
    const int clear = u.len + tmin;                                      // keys up to here are seen by every row
    if (u.ns > 1 && np == 0 && !tail) return;   // no row of the block sees the split: its record is not read

    // ---- pages. Lane i of `ids` and `scl` has the number and the scales of full page 64 n + i of the range; each is read
    // anew every 64 pages, with its wait in the branch (no other load then waits for it). A page that the pool has not: NaN scores.
    const int* table = b.table + (size_t)u.seq * b.max_pages + p0;
    int ids = 0;
    u4 scl = {};
    auto load_ids = [&](int j) __attribute__((always_inline)) {
        ids = table[min(j + l, max(np - 1, 0))];
        asm volatile("" : "+v"(ids));
    };
    auto load_scales = [&]() __attribute__((always_inline)) {
        const bool known = (unsigned)ids < (unsigned)c.npages;
        scl = *(const u4*)(c.sc + (known ? (size_t)ids * nkv + kh : 0) * 8);
        if (!known) scl = u4{0x7E007E00u, 0x7E007E00u, 0u, 0u};
    };
    auto page_of = [&](int j) __attribute__((always_inline)) {
        const unsigned id = __builtin_amdgcn_readlane(ids, j & 63);
        return id < (unsigned)c.npages ? id : 0u;
    };
    // This wave's quarter of a page's codes, K by block or V by dims, to LDS in the order that it is read back by the
    // same wave. Past the end (the loads go out without a branch, so that their count is known): one piece for all lanes.
    auto fetch = [&](const uint8_t* from, uint8_t* to, int j, unsigned id) __attribute__((always_inline)) {
        kib_to_lds<NJ>(from + uniform_off(((size_t)id * nkv + kh) * (kv8::PAGE * HD) + w * QUARTER), j < np ? 16 * l : 0,
                       to + w * QUARTER);
    };
    auto qrow = [&](int x) __attribute__((always_inline)) {
        const int i = min(16 * x + lr, R - 1 - r0), r = r0 + i, t = token(i);
        return q + (size_t)(u.t0 + t) * qts + (size_t)(kh * G + r - t * G) * 2 * HD;
    };

    // What the first wait is not for goes out before it: q, and the open page's keys
    const size_t open = ((size_t)(u.seq * 2 + (closed & 1)) * nkv + kh) * (kv8::PAGE * HD) + w * QUARTER + 16 * l;
    f4 y[RB][4];
    if (w < NJ) {
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            const float* at = qrow(x) + 64 * w + 8 * g;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[x][e] = ld_f4(at + 32 * (e >> 1) + 4 * (e & 1));
        }
    }
    h8 ko[NK];
    if (tail) {
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) ko[ks] = ld_h8(c.tk + open + KIB * (ks >> 1) + 8 * (ks & 1));
    }
    if (np > 0) {
        load_ids(0);
        fetch(c.kp, kbuf[0], 0, page_of(0));
        if constexpr (VB == 2) fetch(c.vp, vbuf[0], 0, page_of(0));
        if constexpr (KB == 2) fetch(c.kp, kbuf[1], 1, page_of(1));
        load_scales();
    }

    f4 o[RB][ND], sc[RB];                 // sc: products of a page, times back * ksc in log2 units
    // top: a row's reference + 15, neg: minus the reference (0 while there is none); back: from integer products to log2 units but
    // for K's scale ksc of the page that sc holds
    float top[RB], neg[RB], l_run[RB], back[RB], ksc = 1.f;
    u4 qd[RB][NR][DG];                    // q's digits, the highest first
    const float neg1 = in_register(-1.0f);
#pragma unroll
    for (int x = 0; x < RB; ++x) {
#pragma unroll
        for (int d = 0; d < ND; ++d) o[x][d] = f4{};
        top[x] = -INFINITY;
        neg[x] = 0.f;
        l_run[x] = 0.f;
    }

    // The keys that rows do not see get -inf (this lane's keys of page p are 16 w + 4 g + 0..3). An unknown page's scale is NaN, which
    // would reach these rows as NaN * -inf: there the scores that are seen become NaN in its place.
    auto mask_keys = [&](int p) __attribute__((always_inline)) {
        if (__any(ksc != ksc)) {
#pragma unroll
            for (int x = 0; x < RB; ++x) sc[x] = f4{NAN, NAN, NAN, NAN};
            ksc = 1.f;
        }
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            const int lim = qlim[16 * x + lr] - (p * kv8::PAGE + 16 * w + 4 * g);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[x][i] = i > lim ? -INFINITY : sc[x][i];
        }
    };
    // The rows' maxima over the wave's 16 keys, to LDS. Values of different row blocks share the lane exchanges: lane row g ends with
    // row block g of four, a half-wave with a row block of two.
    auto maxima = [&]() __attribute__((always_inline)) {
        float m[RB];
#pragma unroll
        for (int x = 0; x < RB; ++x) m[x] = fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3])) * (back[x] * ksc);
        int x = 0;
        float v;
        if constexpr (RB == 1) {
            v = max_xor32(max_xor16(m[0]));
        } else if constexpr (RB == 2) {
            swap32(m[0], m[1]);
            v = max_xor16(fmaxf(m[0], m[1]));
            x = g >> 1;
        } else {
            float m3 = m[RB - 1];
            swap32(m[0], m[2]);
            swap32(m[1], m3);
            float a = fmaxf(m[0], m[2]), e = fmaxf(m[1], m3);
            swap16(a, e);
            v = fmaxf(a, e);
            x = min(2 * (g >> 1) + (g & 1), RB - 1);
        }
        mbuf[16 * x + lr][w] = v;
    };
    // ---- q in units of its row's largest value / 2^(8 DG - 1), as DG signed digits of 8 bits, for integer products with the
    // codes. Wave w makes those of dims 64 w .. (hd 128: two waves); they meet in LDS that is not in use yet, a row block at a time.
    // A negative scale turns q round, and no unit is zero, so that -inf times it stays; where q or the scale is not finite it is NaN (the
    // maximum with the least unit would make one of a NaN).
    const float size = fabsf(scale) * LOG2E, sign = scale < 0.f ? -1.f : 1.f;
    if (tid < ROWS) qlim[tid] = r0 + tid < R ? u.len + token(tid) : -1;
    {
        if (w < NJ) {
#pragma unroll
            for (int x = 0; x < RB; ++x) {
                uint32_t mb = 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = y[x][i >> 2][i & 3];   // (a bit cast of the vector's element itself takes the first)
                    mb = max(mb, __builtin_bit_cast(uint32_t, e) & 0x7FFFFFFFu);
                }
                float m = __builtin_bit_cast(float, min(mb, 0x7F800000u));   // (infinity for a NaN)
                lbuf[16 * x + lr][w] = max_xor32(max_xor16(m));
            }
        }
        lds_barrier();
        auto row_max = [&](int x) __attribute__((always_inline)) {
            const f4 m4 = *(const f4*)lbuf[16 * x + lr];
            return NJ == 4 ? fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) : fmaxf(m4[0], m4[1]);
        };
        auto row_exp = [&](int x) __attribute__((always_inline)) { return max(__builtin_amdgcn_frexp_expf(row_max(x)), -100); };   // (so that 2^-ex is finite)
        // |q| / 2^ex < 1; the highest digit at most 127 for all digits' roundings
        constexpr float TOP = PAIRS ? 127 * 65536.f : 127 * 256.f;
        constexpr uint32_t BIAS = PAIRS ? 0x808080u : 0x8080u;
        // The open page comes first. Its keys are f16, so its products take q as f16 pairs (each row times the power of two that
        // takes its largest value to 2^13 .. 2^14). Wave w makes those of its dims too: all of the row in each wave is four times
        // the code, and code that few workgroups run is as slow as its fetching (16 rows 2.4, 32 rows 6.5 us).
        u4* meet = VB == 2 ? (u4*)vbuf[VB - 1] : (u4*)pbuf;
        static_assert(VB == 2 || sizeof(pbuf) >= 4 * NJ * KIB, "room for a row block's pairs");
        if (tail) {
#pragma unroll
            for (int x = 0; x < RB; ++x) {
                const int ex = 14 - row_exp(x);
                if (w < NJ) {
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks) {
                        const f4* z = &y[x][2 * ks];
                        h8 hi, lo;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            h2 h, e;
                            split2(f2{__builtin_amdgcn_ldexpf(z[i >> 1][2 * (i & 1)] * sign, ex),
                                      __builtin_amdgcn_ldexpf(z[i >> 1][2 * (i & 1) + 1] * sign, ex)}, neg1, h, e);
                            hi[2 * i] = h[0];
                            hi[2 * i + 1] = h[1];
                            lo[2 * i] = e[0];
                            lo[2 * i + 1] = e[1];
                        }
                        meet[(2 * w + ks) * 128 + l] = __builtin_bit_cast(u4, hi);
                        meet[(2 * w + ks) * 128 + 64 + l] = __builtin_bit_cast(u4, lo);
                    }
                }
                lds_barrier();
                f4 a = {}, a2 = {};
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    a = mfma16x16x32(ko[ks], ld_h8(meet + ks * 128 + l), a);
                    a2 = mfma16x16x32(ko[ks], ld_h8(meet + ks * 128 + 64 + l), a2);
                }
                const f4 both = a + a2;
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[x][i] = both[i] * (TOP * 0x1p-14f);   // in units of back
                lds_barrier();
            }
        }
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            const float m = row_max(x);
            const int ex = row_exp(x);
            const float to = __builtin_amdgcn_ldexpf(TOP * sign, -ex);
            back[x] = m < INFINITY && size < INFINITY ? fmaxf(__builtin_amdgcn_ldexpf(size / TOP, ex), 1e-30f) : NAN;
            if (w < NJ) {
                u4 dg[DG];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t n[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)   // the digits: bytes of n + BIAS, each less 128
                        n[i] = ((uint32_t)(int)rintf(y[x][e][i] * to) + BIAS) ^ BIAS;
#pragma unroll
                    for (int k = 0; k < DG; ++k) dg[k][e] = bytes_of(n[0], n[1], n[2], n[3], DG - 1 - k);
                }
#pragma unroll
                for (int k = 0; k < DG; ++k) meet[(w * DG + k) * 64 + l] = dg[k];
            }
            lds_barrier();
#pragma unroll
            for (int j = 0; j < NR; ++j)
#pragma unroll
                for (int k = 0; k < DG; ++k) qd[x][j][k] = meet[(j * DG + k) * 64 + l];
            if constexpr (QL > 0) {
                for (int i = w; i < QL * DG; i += 4) qlast[x][i / DG][i % DG][l] = meet[(NR * DG + i) * 64 + l];
            }
            lds_barrier();
        }
    }
    // Scores of the wave's 16 keys of full page j
    auto scores = [&](int j) __attribute__((always_inline)) {
        const h2 two = __builtin_bit_cast(h2, (uint32_t)__builtin_amdgcn_readlane(w & 2 ? scl[1] : scl[0], j & 63));
        ksc = (float)two[w & 1];
        landed<KB * NJ>();   // all but the V that went out last, and with two pages of K the K before it
        const uint8_t* from = kbuf[KB == 2 ? j & 1 : 0] + w * QUARTER + 16 * l;
        u4 k[NJ];
#pragma unroll
        for (int i = 0; i < NJ; ++i) k[i] = *(const u4*)(from + KIB * i) ^ 0x80808080u;   // signed
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            i4 a[DG];
#pragma unroll
            for (int d = 0; d < DG; ++d) a[d] = i4{};
#pragma unroll
            for (int i = 0; i < NR; ++i)
#pragma unroll
                for (int d = 0; d < DG; ++d) a[d] = mfma_i8(k[i], qd[x][i][d], a[d]);
#pragma unroll
            for (int i = 0; i < QL; ++i)
#pragma unroll
                for (int d = 0; d < DG; ++d) a[d] = mfma_i8(k[NR + i], qlast[x][i][d][l], a[d]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float t = (float)(a[0][i] * 256 + a[1][i]);   // (|sums| of a digit < 2^23)
                sc[x][i] = PAIRS ? __builtin_fmaf(t, 256.f, (float)a[DG - 1][i]) : t;
            }
        }
    };
    // Weights are 2^(s - m), with a reference m that is 7 below the row's maximum when it is set, and set anew when a weight passes
    // 2^15. So weights stay inside f16, and small ones keep their digits: hi + lo resolves 2^-24, 2^-31 of a fresh
    // maximum, and one f16 2^-24 in subnormals. `reference` takes the maxima of the page that sc holds to all waves.
    auto reference = [&]() __attribute__((always_inline)) {
        maxima();
        lds_barrier();
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            const f4 m4 = *(const f4*)mbuf[16 * x + lr];
            const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            if (mx > top[x]) {   // (from -inf at the first visible key; all waves find the same)
                const float to = P_BITS - mx;
                const float f = top[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(to - neg[x]);
                l_run[x] *= f;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[x][d][i] *= f;
                neg[x] = to;
                top[x] = 2 * P_BITS + 1 - to;
            }
        }
    };
    // The weights of the page that sc holds to LDS; returns their sums, of the weights as rounded, and whether one is too large
    struct Sums { float s[RB]; bool over; };
    auto weights = [&](int par) __attribute__((always_inline)) {
        Sums r;
        float most = 0.f;
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[x][i], back[x] * ksc, neg[x]));
            most = fmaxf(fmaxf(most, fmaxf(e[0], e[1])), fmaxf(e[2], e[3]));
            _Float16* to = &pbuf[par][x][w >> 1][0][l * 8 + 4 * (w & 1)];
            if constexpr (PAIRS) {
                h2 h0, h1, l0, l1;
                split2(f2{e[0], e[1]}, neg1, h0, l0);
                split2(f2{e[2], e[3]}, neg1, h1, l1);
                *(h4*)to = h4{h0[0], h0[1], h1[0], h1[1]};
                *(h4*)(to + 64 * 8) = h4{l0[0], l0[1], l1[0], l1[1]};
                r.s[x] = (e[0] + e[1]) + (e[2] + e[3]);
            } else {
                const h2 h0 = __builtin_convertvector((f2{e[0], e[1]}), h2);
                const h2 h1 = __builtin_convertvector((f2{e[2], e[3]}), h2);
                const h2 ones = {(_Float16)1.f, (_Float16)1.f};
                *(h4*)to = h4{h0[0], h0[1], h1[0], h1[1]};
                r.s[x] = __builtin_amdgcn_fdot2(h1, ones, __builtin_amdgcn_fdot2(h0, ones, 0.f, false), false);
            }
        }
        r.over = __any(most > 32768.f);
        return r;
    };
    // The page's weights behind a barrier, under a reference that holds them (nearly always the one that there is)
    auto settle = [&](int par) __attribute__((always_inline)) {
        Sums r = weights(par);
        if (l == 0) over[par][w] = r.over;
        lds_barrier();
        const i4 any = *(const i4*)over[par];
        if (__builtin_amdgcn_readfirstlane(any[0] | any[1] | any[2] | any[3])) {
            reference();
            r = weights(par);
            lds_barrier();
        }
#pragma unroll
        for (int x = 0; x < RB; ++x) l_run[x] += r.s[x];
    };
    // O of the wave's dims (vf: the V operand of a dim block and half of the keys)
    auto values = [&](int par, auto&& vf) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            h8 ph[RB], pl[RB];
#pragma unroll
            for (int x = 0; x < RB; ++x) {
                ph[x] = *(const h8*)&pbuf[par][x][s][0][l * 8];
                if constexpr (PAIRS) pl[x] = *(const h8*)&pbuf[par][x][s][NP - 1][l * 8];
            }
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const h8 v = vf(d, s);
#pragma unroll
                for (int x = 0; x < RB; ++x) o[x][d] = mfma16x16x32(v, ph[x], o[x][d]);
                if constexpr (PAIRS) {
#pragma unroll
                    for (int x = 0; x < RB; ++x) o[x][d] = mfma16x16x32(v, pl[x], o[x][d]);
                }
            }
        }
    };
    // Full page j: its weights, then the next page's scores and its values. K and V of a later page go out when their buffers
    // have been read: on arrival here K of j + 1 .. j + KB and V of j .. j + VB - 1 are under way or there.
    auto step = [&](int j, int par) __attribute__((always_inline)) {
        const h2 s01 = __builtin_bit_cast(h2, (uint32_t)__builtin_amdgcn_readlane(scl[2], j & 63));
        const h2 s23 = __builtin_bit_cast(h2, (uint32_t)__builtin_amdgcn_readlane(scl[3], j & 63));
        if (((j + 1) & 63) == 0) {
            load_scales();
            asm volatile("" : "+v"(scl));
        }
        unsigned vid = page_of(j + VB);
        if (((j + 1 + KB) & 63) == 0) load_ids(j + 1 + KB);
        const unsigned kid = page_of(j + 1 + KB);
        if constexpr (VB == 1 + KB) vid = kid;   // (the same page: its number may be among those just read)
        static_assert(VB <= 1 + KB, "V's page numbers are read no later than K's");
        if ((p0 + j) * kv8::PAGE + kv8::PAGE - 1 > clear) mask_keys(p0 + j);
        __builtin_amdgcn_s_setprio(0);
        settle(par);
        __builtin_amdgcn_s_setprio(1);
        scores(j + 1);   // (past the end: not used)
        fetch(c.kp, kbuf[KB == 2 ? (j + 1) & 1 : 0], j + 1 + KB, kid);
        uint8_t* vj = vbuf[VB == 2 ? j & 1 : 0];
        const uint8_t* v = vj + w * QUARTER + 16 * l;
        if constexpr (VB == 1) landed<NJ>();   // all but K of page j + 2
        values(par, [&](int d, int s) __attribute__((always_inline)) {
            const u2 r = *(const u2*)(v + KIB * d + 8 * s);
            const h2 f = s ? s23 : s01;
            const h4 f0 = {f[0], f[0], f[0], f[0]}, f1 = {f[1], f[1], f[1], f[1]};
            return cat_h4(codes4(r[0]) * f0, codes4(r[1]) * f1);
        });
        fetch(c.vp, vj, j + VB, vid);
    };
    if (np > 0) asm volatile("" : "+v"(scl));
    int par = 0;
    h8 vo[ND][2];
    if (tail) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) vo[d][e] = ld_h8(c.tv + open + KIB * d + 8 * e);
        mask_keys(closed);
        reference();
        const Sums r = weights(0);   // (none too large)
        lds_barrier();
#pragma unroll
        for (int x = 0; x < RB; ++x) l_run[x] += r.s[x];
        par = 1;
    }
    if (np > 0) {
        if constexpr (VB == 1) landed<0>();
        scores(0);
        fetch(c.kp, kbuf[0], KB, page_of(KB));
        fetch(c.vp, vbuf[VB - 1], VB - 1, page_of(VB - 1));
    }
    if (tail) {
        const int have = total - closed * kv8::PAGE;   // rows that are not there hold anything
        values(0, [&](int d, int s) __attribute__((always_inline)) {
            h8 v = vo[d][s];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (32 * s + 16 * (i >> 2) + 4 * g + (i & 3) >= have) v[i] = (_Float16)0.f;
            return v;
        });
    }
    if (np > 0 && (!tail || closed * kv8::PAGE > clear)) {   // rows without a reference: all, or those that see no open row
        if (p0 * kv8::PAGE + kv8::PAGE - 1 > clear) mask_keys(p0);
        reference();   // (behind the open page's values: it rescales O)
    }
    for (int j = 0; j < np; ++j) step(j, (j + par) & 1);
    landed<0>();   // the fetches past the end

    // ---- sums over the key blocks, then the rows out
#pragma unroll
    for (int x = 0; x < RB; ++x) lbuf[16 * x + lr][w] = sum_xor32(sum_xor16(l_run[x]));
    lds_barrier();
    if (u.ns > 1) {
        const int nrec = kv8::max_records(wgs), rec = u.rec + kv8::record(split, u.nrb, rb, nkv, kh);
        if (rec >= nrec) return;   // (cannot be: see max_records)
        f2* ml = (f2*)part + (size_t)rec * ROWS;
        float* po = part + (size_t)nrec * ROWS * 2 + (size_t)rec * ROWS * HD;
#pragma unroll
        for (int x = 0; x < RB; ++x) {
            const int row = 16 * x + lr;
            if (r0 + row >= R) continue;
            const f4 s4 = *(const f4*)lbuf[row];
            if (w == 0 && g == 0) ml[row] = f2{top[x] == -INFINITY ? -INFINITY : -neg[x], (s4[0] + s4[1]) + (s4[2] + s4[3])};
#pragma unroll
            for (int d = 0; d < ND; ++d) *(f4*)(po + (size_t)row * HD + 16 * (ND * w + d) + 4 * g) = o[x][d];
        }
        return;
    }
#pragma unroll
    for (int x = 0; x < RB; ++x) {
        const int r = r0 + 16 * x + lr;
        if (r >= R) continue;
        const f4 s4 = *(const f4*)lbuf[16 * x + lr];
        const float inv = 1.0f / ((s4[0] + s4[1]) + (s4[2] + s4[3]));
        const int t = token(16 * x + lr), h = kh * G + r - t * G;
        const float* gates = q + (size_t)(u.t0 + t) * qts + (size_t)h * 2 * HD + HD;
        OutT* to = out + (size_t)(u.t0 + t) * ots + (size_t)h * HD;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int dim = 16 * (ND * w + d) + 4 * g;
            const f4 gate = ld_f4(gates + dim);
            f4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = o[x][d][i] * inv * sigmoid_hw(gate[i]);
            store4(to + dim, v);
        }
    }
}

// Joins the records of sequences with more than one split. A workgroup takes (group of rows, row, 4 DL dims), with 256 / DL split
// lanes; where DL is 32 and a sequence has few splits, each of its waves takes a row alone, and fewer workgroups do. NB records are
// in flight a thread. rows: those that a group can have. The launch is as many workgroups as there can be items, or fewer,
// each taking several; groups come side by side, so that those with work are spread.
template <int HD, int ROWS, int DL, class OutT>
__global__ __launch_bounds__(256) void attn_kv8_merge_kernel(Kv8 c, Kv8Batch b, const float* __restrict__ q, int qts,
                                                             int G, OutT* __restrict__ out, int ots,
                                                             const float* __restrict__ part, int wgs, int rows) {
    constexpr int SL = 256 / DL, DQ = HD / (4 * DL), NB = 4, ALONE = DL == 32 ? 16 : 0, WL = HD / 4;   // WL: lanes of a wave's row
    __shared__ float red_m[4], red_l[4][DL];
    __shared__ __align__(16) f4 red_o[4][DL];
    const int nkv = c.nkv, kh = blockIdx.x, tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const Kv8Seq s0 = kv8_seq(b, l);
    const int chunk = call_chunk<ROWS>(b, s0, G, nkv, wgs, l);
    const int nrec = kv8::max_records(wgs);
    // weight of a record or partial result whose maximum is m, against the largest M
    auto share = [](float m, float sum, float M) { return m == -INFINITY ? (sum == 0.f ? 0.f : NAN) : __builtin_amdgcn_exp2f(m - M); };
    struct Part { float m, sum; f4 o; };
    int groups = 0;          // row blocks that were split
    bool alone_all = true;   // and all into few
    for (int i0 = 0; i0 < b.nseq; i0 += 64) {
        const Kv8Seq s = i0 == 0 ? s0 : kv8_seq(b, i0 + l);
        const int ns = kv8::splits(s.pages, chunk), n = ns > 1 ? (s.n * G + ROWS - 1) / ROWS : 0;
        groups += b.nseq == 1 ? __builtin_amdgcn_readfirstlane(n) : __builtin_amdgcn_readlane(prefix_sum(n), 63);
        if (__any(n > 0 && ns > ALONE)) alone_all = false;
    }
    const int each = alone_all ? (rows + 3) / 4 : DQ * rows;
    const float rcp_groups = __builtin_amdgcn_rcpf((float)groups), rcp_G = __builtin_amdgcn_rcpf((float)G);
    for (int item = blockIdx.y; item < groups * each; item += gridDim.y) {   // (at most 520 groups of 128)
        const int sub = div_small(item, rcp_groups);
        const Found u = find<ROWS, true>(b, s0, G, nkv, chunk, item - sub * groups, l);
        if (!u.any) return;   // (cannot be)
        const bool alone = u.ns <= ALONE;
        const int rb = u.at, row = alone ? 4 * sub + w : sub / DQ, r = rb * ROWS + row;
        if (row >= rows || r >= u.n * G) continue;   // (all threads that join the row)
        const int t = u.nrb == 1 ? div_small(row, rcp_G) : (int)((unsigned)r / (unsigned)G), h = kh * G + r - t * G;
        const int last = (u.len + t) / kv8::PAGE, need = (chunk == 1 ? last : (int)((unsigned)last / (unsigned)chunk)) + 1;
        const float* base = part + (size_t)nrec * ROWS * 2;
        const int dim = 4 * (alone ? l % WL : DL * (sub % DQ) + tid % DL);
        const f4 gate = ld_f4(q + (size_t)(u.t0 + t) * qts + (size_t)h * 2 * HD + HD + dim);   // (beside the records)
        auto gather = [&](int first, int lanes) __attribute__((always_inline)) {
            Part p = {-INFINITY, 0.f, f4{}};
            for (int s = first; s < need; s += lanes * NB) {   // (past the last record: the last again, uncounted)
                f2 ml[NB];
                f4 v[NB];
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const size_t at = (size_t)(u.rec + kv8::record(min(s + i * lanes, need - 1), u.nrb, rb, nkv, kh)) * ROWS + row;
                    ml[i] = *((const f2*)part + at);
                    v[i] = ld_f4(base + at * HD + dim);
                }
                float M = p.m;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    if (s + i * lanes >= need) ml[i] = f2{-INFINITY, 0.f};
                    M = fmaxf(M, ml[i][0]);
                }
                const float a = share(p.m, p.sum, M);
                p.sum *= a;
                p.o *= a;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const float e = share(ml[i][0], ml[i][1], M);
                    p.sum += ml[i][1] * e;
                    if (s + i * lanes < need) p.o += v[i] * e;
                }
                p.m = M;
            }
            return p;
        };
        auto finish = [&](const Part& p) __attribute__((always_inline)) {
            const float inv = 1.0f / p.sum;
            f4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = p.o[i] * inv * sigmoid_hw(gate[i]);
            store4(out + (size_t)(u.t0 + t) * ots + (size_t)h * HD + dim, v);
        };
        // p against the largest M of the lanes it is joined with
        auto scaled = [&](Part p, float M) __attribute__((always_inline)) {
            const float e = share(p.m, p.sum, M);
            return Part{M, p.sum * e, p.o * e};
        };
        if (alone) {
            Part p = gather(l / WL, 64 / WL);
            if constexpr (WL == 32) {
                p = scaled(p, max_xor32(p.m));
                p.sum = sum_xor32(p.sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) p.o[i] = sum_xor32(p.o[i]);
            }
            if (l < WL) finish(p);
            continue;
        }
        // the split lanes of a wave, then the four waves
        Part p = gather(tid / DL, SL);
        float M = max_xor32(p.m);
        if constexpr (DL == 8) {
            M = max_xor16(M);
            M = fmaxf(M, dppc<0x128>(M));   // row_ror 8
        }
        p = scaled(p, M);
        float all[5] = {p.sum, p.o[0], p.o[1], p.o[2], p.o[3]};
#pragma unroll
        for (int i = 0; i < 5; ++i) {
            all[i] = sum_xor32(all[i]);
            if constexpr (DL == 8) {
                all[i] = sum_xor16(all[i]);
                all[i] += dppc<0x128>(all[i]);
            }
        }
        __syncthreads();   // the last item's partial results have been read
        if (l < DL) {
            if (l == 0) red_m[w] = M;
            red_l[w][l] = all[0];
            red_o[w][l] = f4{all[1], all[2], all[3], all[4]};
        }
        __syncthreads();
        if (tid < DL) {
            M = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
            p = Part{M, 0.f, f4{}};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = share(red_m[i], red_l[i][tid], M);
                p.sum += red_l[i][tid] * f;
                p.o += red_o[i][tid] * f;
            }
            finish(p);
        }
    }
}

constexpr int WGS = 512;   // workgroups that a call's pages are shared out to: two a CU, as many as fit side by side

// Row blocks of 16 rb rows that the sequences of a call can have, of a KV head
long max_groups(int rb, int nseq, int ntok, int max_nt, int G) {
    const long rows = 16 * rb, each = ((long)max_nt * G + rows - 1) / rows;
    return std::min((long)ntok * G / rows + std::min(nseq, ntok), each * nseq);
}
// Groups of 16 rows that share a workgroup's pages. One, if there are no more rows, or up to four times as many over tables of
// few pages: then several workgroups with a short way to their pages are sooner than one with a long way. Else all of a sequence's
// rows up to 32; of more, blocks of 32 have the shorter steps and the sooner first page, blocks of 48 or 64 (f16 outputs: more do
// not fit the registers) fewer conversions of V a row, so the large ones where there are enough of them to fill the card, by
// the most that the call's shapes allow. 64 for full batches of few tokens that it divides better; 48 else, which leave more of
// q in registers and share out the unlike blocks of a prompt more evenly.
// us (16 heads, 2 KV heads, hd 256; tokens after rows):
//   16 / 32, f32, in a graph    4 after 508   10.8 / 12.4    4 after 8188   15.4 / 16.5    8 after 504   12.7 / 14.5    4 after 131068   51.7 / 43.5
//   32 / 48 / 64, f16   64 after 4032   30 / - / 37    256 after 3840   47 / 45 / 51    256 after 32512   233 / 192 / 192    2048 after 0   68 / 60 / 78
//                       8192 after 0   734 / 619 / 626    512 after 32256   467 / 394 / 376    32 sequences of 5 after 8187   94 / 63 / 68
//                       of 8 after 8184   95 / 98 / 75    of 64 after 1984   118 / 113 / 100    1000 after 3000, 24 heads   - / 112 / 139
//   32 / 48, f32   64 after 4032   32 / 36    512 after 3584   86 / 88    4096 after 0   265 / 262    32 of 5 after 8187   106 / 83
//                  seven prompts of 24 heads   461 / 435
// (512 tokens after 32256 are the one size seen where 48 rows, f16, are behind 64, by 2 to 5 %; 256 after 32512 180 / 183, 1000 after
// 16000 386 / 460.) The tables' widths count, not the lengths, which the host has not: 4 tokens after 508 rows 10.5 where the tables
// have 10 pages, 12.1 where they have 2049.
int row_groups(const Kv8Batch& b, int G, int nkv, bool f16out) {
    const long rows = (long)b.max_nt * G;
    if (rows <= 16 || (rows <= 64 && (long)std::min(b.nseq, b.ntok) * nkv * b.max_pages < WGS)) return 1;
    if (rows <= 32) return 2;
    const long groups = max_groups(f16out ? 4 : 3, b.nseq, b.ntok, b.max_nt, G) * nkv;
    if (!f16out) return groups >= 2048 || (rows <= 48 && groups >= 32) ? 3 : 2;
    if (groups < 64) return 2;
    const bool full = b.nseq > 1 && (long)b.nseq * b.max_nt == b.ntok && rows <= 1024;
    return full && (rows + 63) / 64 * 64 <= (rows + 47) / 48 * 48 ? 4 : 3;
}

template <int HD, int RB, class OutT>
hipError_t launch(const Kv8& c, const Kv8Batch& b, const float* q, int qts, int nh, float scale, OutT* out, int ots,
                  float* part, hipStream_t st) {
    const int G = nh / c.nkv;
    const long groups = max_groups(RB, b.nseq, b.ntok, b.max_nt, G), units = std::min(groups + (WGS + c.nkv - 1) / c.nkv + 1, groups * b.max_pages);
    const long fold = (units + 65534) / 65535;
    constexpr bool pairs = sizeof(OutT) == 4 || RB == 1;   // (see the top: in blocks of 16 rows fewer bits save next to nothing)
    attn_kv8_kernel<HD, RB, pairs, OutT>
        <<<dim3(c.nkv, (unsigned)((units + fold - 1) / fold), (unsigned)fold), 256, 0, st>>>(c, b, q, qts, G, scale, out, ots, part, WGS);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // split groups have two splits at least, so there are at most max_records / 2 of them. Few rows: many splits, so many
    // split lanes
    const int rows = (int)std::min((long)16 * RB, (long)b.max_nt * G);
    const long split_rows = std::min(groups, (long)kv8::max_records(WGS) / 2 / c.nkv + 1) * rows, most = std::max(2048 / c.nkv, 1);
    if (split_rows * c.nkv * (HD / 32) <= 1024)
        attn_kv8_merge_kernel<HD, 16 * RB, 8, OutT><<<dim3(c.nkv, (unsigned)(split_rows * (HD / 32))), 256, 0, st>>>(
            c, b, q, qts, G, out, ots, part, WGS, rows);
    else
        attn_kv8_merge_kernel<HD, 16 * RB, 32, OutT><<<dim3(c.nkv, (unsigned)std::min(split_rows * (HD / 128), most)), 256, 0, st>>>(
            c, b, q, qts, G, out, ots, part, WGS, rows);
    return hipGetLastError();
}
template <int HD, class OutT>
hipError_t launch_rb(const Kv8& c, const Kv8Batch& b, const float* q, int qts, int nh, float scale, OutT* out, int ots,
                     float* part, hipStream_t st) {
    const int rb = row_groups(b, nh / c.nkv, c.nkv, sizeof(OutT) == 2);
    if (rb == 1) return launch<HD, 1, OutT>(c, b, q, qts, nh, scale, out, ots, part, st);
    if (rb == 2) return launch<HD, 2, OutT>(c, b, q, qts, nh, scale, out, ots, part, st);
    if constexpr (sizeof(OutT) == 2) {
        if (rb == 4) return launch<HD, 4, OutT>(c, b, q, qts, nh, scale, out, ots, part, st);
    }
    return launch<HD, 3, OutT>(c, b, q, qts, nh, scale, out, ots, part, st);
}

}  // namespace

size_t attn_kv8_scratch_bytes(int max_nt, int hd, int nh, int nkv) {
    const long rows = (long)max_nt * (nh / nkv);
    const int rb = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;   // (the most that `row_groups` takes, for any number of sequences)
    return (size_t)kv8::max_records(WGS) * 16 * rb * (hd + 2) * sizeof(float);
}
hipError_t launch_attn_kv8(const Kv8& c, const Kv8Batch& b, const float* q, int qts, int nh, float scale, void* out,
                           int ots, bool f16out, float* part, hipStream_t st) {
    if (f16out) {
        _Float16* o = (_Float16*)out;
        return c.hd == 256 ? launch_rb<256>(c, b, q, qts, nh, scale, o, ots, part, st)
                           : launch_rb<128>(c, b, q, qts, nh, scale, o, ots, part, st);
    }
    float* o = (float*)out;
    return c.hd == 256 ? launch_rb<256>(c, b, q, qts, nh, scale, o, ots, part, st)
                       : launch_rb<128>(c, b, q, qts, nh, scale, o, ots, part, st);
}

}  // namespace it
