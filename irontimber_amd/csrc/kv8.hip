// The paged 8-bit K/V cache: rows appended and quantised, rows read back, pages and open rows copied.
//
// A page holds 64 rows of every KV head; each block of 16 rows and head has one scale s for K and one for V, and a value is
// (code - 128) * s. s has four significant bits (or is a multiple of 2^-24), so code * s has eleven: every stored value is an
// f16 number, and what reads the cache computes with exact operands. s is the block's largest size / 127 rounded up,
// which costs 1/16 of a step on average (1/8 at most) against 127 steps exactly.
// A scale belongs to whole blocks, so a page is quantised once, when its last row arrives; until then its rows stand in
// the sequence's open buffer, in f16 and in the page's own element order. That buffer has room for two pages, so that a call's rows
// that are taken back (drafts that a check rejects) need nothing but a smaller length.
#include "internal.h"
#include "kv8.h"

namespace it {
namespace {

// The largest size among 8 values, as f16 bits (of two halves: the packed maximum), which order as the sizes do; 0x7C00 and up:
// one is not finite.
__device__ __forceinline__ uint32_t sizes(h8 x) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    const u4 u = __builtin_bit_cast(u4, x) & 0x7FFF7FFFu;
    const us2 a = __builtin_elementwise_max(__builtin_bit_cast(us2, (uint32_t)u[0]), __builtin_bit_cast(us2, (uint32_t)u[1]));
    const us2 b = __builtin_elementwise_max(__builtin_bit_cast(us2, (uint32_t)u[2]), __builtin_bit_cast(us2, (uint32_t)u[3]));
    const us2 m = __builtin_elementwise_max(a, b);
    return m[0] > m[1] ? m[0] : m[1];
}
__device__ __forceinline__ float size_of(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (unsigned short)bits); }
// An infinity is stored as the largest f16, a NaN as 0: a value that no query may see must not reach its products.
__device__ __forceinline__ h8 finite8(h8 x) {
    if (__any(sizes(x) >= 0x7C00u)) {
        const _Float16 top = (_Float16)65504.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const _Float16 v = x[i];
            x[i] = v != v ? (_Float16)0.f : v > top ? top : v < -top ? -top : v;
        }
    }
    return x;
}
// A block's scale from its largest size. amax has 11 bits and 127 * s 11, so they differ by 2^-15 or not at all, and the
// rounded quotient falls on the same side of s as the exact one.
__device__ __forceinline__ float block_scale(float amax) {
    const float t = amax / 127.0f;
    if (t < 0x1p-21f) return fmaxf(ceilf(t * 0x1p24f), 1.0f) * 0x1p-24f;
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, t) + 0xFFFFFu) & ~0xFFFFFu);
}
// Steps of a block: x / s to the nearest, ties to even, at most 127 (113 at s = 576, the one scale above 512: more is no f16).
// The quotient is x * (1 / s) with one correction by the residual, which is exact: a tie comes out as one, and no other
// quotient is nearer to a tie than 2^-13. 
struct Steps {
    float s, inv, top;
    __device__ __forceinline__ explicit Steps(float scale) : Steps(scale, 1.0f / scale) {}
    __device__ __forceinline__ Steps(float scale, float inverse) : s(scale), inv(inverse), top(scale > 512.f ? 113.f : 127.f) {}
    __device__ __forceinline__ float of(_Float16 v) const {
        const float x = (float)v, q = x * inv;
        return __builtin_amdgcn_fmed3f(rintf(__builtin_fmaf(__builtin_fmaf(-q, s, x), inv, q)), -top, top) + 128.f;
    }
};
// Codes of four values, the first lowest
__device__ __forceinline__ uint32_t codes_of(const Steps& t, _Float16 a, _Float16 b, _Float16 c, _Float16 d) {
    uint32_t u = __builtin_amdgcn_cvt_pk_u8_f32(t.of(a), 0, 0);
    u = __builtin_amdgcn_cvt_pk_u8_f32(t.of(b), 1, u);
    u = __builtin_amdgcn_cvt_pk_u8_f32(t.of(c), 2, u);
    return __builtin_amdgcn_cvt_pk_u8_f32(t.of(d), 3, u);
}

// Workgroup = (sequence, touched page or half of the open buffer, KV head, K or V). A page is quantised if the call fills it;
// a half takes the new rows of its page among the last two. Where it still holds old rows that the first page needs and that
// another page's rows replace, the first page's workgroup writes it, after it has read them.
// Both kinds work in the page's order, which the old open rows have already. New rows of V get there through LDS.
// A wave U = 2 KiB of codes, 32 values a lane: with more to a wave the call is as slow as the fetching of the code that each CU then
// runs once or twice, with less as the starting of its waves (U 1, 2, 4: 8192 rows 12.1, 10.8, 11.3 us, one page 5.3, 5.0, 5.8,
// in a graph of three inputs, which the last cache holds, on one card; U 2 over twelve inputs 12.1, by the profiler 11.6, a page 5.4).
// Bound by bytes, two read and one written a value, and in short calls by three dependent round trips (bounds, rows, stores).
template <int HD>
__global__ __launch_bounds__(2 * HD) void kv8_append_kernel(Kv8 c, Kv8Batch b, const _Float16* __restrict__ k,
                                                            const _Float16* __restrict__ v, int kts) {
    constexpr int NT = 2 * HD, NW = NT / 64, U = 2, CH = HD / 8, PITCH = HD + 8;   // (rows four apart in LDS: 16 banks apart)
    __shared__ __align__(16) _Float16 tile[kv8::PAGE * PITCH];
    __shared__ float most[HD / 16][4];
    const int i = blockIdx.z, kh = blockIdx.y >> 1, which = blockIdx.y & 1, j = (int)blockIdx.x - 2;   // -2, -1: halves
    const Kv8Seq s = kv8_seq(b, i);
    if (s.n == 0 || s.bad) return;
    const int first = s.len / kv8::PAGE, p = first + j, total = s.len + s.n, last = (total - 1) / kv8::PAGE;
    if (p > last) return;
    const bool behind = s.len % kv8::PAGE != 0 && last >= first + 2;   // half first % 2 is written behind page `first`
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, lr = l & 15;
    const _Float16* src = (which ? v : k) + (size_t)s.t0 * kts + (size_t)kh * HD;   // token t at t * kts
    _Float16* open = (which ? c.tv : c.tk) + ((size_t)i * 2 * c.nkv + kh) * (kv8::PAGE * HD);
    const size_t half = (size_t)c.nkv * kv8::PAGE * HD;
    // Rows from .. to - 1 of V, from row0 on, into the tile, a row of 8 dims a thread and turn
    auto stage = [&](int row0, int from, int to) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < 2 * U; ++n) {
            const int row = row0 + (n * NT + tid) / CH, ch = tid % CH;
            if (row >= from && row < to)
                *(h8*)(tile + (row - row0) * PITCH + 8 * ch) = finite8(ld_h8(src + (size_t)(row - s.len) * kts + 8 * ch));
        }
    };
    // This lane's four rows of each block and one dim of dim block kib, from the tile where they are from .. to - 1, else x
    auto pick = [&](int kib, int row0, int from, int to, h8 (&x)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int r = 16 * (e >> 2) + 4 * g + (e & 3);
            const _Float16 z = tile[r * PITCH + 16 * kib + lr];
            x[e >> 3][e & 7] = row0 + r >= from && row0 + r < to ? z : x[e >> 3][e & 7];
        }
    };
    const int row0 = p * kv8::PAGE;
    if (j >= 0 && row0 + kv8::PAGE <= total) {
        const int id = b.table[(size_t)i * b.max_pages + p];
        const bool known = (unsigned)id < (unsigned)c.npages;
        const size_t unit = known ? (size_t)id * c.nkv + kh : 0;
        const _Float16* old = open + (p & 1) * half + (w * 64 + l) * 16;   // (KiB w + NW u: 1024 NW u on)
        h8 x[U][2] = {};
        if (!which) {
            // KiB = (block, 64 dims): each lane holds two runs of 8 dims of a row
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kib = w + NW * u, row = row0 + 16 * (kib / (HD / 64)) + lr, dim = 64 * (kib % (HD / 64)) + 8 * g;
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[u][h] = finite8(ld_h8(row >= s.len ? src + (size_t)(row - s.len) * kts + dim + 32 * h : old + NW * 1024 * u + 8 * h));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float m = wave_max(size_of(max(sizes(x[u][0]), sizes(x[u][1]))));
                if (l == 0) most[w + NW * u][0] = m;
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int kib = w + NW * u, a = kib / (HD / 64);
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < HD / 64; ++n) top = fmaxf(top, most[a * (HD / 64) + n][0]);
                const Steps t(block_scale(top));
                if (known) {
                    u4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const h8 z = x[u][e >> 1];
                        const int o = 4 * (e & 1);
                        y[e] = codes_of(t, z[o], z[o + 1], z[o + 2], z[o + 3]);
                    }
                    *(u4*)(c.kp + unit * (kv8::PAGE * HD) + (kib * 64 + l) * 16) = y;
                    if (l == 0 && kib % (HD / 64) == 0) c.sc[unit * 8 + a] = (_Float16)t.s;
                }
            }
        } else {
            if (row0 < s.len) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    x[u][0] = ld_h8(old + NW * 1024 * u);
                    x[u][1] = ld_h8(old + NW * 1024 * u + 8);
                }
            }
            stage(row0, s.len, total);
            __syncthreads();
#pragma unroll
            for (int u = 0; u < U; ++u) pick(w + NW * u, row0, s.len, total, x[u]);
            // largest sizes of the four blocks, lane row g ending with block g, then one lane in four with each wave's
            float m[4];
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                uint32_t most_bits = 0;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    h8 z = {};
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[e] = x[u][a >> 1][4 * (a & 1) + e];
                    most_bits = max(most_bits, sizes(z));
                }
                m[a] = size_of(most_bits);
            }
            swap32(m[0], m[2]);
            swap32(m[1], m[3]);
            float m0 = fmaxf(m[0], m[2]), m1 = fmaxf(m[1], m[3]);
            swap16(m0, m1);
            m0 = fmaxf(m0, m1);
            m0 = fmaxf(m0, dppc<0xB1>(m0));
            m0 = fmaxf(m0, dppc<0x4E>(m0));
            m0 = fmaxf(m0, dppc<0x141>(m0));
            m0 = fmaxf(m0, dppc<0x140>(m0));
            if (lr == 0) most[w][2 * (g >> 1) + (g & 1)] = m0;
            __syncthreads();
            m0 = most[min(l >> 2, NW - 1)][l & 3];
            m0 = fmaxf(m0, dppc<0x124>(m0));   // row_ror 4, 8
            m0 = fmaxf(m0, dppc<0x128>(m0));
            const Steps mine(block_scale(max_xor32(max_xor16(m0))));   // of block l % 4
            if (known && tid < 4) c.sc[unit * 8 + 4 + tid] = (_Float16)mine.s;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                u4 y;
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const Steps t(readlane_f(mine.s, a), readlane_f(mine.inv, a));
                    const h8 z = x[u][a >> 1];
                    const int o = 4 * (a & 1);
                    y[a] = codes_of(t, z[o], z[o + 1], z[o + 2], z[o + 3]);
                }
                if (known) *(u4*)(c.vp + unit * (kv8::PAGE * HD) + ((w + NW * u) * 64 + l) * 16) = y;
            }
        }
        __syncthreads();   // old open rows read before the half is written below, and the tile before it is filled anew
    }
    if (j > 0 || (j == 0 && !behind)) return;
    const int parity = j < 0 ? j + 2 : first & 1, pt = last - ((last ^ parity) & 1);   // the half's page among the last two
    if (pt < first || (j < 0 && behind && parity == (first & 1))) return;
    const int r0 = pt * kv8::PAGE, from = max(s.len, r0), to = (int)min((long)total, (long)r0 + kv8::PAGE);
    _Float16* dst = open + (pt & 1) * half;
    if (!which || to - from <= 4) {
        for (int n = tid; n < (to - from) * CH; n += NT) {
            const int row = from + n / CH, ch = n % CH;
            const h8 x = finite8(ld_h8(src + (size_t)(row - s.len) * kts + 8 * ch));
            if (!which) {
                *(h8*)(dst + kv8::k_elem(HD, row - r0, 8 * ch)) = x;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) dst[kv8::v_elem(row - r0, 8 * ch + e)] = x[e];
            }
        }
        return;
    }
    // many rows of V: through LDS, in whole pieces of the page's order that keep the rows before `from`; the rows from `to` on
    // hold anything
    h8* piece = (h8*)(dst + (w * 64 + l) * 16);   // (KiB w + NW u: 128 NW u on)
    h8 x[U][2] = {};
    if (from > r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x[u][0] = piece[NW * 128 * u];
            x[u][1] = piece[NW * 128 * u + 1];
        }
    }
    stage(r0, from, to);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
        pick(w + NW * u, r0, from, to, x[u]);
        piece[NW * 128 * u] = x[u][0];
        piece[NW * 128 * u + 1] = x[u][1];
    }
}

// Workgroup = (sequence, page, KV head, K or V): rows first[i] .. of a sequence that holds len[i] rows, as f16.
// A wave two KiB, as in appending (four waves of four KiB, one after the other: a page 4.2 us, so 3.4; 8192 rows 8.2, so 7.6, taken as
// there; over twelve inputs 8.7, by the profiler 7.9, a page 3.9).
template <int HD>
__global__ __launch_bounds__(2 * HD) void kv8_read_kernel(Kv8 c, Kv8Batch b, const int* __restrict__ first,
                                                       _Float16* __restrict__ k, _Float16* __restrict__ v, int kts) {
    constexpr int NT = 2 * HD, NW = NT / 64, U = 2, CH = HD / 8, PITCH = HD + 8;
    __shared__ __align__(16) _Float16 tile[kv8::PAGE * PITCH];
    const int i = blockIdx.z, kh = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int t0 = b.start[i], t1 = b.start[i + 1], r0 = first[i], total = b.len[i];
    if (t0 < 0 || t1 > b.ntok || t1 <= t0) return;
    const int count = min(t1 - t0, b.max_nt);
    if (r0 < 0 || total < 0 || total > (long)b.max_pages * kv8::PAGE) {   // rows that cannot be: NaN (grid.x * 64 >= count)
        const uint32_t nans = 0x7E007E00u;
        _Float16* lost = (which ? v : k) + (long)t0 * kts + (size_t)kh * HD;
        for (int n = threadIdx.x; n < kv8::PAGE * CH; n += NT) {
            const int row = (int)blockIdx.x * kv8::PAGE + n / CH;
            if (row < count) *(u4*)(lost + (long)row * kts + 8 * (n % CH)) = u4{nans, nans, nans, nans};
        }
        return;
    }
    const int r1 = (int)min((long)total, (long)r0 + count);   // one past the last row
    const int p = r0 / kv8::PAGE + blockIdx.x, row0 = p * kv8::PAGE;
    if ((long)p * kv8::PAGE >= r1) return;
    const int lo = max(r0, row0) - row0, hi = min(r1 - row0, kv8::PAGE);       // rows of the page
    const int tid = threadIdx.x, l = tid & 63, w = tid >> 6;
    _Float16* dst = (which ? v : k) + ((long)t0 + row0 - r0) * kts + (size_t)kh * HD;   // row r of the page at r * kts
    const bool is_open = p == total / kv8::PAGE;
    const _Float16* open = (which ? c.tv : c.tk) + (((size_t)i * 2 + (p & 1)) * c.nkv + kh) * (kv8::PAGE * HD);
    const int id = is_open ? 0 : b.table[(size_t)i * b.max_pages + p];
    const bool known = (unsigned)id < (unsigned)c.npages;
    const size_t unit = known ? (size_t)id * c.nkv + kh : 0;
    const uint8_t* page = (which ? c.vp : c.kp) + unit * (kv8::PAGE * HD);
    const _Float16 bad = __builtin_bit_cast(_Float16, (uint16_t)0x7E00);   // a page that the pool has not: NaN
    const _Float16* sc = c.sc + unit * 8 + 4 * which;
    // this wave's KiB w and w + NW of the page, both under way at once
    h8 x[U][2];
    if (is_open) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x[u][0] = ld_h8(open + ((w + NW * u) * 64 + l) * 16);
            x[u][1] = ld_h8(open + ((w + NW * u) * 64 + l) * 16 + 8);
        }
    } else {
        u4 y[U];
        const h4 four = *(const h4*)sc;
#pragma unroll
        for (int u = 0; u < U; ++u) y[u] = *(const u4*)(page + ((w + NW * u) * 64 + l) * 16);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const h4 z = codes4(y[u][a]);
                const _Float16 f = known ? which ? four[a] : sc[(w + NW * u) / (HD / 64)] : bad;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][a >> 1][4 * (a & 1) + e] = z[e] * f;
            }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int n = w + NW * u;
        if (!which) {
            const int row = 16 * (n / (HD / 64)) + (l & 15), dim = 64 * (n % (HD / 64)) + 8 * (l >> 4);
            if (row >= lo && row < hi) {
                *(h8*)(dst + (long)row * kts + dim) = x[u][0];
                *(h8*)(dst + (long)row * kts + dim + 32) = x[u][1];
            }
        } else {
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    tile[(16 * a + 4 * (l >> 4) + e) * PITCH + 16 * n + (l & 15)] = x[u][a >> 1][4 * (a & 1) + e];
        }
    }
    if (!which) return;   // (whole workgroup)
    __syncthreads();
    for (int n = tid; n < (hi - lo) * CH; n += NT) {
        const int row = lo + n / CH, ch = n % CH;
        *(h8*)(dst + (long)row * kts + 8 * ch) = *(const h8*)(tile + row * PITCH + 8 * ch);
    }
}

// Workgroup = one KV head's K or V of a page pair, or of a half of the open rows of a sequence pair. Bound by bytes.
template <int HD>
__global__ __launch_bounds__(256) void kv8_copy_kernel(Kv8 c, const int* __restrict__ src, const int* __restrict__ dst,
                                                       int n, const int* __restrict__ seq_src,
                                                       const int* __restrict__ seq_dst) {
    constexpr int QP = kv8::PAGE * HD / 16 / 256;   // 16-byte pieces a thread of a page and head
    const int tid = threadIdx.x, per = 2 * c.nkv;
    long id = blockIdx.x;
    if (id < (long)n * per) {
        const int pair = (int)(id / per), which = (int)(id % per) / c.nkv, kh = (int)(id % c.nkv);
        const int from = src[pair], to = dst[pair];
        if ((unsigned)from >= (unsigned)c.npages || (unsigned)to >= (unsigned)c.npages || from == to) return;
        uint8_t* p = which ? c.vp : c.kp;
        const size_t uf = (size_t)from * c.nkv + kh, ut = (size_t)to * c.nkv + kh;
        const u4* x = (const u4*)(p + uf * (kv8::PAGE * HD));
        u4* y = (u4*)(p + ut * (kv8::PAGE * HD));
        u4 r[QP];
#pragma unroll
        for (int e = 0; e < QP; ++e) r[e] = x[e * 256 + tid];
#pragma unroll
        for (int e = 0; e < QP; ++e) y[e * 256 + tid] = r[e];
        if (tid == 0) *(u2*)(c.sc + ut * 8 + 4 * which) = *(const u2*)(c.sc + uf * 8 + 4 * which);
        return;
    }
    id -= (long)n * per;
    const int per2 = 4 * c.nkv, pair = (int)(id / per2), rest = (int)(id % per2), which = rest / (2 * c.nkv);
    const int from = seq_src[pair], to = seq_dst[pair];
    if ((unsigned)from >= (unsigned)c.nseq || (unsigned)to >= (unsigned)c.nseq || from == to) return;
    _Float16* p = which ? c.tv : c.tk;
    const size_t part = rest % (2 * c.nkv);
    const u4* x = (const u4*)(p + ((size_t)from * 2 * c.nkv + part) * (kv8::PAGE * HD));
    u4* y = (u4*)(p + ((size_t)to * 2 * c.nkv + part) * (kv8::PAGE * HD));
    u4 r[2 * QP];
#pragma unroll
    for (int e = 0; e < 2 * QP; ++e) r[e] = x[e * 256 + tid];
#pragma unroll
    for (int e = 0; e < 2 * QP; ++e) y[e * 256 + tid] = r[e];
}

}  // namespace

// Pages that rows of one sequence can touch
static int touched(int rows) { return (int)(((long)rows + 2 * (kv8::PAGE - 1)) / kv8::PAGE); }

hipError_t launch_kv8_append(const Kv8& c, const Kv8Batch& b, const uint16_t* k, const uint16_t* v, int kts,
                             hipStream_t st) {
    const dim3 grid(2 + touched(b.max_nt), 2 * c.nkv, b.nseq);
    const auto *kk = (const _Float16*)k, *vv = (const _Float16*)v;
    if (c.hd == 256) kv8_append_kernel<256><<<grid, 512, 0, st>>>(c, b, kk, vv, kts);
    else kv8_append_kernel<128><<<grid, 256, 0, st>>>(c, b, kk, vv, kts);
    return hipGetLastError();
}
hipError_t launch_kv8_read(const Kv8& c, const Kv8Batch& b, const int* first, uint16_t* k, uint16_t* v, int kts,
                           hipStream_t st) {
    const dim3 grid(touched(b.max_nt), 2 * c.nkv, b.nseq);
    auto *kk = (_Float16*)k, *vv = (_Float16*)v;
    if (c.hd == 256) kv8_read_kernel<256><<<grid, 512, 0, st>>>(c, b, first, kk, vv, kts);
    else kv8_read_kernel<128><<<grid, 256, 0, st>>>(c, b, first, kk, vv, kts);
    return hipGetLastError();
}
hipError_t launch_kv8_copy(const Kv8& c, const int* src, const int* dst, int n, const int* seq_src, const int* seq_dst,
                           int nseq, hipStream_t st) {
    const long grid = ((long)n * 2 + (long)nseq * 4) * c.nkv;
    if (grid == 0) return hipSuccess;
    if (c.hd == 256) kv8_copy_kernel<256><<<dim3((unsigned)grid), 256, 0, st>>>(c, src, dst, n, seq_src, seq_dst);
    else kv8_copy_kernel<128><<<dim3((unsigned)grid), 256, 0, st>>>(c, src, dst, n, seq_src, seq_dst);
    return hipGetLastError();
}

}  // namespace it
