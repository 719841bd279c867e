// The paged 8-bit K/V cache: rows appended and quantised, rows read back, pages and open rows copied.
//
// A page holds 64 rows of every KV head; each block of 16 rows and head has one scale s for K and one for V, and a value is
// (code - 128) * s. s has four significant bits (or is a multiple of 2^-24), so code * s has eleven: every stored value is an
// f16 number, and what reads the cache computes with exact operands. s is the block's largest size / 127 rounded up,
// which costs 1/16 of a step on average (1/8 at most) against 127 steps exactly.
// A scale belongs to whole blocks, so a page is quantised once, when its last row arrives; until then its rows stand in
// the sequence's open buffer, in f16 and in the page's own element order. That buffer keeps the last two pages' rows, so
// that rows taken back (drafts that a check rejects) need nothing but a smaller length.
#include "internal.h"
#include "kv8.h"

namespace it {
namespace {

// An infinity is stored as the largest f16, a NaN as 0: a value that no query may see must not reach its products.
__device__ __forceinline__ _Float16 finite(_Float16 x) {
    const _Float16 top = (_Float16)65504.f;
    return x != x ? (_Float16)0.f : x > top ? top : x < -top ? -top : x;
}
__device__ __forceinline__ h8 finite8(h8 x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = finite(x[i]);
    return x;
}
__device__ __forceinline__ float largest(h8 x, float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf((float)x[i]));
    return m;
}
// A block's scale from its largest size. amax has 11 bits and 127 * s 11, so they differ by 2^-15 or not at all, and the
// rounded quotient falls on the same side of s as the exact one.
__device__ __forceinline__ float block_scale(float amax) {
    const float t = amax / 127.0f;
    if (t < 0x1p-21f) return fmaxf(ceilf(t * 0x1p24f), 1.0f) * 0x1p-24f;
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, t) + 0xFFFFFu) & ~0xFFFFFu);
}
// x / s to the nearest step, ties to even; likewise no quotient is nearer to a tie than f32 tells. s is above 512 only
// as 576, of which 113 steps still are f16.
__device__ __forceinline__ uint32_t code(_Float16 x, float s) {
    const float top = s > 512.f ? 113.f : 127.f;
    return (uint32_t)(int)(fminf(fmaxf(rintf((float)x / s), -top), top) + 128.f);
}

// Workgroup = (sequence, touched page, KV head, K or V). Quantises the page if the call fills it; the workgroups of the
// first two pages also write the new rows of the last two pages to the open buffer, each those of its own half of it,
// after its page's old open rows have been read (a half is read and written by one workgroup only).
// Bound by bytes: two read and one written a value (two where a page stays open).
template <int HD>
__global__ __launch_bounds__(256) void kv8_append_kernel(Kv8 c, Kv8Batch b, const _Float16* __restrict__ k,
                                                         const _Float16* __restrict__ v, int kts) {
    constexpr int CH = HD / 8, PITCH = HD + 8;   // (rows four apart in LDS: 16 banks apart)
    __shared__ __align__(16) _Float16 tile[kv8::PAGE * PITCH];
    __shared__ float vs[4];
    const int i = blockIdx.z, kh = blockIdx.y >> 1, which = blockIdx.y & 1, j = blockIdx.x;
    const Kv8Seq s = kv8_seq(b, i);
    const int p = s.len / kv8::PAGE + j, total = s.len + s.n;
    if (s.n == 0 || s.bad || (long)p * kv8::PAGE >= total) return;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const int row0 = p * kv8::PAGE;
    const _Float16* src = (which ? v : k) + (size_t)s.t0 * kts + (size_t)kh * HD;   // token t at t * kts
    _Float16* open = (which ? c.tv : c.tk) + ((size_t)i * 2 * c.nkv + kh) * (kv8::PAGE * HD);
    const size_t half = (size_t)c.nkv * kv8::PAGE * HD;
    if (row0 + kv8::PAGE <= total) {
        const int id = b.table[(size_t)i * b.max_pages + p];
        const bool known = (unsigned)id < (unsigned)c.npages;
        const size_t unit = known ? (size_t)id * c.nkv + kh : 0;
        const _Float16* old = open + (p & 1) * half;
        if (!which) {
            // wave = block: each lane holds a row's runs of 8 dims as the page orders them
            const int row = 16 * w + (l & 15), t = row0 + row - s.len;
            h8 x[CH / 4];
            float m = 0.f;
#pragma unroll
            for (int ks = 0; ks < CH / 4; ++ks) {
                const _Float16* at = t >= 0 ? src + (size_t)t * kts + 32 * ks + 8 * (l >> 4)
                                            : old + ((w * (HD / 64) + (ks >> 1)) * 64 + l) * 16 + 8 * (ks & 1);
                x[ks] = ld_h8(at);
            }
#pragma unroll
            for (int ks = 0; ks < CH / 4; ++ks) {
                x[ks] = finite8(x[ks]);
                m = largest(x[ks], m);
            }
            const float sc = block_scale(wave_max(m));
            if (known) {
#pragma unroll
                for (int jj = 0; jj < HD / 64; ++jj) {
                    u4 y;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const h8 z = x[2 * jj + (e >> 1)];
                        const int o = 4 * (e & 1);
                        y[e] = code(z[o], sc) | code(z[o + 1], sc) << 8 | code(z[o + 2], sc) << 16 | code(z[o + 3], sc) << 24;
                    }
                    *(u4*)(c.kp + unit * (kv8::PAGE * HD) + ((w * (HD / 64) + jj) * 64 + l) * 16) = y;
                }
                if (l == 0) c.sc[unit * 8 + w] = (_Float16)sc;
            }
        } else {
            // wave = block for the rows in; through LDS to four rows of each block and one dim a lane
            float m = 0.f;
#pragma unroll
            for (int n = 0; n < CH / 4; ++n) {
                const int row = 16 * w + (n * 64 + l) / CH, ch = (n * 64 + l) % CH, t = row0 + row - s.len;
                h8 x;
                if (t >= 0) {
                    x = finite8(ld_h8(src + (size_t)t * kts + 8 * ch));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = old[kv8::v_elem(row, 8 * ch + e)];
                }
                m = largest(x, m);
                *(h8*)(tile + row * PITCH + 8 * ch) = x;
            }
            const float sc = block_scale(wave_max(m));
            if (l == 0) {
                vs[w] = sc;
                if (known) c.sc[unit * 8 + 4 + w] = (_Float16)sc;
            }
            __syncthreads();
            if (known) {
#pragma unroll
                for (int db = w; db < HD / 16; db += 4) {
                    u4 y;
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const _Float16* z = tile + (16 * a + 4 * (l >> 4)) * PITCH + 16 * db + (l & 15);
                        y[a] = code(z[0], vs[a]) | code(z[PITCH], vs[a]) << 8 | code(z[2 * PITCH], vs[a]) << 16 |
                               code(z[3 * PITCH], vs[a]) << 24;
                    }
                    *(u4*)(c.vp + unit * (kv8::PAGE * HD) + (db * 64 + l) * 16) = y;
                }
            }
        }
        __syncthreads();   // old open rows read before the half is written below
    }
    if (j >= 2) return;
    const int last = (total - 1) / kv8::PAGE, pt = last - ((last ^ p) & 1);   // the page of this half among the last two
    const int lo = max(s.len, pt * kv8::PAGE), hi = min(total, (pt + 1) * kv8::PAGE);
    _Float16* to = open + (pt & 1) * half;
    for (int n = tid; n < (hi - lo) * CH; n += 256) {
        const int row = lo + n / CH, ch = n % CH;
        const h8 x = finite8(ld_h8(src + (size_t)(row - s.len) * kts + 8 * ch));
        const int r = row - pt * kv8::PAGE;
        if (!which) {
            *(h8*)(to + kv8::k_elem(HD, r, 8 * ch)) = x;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) to[kv8::v_elem(r, 8 * ch + e)] = x[e];
        }
    }
}

// Workgroup = (sequence, page, KV head, K or V): rows first[i] .. of a sequence that holds len[i] rows, as f16.
template <int HD>
__global__ __launch_bounds__(256) void kv8_read_kernel(Kv8 c, Kv8Batch b, const int* __restrict__ first,
                                                       _Float16* __restrict__ k, _Float16* __restrict__ v, int kts) {
    constexpr int CH = HD / 8, PITCH = HD + 8;
    __shared__ __align__(16) _Float16 tile[kv8::PAGE * PITCH];
    const int i = blockIdx.z, kh = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int t0 = b.start[i], t1 = b.start[i + 1], r0 = first[i], total = b.len[i];
    if (t0 < 0 || t1 > b.ntok || t1 <= t0 || r0 < 0 || total > (long)b.max_pages * kv8::PAGE) return;
    const int r1 = (int)min((long)total, (long)r0 + min(t1 - t0, b.max_nt));   // one past the last row
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
    for (int n = w; n < HD / 16; n += 4) {   // KiB n of the page
        h8 x[2];
        if (is_open) {
            x[0] = ld_h8(open + (n * 64 + l) * 16);
            x[1] = ld_h8(open + (n * 64 + l) * 16 + 8);
        } else {
            const u4 y = *(const u4*)(page + (n * 64 + l) * 16);
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const h4 z = codes4(y[a]);
                const _Float16 f = known ? sc[which ? a : n / (HD / 64)] : bad;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[a >> 1][4 * (a & 1) + e] = z[e] * f;
            }
        }
        if (!which) {
            const int row = 16 * (n / (HD / 64)) + (l & 15), dim = 64 * (n % (HD / 64)) + 8 * (l >> 4);
            if (row >= lo && row < hi) {
                *(h8*)(dst + (long)row * kts + dim) = x[0];
                *(h8*)(dst + (long)row * kts + dim + 32) = x[1];
            }
        } else {
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    tile[(16 * a + 4 * (l >> 4) + e) * PITCH + 16 * n + (l & 15)] = x[a >> 1][4 * (a & 1) + e];
        }
    }
    if (!which) return;   // (whole workgroup)
    __syncthreads();
    for (int n = tid; n < (hi - lo) * CH; n += 256) {
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
    const dim3 grid(touched(b.max_nt), 2 * c.nkv, b.nseq);
    const auto *kk = (const _Float16*)k, *vv = (const _Float16*)v;
    if (c.hd == 256) kv8_append_kernel<256><<<grid, 256, 0, st>>>(c, b, kk, vv, kts);
    else kv8_append_kernel<128><<<grid, 256, 0, st>>>(c, b, kk, vv, kts);
    return hipGetLastError();
}
hipError_t launch_kv8_read(const Kv8& c, const Kv8Batch& b, const int* first, uint16_t* k, uint16_t* v, int kts,
                           hipStream_t st) {
    const dim3 grid(touched(b.max_nt), 2 * c.nkv, b.nseq);
    auto *kk = (_Float16*)k, *vv = (_Float16*)v;
    if (c.hd == 256) kv8_read_kernel<256><<<grid, 256, 0, st>>>(c, b, first, kk, vv, kts);
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
