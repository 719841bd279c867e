// The paged 8-bit cache's arguments and what its kernels share.
#pragma once
#include "common.h"
#include "kv8_index.h"

namespace it {

struct Kv8 {
    uint8_t *kp, *vp;    // codes [npages][nkv][64*hd], value (code - 128) * scale
    _Float16* sc;        // [npages][nkv][8]: K's four blocks, V's four
    _Float16 *tk, *tv;   // open rows [nseq][2][nkv][64*hd]
    int npages, nseq, nkv, hd;
};
// The sequences of a call: tokens start[i] .. start[i+1]-1 are sequence i's next rows after its len[i].
struct Kv8Batch {
    const int *start, *len, *table;
    int nseq, ntok, max_pages, max_nt;
};
struct Kv8Seq {
    int t0, n, len, pages;   // n 0: nothing to do; bad: a length or a page count that cannot be
    bool bad;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch& b, int i) {
    Kv8Seq s = {0, 0, 0, 0, false};
    if (i < b.nseq) {
        const int t0 = b.start[i], t1 = b.start[i + 1], len = b.len[i];
        if (t0 >= 0 && t1 <= b.ntok && t1 > t0) {
            s.t0 = t0;
            s.n = min(t1 - t0, b.max_nt);
            s.len = len;
            s.bad = len < 0 || (long)len + s.n > (long)b.max_pages * kv8::PAGE;
            s.pages = s.bad ? 1 : (len + s.n - 1) / kv8::PAGE + 1;
        }
    }
    return s;
}

// 4 codes as f16 (exact): 0x6400 | byte is 1024 + byte in f16.
__device__ __forceinline__ h4 codes4(uint32_t u) {
    const h2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return h4{a[0], a[1], b[0], b[1]};
}

}  // namespace it
