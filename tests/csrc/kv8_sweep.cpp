// Host sweep of the paged 8-bit cache's index and split arithmetic, on the header that the kernels use: every element of a
// page is named once, every page of every sequence belongs to one split of it, and the records of split sequences fit the
// room that is planned for them.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>
#include "../../irontimber_amd/csrc/kv8_index.h"

using namespace it;

static void die(const char* what, long a, long b) { std::printf("FAIL %s %ld %ld\n", what, a, b); std::exit(1); }

int main() {
    long checks = 0;
    for (int hd : {128, 256}) {
        std::vector<int> k(64 * hd, 0), v(64 * hd, 0);
        for (int r = 0; r < 64; ++r)
            for (int d = 0; d < hd; ++d) {
                const int a = kv8::k_elem(hd, r, d), b = kv8::v_elem(r, d);
                if (a < 0 || a >= 64 * hd || k[a]++) die("K element", r, d);
                if (b < 0 || b >= 64 * hd || v[b]++) die("V element", r, d);
                // 16-byte pieces: 8 dims of a K row, four rows of a V dim
                if (d % 8 && a != kv8::k_elem(hd, r, d - 1) + 1) die("K run", r, d);
                if (r % 4 && b != kv8::v_elem(r - 1, d) + 1) die("V run", r, d);
                checks += 4;
            }
    }
    unsigned seed = 12345;
    auto rnd = [&](int n) { seed = seed * 1664525u + 1013904223u; return (int)((seed >> 8) % (unsigned)n); };
    for (int it = 0; it < 20000; ++it) {
        const int nseq = 1 + rnd(it % 3 ? 8 : 130), nkv = 1 + rnd(8), wgs = it % 2 ? 256 : 512, most = 1 << (1 + rnd(it % 7 ? 12 : 25));
        std::vector<int> nrb(nseq), pages(nseq);
        float sum = 0.f, blocks = 0.f;
        for (int i0 = 0; i0 < nseq; i0 += 64) {
            float part = 0.f;
            for (int i = i0; i < nseq && i < i0 + 64; ++i) {
                nrb[i] = rnd(4) ? 1 + rnd(it % 5 ? 3 : 500) : 0;
                pages[i] = 1 + rnd(most);
                part += (float)nrb[i] * (float)pages[i];
                blocks += (float)nrb[i];
            }
            sum += part;
        }
        const int chunk = kv8::chunk_pages(sum * (float)nkv, blocks * (float)nkv, wgs);
        if (chunk < 1) die("chunk", chunk, it);
        long units = 0, groups = 0, recs = 0, split_groups = 0;
        for (int i = 0; i < nseq; ++i) {
            if (!nrb[i]) continue;
            const int ns = kv8::splits(pages[i], chunk);
            if ((long)(ns - 1) * chunk >= pages[i] || (long)ns * chunk < pages[i]) die("splits", pages[i], chunk);
            units += (long)nrb[i] * ns * nkv;
            groups += (long)nrb[i] * nkv;
            if (ns > 1) {
                recs += (long)nrb[i] * ns * nkv;
                split_groups += (long)nrb[i] * nkv;
                if (nrb[i] < 20 && ns < 50) {
                    std::set<int> seen;
                    for (int s = 0; s < ns; ++s)
                        for (int rb = 0; rb < nrb[i]; ++rb)
                            for (int kh = 0; kh < nkv; ++kh) seen.insert(kv8::record(s, nrb[i], rb, nkv, kh));
                    if ((long)seen.size() != (long)nrb[i] * ns * nkv || *seen.rbegin() != nrb[i] * ns * nkv - 1) die("record", i, it);
                }
            }
            ++checks;
        }
        if (units > groups + wgs + 1) die("units", units, groups);   // the launch's workgroups: groups + wgs and one for rounding
        if (recs > kv8::max_records(wgs)) die("records", recs, wgs);
        if (2 * split_groups > kv8::max_records(wgs)) die("groups", split_groups, wgs);
    }
    // Fewer pages per split where the count allows: the records still fit, whatever the count is off by
    for (int it = 0; it < 20000; ++it) {
        const int nseq = 1 + rnd(130), nkv = 1 + rnd(8), wgs = 512, most = 1 << (1 + rnd(it % 7 ? 12 : 25));
        std::vector<int> nrb(nseq), pages(nseq);
        float sum = 0.f, blocks = 0.f;
        for (int i = 0; i < nseq; ++i) {
            nrb[i] = rnd(4) ? 1 + rnd(3) : 0;
            pages[i] = it % 3 ? 1 + rnd(most) : most;
            sum += (float)nrb[i] * (float)pages[i];
            blocks += (float)nrb[i];
        }
        for (int k = 0; k < kv8::TRIES; ++k) {
            const int chunk = kv8::fewer_pages(sum * (float)nkv, blocks * (float)nkv, wgs, k);
            if (chunk < 1 || (k && chunk < kv8::fewer_pages(sum * (float)nkv, blocks * (float)nkv, wgs, k - 1))) die("fewer", chunk, k);
            if (chunk == 33554432) continue;
            float units = 0.f;
            long exact = 0, recs = 0;
            for (int i = 0; i < nseq; ++i) {
                const int ns = kv8::splits(pages[i], chunk);
                const float about = kv8::about_splits(pages[i], 1.0f / (float)chunk);
                if (about > (float)ns || about < (float)ns - 1) die("about", pages[i], chunk);
                units += (float)nrb[i] * about;
                exact += (long)nrb[i] * ns * nkv;
                if (ns > 1) recs += (long)nrb[i] * ns * nkv;
            }
            if (units * (float)nkv > (float)wgs) continue;
            if (exact > (long)(blocks * (float)nkv) + wgs + 1) die("fewer units", exact, it);
            if (recs > kv8::max_records(wgs)) die("fewer records", recs, it);
            ++checks;
        }
    }
    std::printf("ok %ld\n", checks);
    return 0;
}
