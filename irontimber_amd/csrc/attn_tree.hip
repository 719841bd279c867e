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

namespace it {

namespace {
constexpr int HD = 256;
constexpr int PART = idx::PART;
constexpr int SPL = 8;   // context records a lane loads per batch
}

// One workgroup per (256 / SL * 4 dims, head, node). Thread = (split lane sg of SL, dim lane of 256 / SL, 4
// dims each): split lane sg takes the context's records sg, sg + SL, ... and the path's keys likewise.
template <int SL>
__global__ __launch_bounds__(256) void attn_tree_merge_kernel(const float* __restrict__ q, int qts,
                                                              const uint16_t* __restrict__ kc,
                                                              const uint16_t* __restrict__ vc, int kvd, int pos0,
                                                              int nh, int nkv, int nt,
                                                              const uint64_t* __restrict__ anc, float scale,
                                                              const float* __restrict__ part, int smax,
                                                              float* __restrict__ out, int ots) {
    constexpr int DLN = 256 / SL, DW = 4 * DLN;   // dim lanes, dims per workgroup
    constexpr int NK = 64 / SL;                   // path keys per split lane
    __shared__ int node[64];                      // the path's nodes in order
    __shared__ float score[64];
    __shared__ float red_m[SL], red_d[SL];
    __shared__ f4 red_o[SL][DLN];
    const int dq = blockIdx.x, h = blockIdx.y, t = blockIdx.z, tid = threadIdx.x, w = tid >> 6, l = tid & 63;
    const int sg = tid / DLN, dl = tid % DLN, d0 = DW * dq + 4 * dl;
    float* dst = out + (size_t)t * ots + (size_t)h * HD + d0;
    const uint64_t mask = anc[t] & (~(uint64_t)0 >> (64 - nt));
    const int np = (int)__popcll(mask);
    if (np == 0) {   // a padding node
        if (sg == 0) *(f4*)dst = f4{0.f, 0.f, 0.f, 0.f};
        return;
    }
    const float* qrow = q + (size_t)t * qts + (size_t)h * 2 * HD;
    const f4 qv = ld_f4(qrow + 4 * l), gt = ld_f4(qrow + HD + d0);
    if (tid < 64 && (mask >> tid & 1)) node[__popcll(mask & (((uint64_t)1 << tid) - 1))] = tid;
    __syncthreads();
    // ---- the path: this lane's V pieces go out first, then the scores, a key a wave
    const size_t head = (size_t)(h / (nh / nkv)) * HD;
    h4 pv[NK];
#pragma unroll
    for (int j = 0; j < NK; ++j)
        pv[j] = *(const h4*)(vc + (size_t)(pos0 + node[min(sg + SL * j, np - 1)]) * kvd + head + d0);
    for (int j0 = w; j0 < np; j0 += 16) {
        h4 kv[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            kv[j] = *(const h4*)(kc + (size_t)(pos0 + node[min(j0 + 4 * j, np - 1)]) * kvd + head + 4 * l);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float s = wave_sum((qv[0] * (float)kv[j][0] + qv[1] * (float)kv[j][1]) +
                                     (qv[2] * (float)kv[j][2] + qv[3] * (float)kv[j][3]));
            if (l == 0 && j0 + 4 * j < np) score[j0 + 4 * j] = s * scale;
        }
    }
    __syncthreads();
    // ---- the path's own softmax (no reference below the type's range, so that keys of score -inf weigh 0)
    float M = score[0];
    for (int j = 1; j < np; ++j) M = fmaxf(M, score[j]);
    M = fmaxf(M, -FLT_MAX);
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
    // ---- the context's records
    const float* base = part + idx::rec(t * nh + h, 0, smax) * PART;
    for (int s0 = 0; s0 < smax; s0 += SL * SPL) {
        f2 hv[SPL];
        f4 ov[SPL];
#pragma unroll
        for (int j = 0; j < SPL; ++j) {   // slots past the last record reload it and count nothing
            const float* rec = base + (size_t)min(s0 + sg + SL * j, smax - 1) * PART;
            hv[j] = *(const f2*)rec;
            ov[j] = ld_f4(rec + 4 + d0);
        }
        float mloc = M;
#pragma unroll
        for (int j = 0; j < SPL; ++j) mloc = fmaxf(mloc, hv[j][0]);
        if (dl == 0) red_m[sg] = mloc;
        __syncthreads();
        float Mn = red_m[0];
#pragma unroll
        for (int j = 1; j < SL; ++j) Mn = fmaxf(Mn, red_m[j]);
        __syncthreads();
        const float r = __expf(M - Mn);
        den *= r;
        o *= r;
#pragma unroll
        for (int j = 0; j < SPL; ++j) {
            if (s0 + sg + SL * j < smax) {
                const float wgt = __expf(hv[j][0] - Mn);
                den += hv[j][1] * wgt;
                o += ov[j] * wgt;
            }
        }
        M = Mn;
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

// Keys per context split.
int attn_tree_chunk(int pos0, int nt, int nh, int nkv) {
    const long tiles = (pos0 + 63) / 64, groups = (long)nkv * ((nt * (nh / nkv) + 31) / 32);
    return 64 * (int)std::max(1L, (tiles * groups + 511) / 512);
}

hipError_t launch_attn_tree(const float* q, int qts, const uint16_t* kc, const uint16_t* vc, int kvd, int pos0,
                            int nh, int nkv, int nt, const uint64_t* anc, float scale, float* out, int ots,
                            float* part, int chunk, hipStream_t st) {
    int smax = 0;
    if (pos0 > 0) {
        smax = idx::split_count(pos0, chunk);
        const hipError_t e = launch_attn_all_partials(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, scale, part, chunk, st);
        if (e != hipSuccess) return e;
    }
    // few rows: a quarter of the dims a workgroup, 16 split lanes; many: the whole row, 4 split lanes
    if (nt * nh < 512)
        attn_tree_merge_kernel<16><<<dim3(4, nh, nt), 256, 0, st>>>(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, anc, scale,
                                                                  part, smax, out, ots);
    else
        attn_tree_merge_kernel<4><<<dim3(1, nh, nt), 256, 0, st>>>(q, qts, kc, vc, kvd, pos0, nh, nkv, nt, anc, scale,
                                                                 part, smax, out, ots);
    return hipGetLastError();
}

}  // namespace it
