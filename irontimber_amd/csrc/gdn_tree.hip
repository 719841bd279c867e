// The Gated-DeltaNet layer over a drafted token tree, and the commit of one node's states.
//
// The recurrence of cpu.rs:216-232 along every root-to-node path at once. With g_i a node's log decay, G_i
// its sum over the node's path (ancestors and itself) and S0 the committed state, the path's states unroll as in
// the chunk form of the delta rule, the causal mask replaced by "is an ancestor of":
//   A_ij = beta_i (k_i . k_j) e^(G_i - G_j)            j a strict ancestor of i, else 0
//   (I + A) U = beta (V - e^G (K S0))                    row i: the update u_i that node i adds to the state
//   out_i = (e^G_i q_i S0 + sum_j (q_i . k_j) e^(G_i - G_j) u_j) / sqrt(S)     j an ancestor of i or i itself
// Topological order makes A strictly lower triangular. G is summed in f64: far down a strongly decaying path
// the differences would lose f32's digits.
// The commit writes S_i = e^G_i S0 + sum_j e^(G_i - G_j) k_j u_j over i's path from the U, k and G that the layer
// call leaves in its trace. No counterpart in the reference, which steps one token at a time
// (src/vk/mod.rs:790-806) and copies checkpoints (1018-1025).
#include "common.h"
#include "internal.h"

namespace it {

namespace {
constexpr int S = 128;        // state size, and channels per head
constexpr int NW = 8;         // waves per workgroup of gdn_tree_kernel
constexpr int HST = S + 8;    // LDS row of a q or k row or a state column (halves)
constexpr double LOG2E_D = 1.4426950408889634074;

__device__ __forceinline__ f4 mfma4(float a, float b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Node t's mask with later nodes' bits off; 0 for a padding node (its own bit is clear).
__device__ __forceinline__ uint64_t node_mask(const uint64_t* anc, int t) {
    const uint64_t m = anc[t] & (~(uint64_t)0 >> (63 - t));
    return m >> t & 1 ? m : 0;
}

// The rows of a node's conv inputs 1 .. K-1 tokens back, among n nodes' and behind them the conv state's K - 1 (the newest
// last): its ancestors, and beyond the path's start the state. m: the mask of its strict ancestors, taken bit by bit from
// the top.
template <int K>
__device__ __forceinline__ void taps(uint64_t m, int n, int (&row)[K - 1]) {
    int beyond = n + K - 2;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        const int a = 63 - (int)__builtin_clzll(m | 1);
        row[j] = m ? a : beyond;
        if (!m) --beyond;
        m &= ~((uint64_t)1 << a);
    }
}
__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__shfl((int)(uint32_t)v, lane) | (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane) << 32;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }
}  // namespace

// Workgroup = (V head h, CW = 16 or 32 state columns), NW waves; NB blocks of 16 nodes. A head's q and k rows are
// convolved and normalised by each of its eight or four workgroups (into LDS), so no launch or barrier of the whole GPU
// stands between the conv and the products. The inputs of the convs go into LDS first, where each node takes its
// ancestors' rows, and the results take their place. The normalised rows, at length 1, and the state's columns, scaled, are
// kept as f16 pairs hi + lo (2^-22), and their products take three f16 matrix ops of 16 cycles for 32 dims (hi hi, hi lo,
// lo hi) where f32 ones would take eight of 32. The waves share the products out by blocks of rows; the inverses of I + A's
// diagonal blocks go one to a wave, and then each of the first NB waves (a block of columns: NB) solves for all of U in
// registers with f32 products (a few more than its share, but no exchange) and writes the output rows of its block.
// Measured: 3 nodes, 32 V heads 7.2 us; 26 nodes, 48 heads 9.4; 64 nodes, 32 heads 14. The floor is the state's bytes (2 MB:
// 0.4 us) and a launch; what is left is a chain of phases with one workgroup a CU. In cycles, 3 / 64 nodes: loads 2,900 /
// 5,000 (each wave's rows of x, weights, slice through the CU's load path), the ancestors' rows and the slice's maxima 1,500
// / 2,600, conv and norm 1,400 / 4,800 (the vector units of two waves a SIMD are busy), slice 1,000 / 1,000, products 2,000
// / 5,200, inverses, solve and output 3,000 / 5,400.
// Eight waves against four, us: 16 nodes, 32 heads 7.3 / 7.4; 26 nodes 8.9 / 9.4; 64 nodes 14.0 / 14.4.
template <int K, int NB, int CW>
__global__ __launch_bounds__(64 * NW) void gdn_tree_kernel(
    const float* __restrict__ x, int xts, const float* __restrict__ cw, const float* __restrict__ cst,
    const float* __restrict__ br, const float* __restrict__ ar, int bts, const float* __restrict__ dt,
    const float* __restrict__ A, const float* __restrict__ state, const uint64_t* __restrict__ anc,
    float* __restrict__ out, int ots, int nt, int nv, int nk, float eps, float* __restrict__ trace) {
    constexpr int N = 16 * NB, AST = N + 4, RST = CW + 4, CB = CW / 16;
    constexpr int NPR = 64 * NW / CW, CQ = CW / 4;   // nodes whose V a pass over the threads takes, quads of columns
    constexpr int QKB = 4 * N * HST * 2, RAWB = (N + K - 1) * 2 * S * 4;
    __shared__ __align__(16) char rows_[QKB > RAWB ? QKB : RAWB];
    auto raw = (float (*)[2 * S])rows_;                   // q and k inputs of the nodes, then those of the conv state
    auto qk = (_Float16 (*)[2][N][HST])rows_;             // after them: [q, k][hi, lo] rows
    __shared__ __align__(16) _Float16 sp[2][CW][HST];     // [hi, lo] the state slice, column by column, scaled
    __shared__ __align__(16) float mxs[NW][CW];           // column maxima of the waves' rows
    __shared__ float inv[CW];                             // what a column was divided by
    __shared__ __align__(16) float na[N][AST];            // -A
    __shared__ __align__(16) float pm[N][AST];            // (q_i . k_j) e^(G_i - G_j)
    __shared__ __align__(16) float tin[NB][16][20];       // inverses of the diagonal blocks of I + A
    __shared__ float vs[N][RST], os[N][RST];              // conv'd V, then U where it is summed node by node; e^G q S0
    __shared__ float rs[N + K - 1][RST];                  // V inputs, then right-hand sides
    __shared__ double gs[N];                              // G in log2 units
    __shared__ float bs[N];
    __shared__ float len[2][N];                           // lengths of the q and k rows: 1, or less below the norm's floor
    __shared__ int below;                                 // some row is
    __shared__ uint64_t ms[N];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, c = l & 15, g = l >> 4;
    const int cb = blockIdx.x % (S / CW), h = blockIdx.x / (S / CW), kh = h % nk, cd = (2 * nk + nv) * S;

    // ---- all loads but none that hangs on another: gates, the masks (a node a lane, in every wave), the wave's rows of x,
    // the conv state, conv weights, the state slice
    constexpr int PER = N / NW, VN = (N + NPR - 1) / NPR;
    static_assert(PER * NW == N && NW >= K - 1 && NB * CB <= NW, "every node once, none past the LDS rows");
    const int ch = (l < 32 ? kh : nk + kh) * S + 4 * (l & 31);         // lanes 0-31 four q channels each, 32-63 k
    const int chv = 2 * nk * S + h * S + cb * CW + tid % CW;            // V channel; CW lanes a node
    // gates, a node a lane (by every wave, used by the first: under a branch the loads would be waited for at its end)
    const size_t gate = (size_t)min(l, nt - 1) * bts + h;
    const float brv = br[gate], arv = ar[gate], dtv = dt[h], av = A[h];
    const uint64_t m = l < nt ? node_mask(anc, l) : 0;
    f4 own[PER], wt[K];
    float ownv[VN], wv[K];
#pragma unroll
    for (int i = 0; i < PER; ++i) own[i] = ld_f4(x + uniform_off((size_t)min(w + NW * i, nt - 1) * xts) + ch);
    const f4 old = ld_f4(cst + (size_t)min(w, K - 2) * cd + ch);
#pragma unroll
    for (int b = 0; b < VN; ++b) ownv[b] = x[(size_t)min(NPR * b + tid / CW, nt - 1) * xts + chv];
    const float oldv = cst[(size_t)min(tid / CW, K - 2) * cd + chv];
#pragma unroll
    for (int i = 0; i < K; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) wt[i][e] = cw[(size_t)(ch + e) * K + i];
        wv[i] = cw[(size_t)chv * K + i];
    }
    constexpr int SL = S * CW / 4 / (64 * NW);   // 16-byte pieces of the slice per thread
    f4 sl[SL];
#pragma unroll
    for (int i = 0; i < SL; ++i) {
        const int p = tid + 64 * NW * i;
        sl[i] = ld_f4(state + ((size_t)h * S + p / CQ) * S + cb * CW + 4 * (p % CQ));
    }
    const uint64_t above = m & ~((uint64_t)1 << l);   // strict ancestors
    int row[K - 1];   // lane = node
    taps<K>(above, N, row);
    const float neg1 = in_register(-1.0f), ieps = eps > 0.f ? 1.0f / (eps * (float)LOG2E_D) : INFINITY;
    const float most = fmaxf(ieps, 9e18f);   // 1 / |y| where the sum of squares is the least normal number
    if (w == 0) {
        // gates and path sums, a node a lane of the first wave (its loads went out first), while they are on their way
        double G = 0.0;
        float beta = 0.f;
        if (m) {
            beta = sigmoid_hw(brv);
            const float lg = softplus_hw(arv + dtv) * av;
            G = lg < -200.f ? -200.0 : (double)lg;   // e^-200 is 0 in f32 already; sums stay finite
        }
        int up = above ? 63 - (int)__builtin_clzll(above) : -1;
        while (__any(up >= 0)) {   // each round a node's sum covers twice as many nodes of its path
            const int a = up < 0 ? l : up;
            const double more = __builtin_bit_cast(double, shfl_u64(__builtin_bit_cast(uint64_t, G), a));
            const int next = __shfl(up, a);
            if (up >= 0) { G += more; up = next; }
        }
        if (l < N) { ms[l] = m; gs[l] = G * LOG2E_D; bs[l] = beta; len[0][l] = len[1][l] = 1.0f; }
        if (l == 0) below = 0;
    }

    // ---- the inputs of the convs into LDS, where a node finds its ancestors' (from memory they would be a second round
    // trip, and four rows a node through the CU's load path instead of one)
#pragma unroll
    for (int i = 0; i < PER; ++i) *(f4*)&raw[w + NW * i][4 * l] = own[i];
    if (w < K - 1) *(f4*)&raw[N + w][4 * l] = old;
#pragma unroll
    for (int b = 0; b < VN; ++b) {
        const int t = NPR * b + tid / CW;
        if (t < N) rs[t][tid % CW] = ownv[b];
    }
    if (tid / CW < K - 1) rs[N + tid / CW][tid % CW] = oldv;
    __syncthreads();
    f4 in[PER][K - 1];
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < K - 1; ++j) in[i][j] = ld_f4(&raw[__builtin_amdgcn_readlane(row[j], w + NW * i)][4 * l]);
    float inp[VN][K - 1];
#pragma unroll
    for (int b = 0; b < VN; ++b)
#pragma unroll
        for (int j = 0; j < K - 1; ++j) inp[b][j] = rs[__shfl(row[j], min(NPR * b + tid / CW, N - 1))][tid % CW];
    // ---- column maxima of the slice: over the thread's pieces, the lanes of its column quad, the waves
    {
        f4 mx = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < SL; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], fabsf(sl[i][e]));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (CQ == 4) mx[e] = fmaxf(mx[e], dppc<0x124>(mx[e]));   // row_ror:4
            mx[e] = fmaxf(mx[e], dppc<0x128>(mx[e]));   // row_ror:8
            mx[e] = max_xor32(max_xor16(mx[e]));
        }
        if (l < CQ) *(f4*)&mxs[w][4 * l] = mx;
    }
    __syncthreads();   // the q and k rows take their inputs' place
    // ---- conv + SiLU + L2 norm of the q and k heads (padding nodes take the conv state for ancestors; what their rows hold
    // is not used). The weights carry a factor log2 e, so that the conv's result is the exponent of the SiLU; the norm takes
    // the factor out again. A row below the norm's floor, y / eps, is brought to length 1 like the others, which the pairs
    // (their step is 2^-25) hold to 2^-22, and its length goes into the products' results.
#pragma unroll
    for (int i = 0; i < K; ++i) wt[i] *= (float)LOG2E_D;
    float f[PER], fm = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int t = w + NW * i;
        f4 y = in[i][K - 2] * wt[0];
#pragma unroll
        for (int j = K - 3; j >= 0; --j) y += in[i][j] * wt[K - 2 - j];
        y += own[i] * wt[K - 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-y[e]));
        float ss = (y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]);
        ss += dppc<0xB1>(ss);
        ss += dppc<0x4E>(ss);
        ss += dppc<0x141>(ss);
        ss += dppc<0x140>(ss);
        ss = sum_xor16(ss);
        f[i] = fminf(__builtin_amdgcn_rsqf(ss), most);   // 1 / |y|
        y *= f[i];
        h2 h0, h1, l0, l1;
        split2(f2{y[0], y[1]}, neg1, h0, l0);
        split2(f2{y[2], y[3]}, neg1, h1, l1);
        *(h4*)&qk[l >> 5][0][t][4 * (l & 31)] = h4{h0[0], h0[1], h1[0], h1[1]};
        *(h4*)&qk[l >> 5][1][t][4 * (l & 31)] = h4{l0[0], l0[1], l1[0], l1[1]};
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) fm = fmaxf(fm, f[i]);
    if (__any(fm > ieps)) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if ((l & 31) == 0 && f[i] > ieps) len[l >> 5][w + NW * i] = ieps / f[i];
        below = 1;
    }
    // ---- conv + SiLU of the workgroup's V columns
#pragma unroll
    for (int b = 0; b < VN; ++b) {
        const int t = NPR * b + tid / CW;
        float y = ownv[b] * wv[K - 1];
#pragma unroll
        for (int j = 0; j < K - 1; ++j) y += inp[b][j] * wv[K - 2 - j];
        if (t < N) vs[t][tid % CW] = silu_hw(y);
    }
    // ---- the slice as f16 pairs: each column times the power of two that takes its largest value to 2^13 .. 2^14, so that
    // the pairs hold every value to 2^-22 of itself or 2^-39 of the column's largest
    {
        f4 mx = ld_f4(&mxs[0][4 * (tid % CQ)]);
#pragma unroll
        for (int i = 1; i < NW; ++i) {
            const f4 o = ld_f4(&mxs[i][4 * (tid % CQ)]);
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], o[e]);
        }
        int ex[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) ex[e] = mx[e] > 0.f ? 14 - __builtin_amdgcn_frexp_expf(mx[e]) : 0;
#pragma unroll
        for (int i = 0; i < SL; ++i) {
            const int r = (tid + 64 * NW * i) / CQ;
            f4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_amdgcn_ldexpf(sl[i][e], ex[e]);
            h2 hi[2], lo[2];
            split2(f2{v[0], v[1]}, neg1, hi[0], lo[0]);
            split2(f2{v[2], v[3]}, neg1, hi[1], lo[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sp[0][4 * (tid % CQ) + e][r] = hi[e >> 1][e & 1];
                sp[1][4 * (tid % CQ) + e][r] = lo[e >> 1][e & 1];
            }
        }
        if (tid < CQ) {
#pragma unroll
            for (int e = 0; e < 4; ++e) inv[4 * tid + e] = __builtin_amdgcn_ldexpf(1.0f, -ex[e]);
        }
    }
    __syncthreads();
    // ---- products: {K, Q} S0 of each block, {K, Q} K^T of each pair of blocks bi >= bj
    // A wave takes one block of k or q rows through its products, the rows' operands read once: with the state's columns, and
    // with the k rows of every block up to its own. Where there are waves enough, two share them: one the state's.
    constexpr bool SHARE = NW >= 4 * NB;
    const int combo = SHARE ? w >> 1 : w;
    if (combo < 2 * NB) {
        const int which = (combo & 1) ^ 1, bi = combo >> 1;   // 1 k rows, 0 q rows
        h8 ah[4], al[4];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            ah[ks] = ld_h8(&qk[which][0][16 * bi + c][32 * ks + 8 * g]);
            al[ks] = ld_h8(&qk[which][1][16 * bi + c][32 * ks + 8 * g]);
        }
        uint64_t mt[4];
        double gt[4];
        float bt[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            mt[i] = ms[16 * bi + 4 * g + i];
            gt[i] = gs[16 * bi + 4 * g + i];
            bt[i] = which ? -bs[16 * bi + 4 * g + i] : 1.0f;
        }
        auto product = [&](const _Float16* bhp, const _Float16* blp) __attribute__((always_inline)) {
            h8 bh[4], bl[4];
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                bh[ks] = ld_h8(bhp + 32 * ks);
                bl[ks] = ld_h8(blp + 32 * ks);
            }
            __builtin_amdgcn_sched_barrier(0);   // (all operands out before the first product waits for one)
            f4 acc = {0.f, 0.f, 0.f, 0.f}, small = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                acc = mfma16x16x32(ah[ks], bh[ks], acc);
                small = mfma16x16x32(ah[ks], bl[ks], small);
                small = mfma16x16x32(al[ks], bh[ks], small);
            }
            return acc + small;
        };
        if (!SHARE || !(w & 1)) {
#pragma unroll
            for (int cc = c; cc < CW; cc += 16) {
                const f4 acc = product(&sp[0][cc][8 * g], &sp[1][cc][8 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * bi + 4 * g + i;
                    const float d = acc[i] * inv[cc] * __builtin_amdgcn_exp2f((float)gt[i]);
                    const float v = which ? bt[i] * (d - vs[t][cc]) : d;
                    (which ? rs : os)[t][cc] = mt[i] ? v : 0.f;
                }
            }
        }
        if (!SHARE || (w & 1)) {
            for (int bj = 0; bj <= bi; ++bj) {
                const int j = 16 * bj + c;
                const f4 acc = product(&qk[1][0][j][8 * g], &qk[1][1][j][8 * g]);
                const double gj = gs[j];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * bi + 4 * g + i;
                    const bool seen = (uint32_t)(mt[i] >> (16 * bj)) >> c & 1;
                    const float v = acc[i] * __builtin_amdgcn_exp2f((float)(gt[i] - gj)) * bt[i];
                    (which ? na : pm)[t][j] = seen && (!which || j != t) ? v : 0.f;
                }
            }
        }
    }
    __syncthreads();
    if (below) {   // the lengths of short rows into the products (the right-hand sides are beta (V - e^G k S0))
        for (int i = tid; i < N * N; i += 64 * NW) {
            const int t = i / N, j = i % N;
            if (j > t) continue;
            na[t][j] *= len[1][t] * len[1][j];
            pm[t][j] *= len[0][t] * len[1][j];
        }
        for (int i = tid; i < N * CW; i += 64 * NW) {
            const int t = i / CW, cc = i % CW;
            const float bv = bs[t] * vs[t][cc], k = len[1][t];
            os[t][cc] *= len[0][t];
            if (ms[t] && k != 1.0f) rs[t][cc] = (rs[t][cc] - bv) * k + bv;
        }
        __syncthreads();
    }
    const float scale = 1.0f / sqrtf((float)S);
    float* tu = trace + (size_t)h * S + cb * CW;   // U rows, then k rows, then G
    const size_t ustride = (size_t)nv * S;
    // ---- (I + A_bb)^-1, lane column c: a column of the identity, each row's value taken to the rows below as soon as
    // it is known (the four lane groups alike)
    if (w < NB) {
        f4 a[16][4];
        float z[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            z[i] = i == c ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < (i + 3) / 4; ++j) a[i][j] = ld_f4(&na[16 * w + i][16 * w + 4 * j]);
        }
#pragma unroll
        for (int j = 0; j < 15; ++j)
#pragma unroll
            for (int i = j + 1; i < 16; ++i) z[i] += a[i][j / 4][j % 4] * z[j];
        if (g == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i) tin[w][i][c] = z[i];
        }
    }
    __syncthreads();
    if (w < NB * CB) {
        const int cc = 16 * (w / NB) + c;   // column
        // ---- U block by block: u[b] holds rows 4 g + e of column cc, both a product's result and, in the order of
        // the A operand's 16-byte reads, the next one's B operand
        f4 u[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = rs[16 * b + 4 * g + i][cc];
#pragma unroll
            for (int j = 0; j < b; ++j) {
                const f4 a = ld_f4(&na[16 * b + c][16 * j + 4 * g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) r = mfma4(a[e], u[j][e], r);
            }
            const f4 a = ld_f4(&tin[b][c][4 * g]);
            u[b] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) u[b] = mfma4(a[e], r[e], u[b]);
        }
        bool fine = true;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) fine &= finite(u[b][e]);
        // ---- output and trace rows of block w % NB
        if (__any(!fine)) {
            // What is not finite in one branch has gone to others as 0 * inf (wherever it came from, the conv, a gate, the
            // state or the solve itself, U shows it): the same sums node by node over the ancestors alone. All waves of
            // these columns found the same U, and leave them to the first.
            if (w % NB == 0 && g == 0) {
                for (int t = 0; t < nt; ++t) {
                    float v = rs[t][cc], o = os[t][cc];
                    for (int j = 0; j < t; ++j)
                        if (ms[t] >> j & 1) v += na[t][j] * vs[j][cc];
                    vs[t][cc] = v;
                    for (int j = 0; j <= t; ++j)
                        if (ms[t] >> j & 1) o += pm[t][j] * vs[j][cc];
                    out[(size_t)t * ots + (size_t)h * S + cb * CW + cc] = o * scale;
                    tu[t * ustride + cc] = v;
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b != w % NB) continue;   // (static register indexes)
                f4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = os[16 * b + 4 * g + i][cc];
#pragma unroll
                for (int j = 0; j <= b; ++j) {
                    const f4 a = ld_f4(&pm[16 * b + c][16 * j + 4 * g]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o = mfma4(a[e], u[j][e], o);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * b + 4 * g + i;
                    if (t < nt) {
                        out[(size_t)t * ots + (size_t)h * S + cb * CW + cc] = o[i] * scale;
                        tu[t * ustride + cc] = u[b][i];
                    }
                }
            }
        }
    }
    // ---- the rest of the trace: k rows by the QK head's first V head, CW dims a workgroup; G once a head
    if (h < nk) {
        float* tk = trace + (size_t)nt * nv * S + (size_t)h * S + cb * CW;
        for (int i = tid; i < nt * CW; i += 64 * NW) {
            const int t = i / CW, d = cb * CW + i % CW;
            tk[(size_t)t * nk * S + i % CW] = ((float)qk[1][0][t][d] + (float)qk[1][1][t][d]) * len[1][t];
        }
    }
    if (cb == 0 && tid < nt) ((double*)(trace + (size_t)nt * (nv + nk) * S))[(size_t)tid * nv + h] = gs[tid];   // in log2 units
}

size_t gdn_tree_trace_bytes(int nt, int nv, int nk) {
    return (size_t)nt * (nv + nk) * S * sizeof(float) + (size_t)nt * nv * sizeof(double);
}

hipError_t launch_gdn_tree(const float* x, int xts, const float* cw, int K, const float* cst, const float* br,
                           const float* ar, int bts, const float* dt, const float* a, const float* state,
                           const uint64_t* anc, float* out, int ots, int nt, int nv, int nk, float eps, float* trace,
                           hipStream_t st) {
    // 32 columns a workgroup where 16 would take a round of the CUs more. 48 heads, 16 / 32 columns, us: 3 nodes 8.2 / 7.6, 26
    // nodes 12.4 / 9.4, 64 nodes 24.0 / 14.6; with 32 heads 16 columns are one round already, of twice the workgroups.
    const int cus = 256;   // MI355X compute units
    const bool wide = (4 * nv + cus - 1) / cus < (8 * nv + cus - 1) / cus;
#define IT_GDN_TREE(K_, NB_, CW_)                                                                                         \
    gdn_tree_kernel<K_, NB_, CW_><<<S / CW_ * nv, 64 * NW, 0, st>>>(x, xts, cw, cst, br, ar, bts, dt, a, state, anc, out, ots, \
                                                                    nt, nv, nk, eps, trace)
#define IT_GDN_TREE_W(K_, NB_)          \
    if (wide) IT_GDN_TREE(K_, NB_, 32); \
    else IT_GDN_TREE(K_, NB_, 16);      \
    break;
#define IT_GDN_TREE_K(K_)                \
    switch ((nt + 15) / 16) {            \
        case 1: IT_GDN_TREE_W(K_, 1)     \
        case 2: IT_GDN_TREE_W(K_, 2)     \
        case 3: IT_GDN_TREE_W(K_, 3)     \
        default: IT_GDN_TREE_W(K_, 4)    \
    }
    switch (K) {
        case 2: IT_GDN_TREE_K(2) break;
        case 3: IT_GDN_TREE_K(3) break;
        default: IT_GDN_TREE_K(4) break;
    }
#undef IT_GDN_TREE_K
#undef IT_GDN_TREE_W
#undef IT_GDN_TREE
    return hipGetLastError();
}

// Workgroups 0 .. 8 nv - 1: 16 state rows of a head, thread = (row, 8 columns), the path's rank-one updates on top
// of the decayed state. The others: 256 channels of the conv state, whose rows are the last K - 1 inputs of
// {old state, the path's rows of x}; a thread reads its channel's old rows before it writes any. A launch and two dependent
// round trips (mask, then k and U): 3.8 us for one node of 32 heads, 4.1 for a path of two, 5.4 for 48 heads and a path of 9.
__global__ __launch_bounds__(256) void gdn_tree_commit_kernel(const float* __restrict__ x, int xts, int K, float* cst,
                                                              float* __restrict__ state,
                                                              const uint64_t* __restrict__ anc, int leaf, int nt,
                                                              int nv, int nk, const float* __restrict__ trace) {
    __shared__ float coef[64];
    __shared__ int node[64];
    const int tid = threadIdx.x, cd = (2 * nk + nv) * S;
    const uint64_t m = node_mask(anc, leaf);
    const int np = (int)__popcll(m);
    if (np == 0) return;   // a padding node: nothing is kept
    const bool conv = blockIdx.x >= (unsigned)(8 * nv);
    const int h = conv ? 0 : blockIdx.x >> 3;
    const double* G = (const double*)(trace + (size_t)nt * (nv + nk) * S);
    const double Gl = G[(size_t)leaf * nv + h];
    if (tid < 64 && (m >> tid & 1)) {
        const int i = (int)__popcll(m & (((uint64_t)1 << tid) - 1));
        node[i] = tid;
        coef[i] = __builtin_amdgcn_exp2f((float)(Gl - G[(size_t)tid * nv + h]));
    }
    __syncthreads();
    if (conv) {
        const int ch = (blockIdx.x - 8 * nv) * 256 + tid;
        if (ch >= cd) return;
        float r[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {   // row i of the new state: input i + np of {old rows, path}
            const int s = i + np;
            if (i < K - 1) r[i] = s < K - 1 ? cst[(size_t)s * cd + ch] : x[(size_t)node[s - (K - 1)] * xts + ch];
        }
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < K - 1) cst[(size_t)i * cd + ch] = r[i];
        return;
    }
    const int row = (blockIdx.x & 7) * 16 + (tid >> 4), col = (tid & 15) * 8;
    float* s = state + ((size_t)h * S + row) * S + col;
    const float* tu = trace + (size_t)h * S + col;
    const float* tk = trace + (size_t)nt * nv * S + (size_t)(h % nk) * S + row;
    const float eg = __builtin_amdgcn_exp2f((float)Gl);
    f4 s0 = ld_f4(s) * eg, s1 = ld_f4(s + 4) * eg;
#pragma unroll 4
    for (int i = 0; i < np; ++i) {
        const float* u = tu + (size_t)node[i] * nv * S;
        const float k = tk[(size_t)node[i] * nk * S] * coef[i];
        s0 += k * ld_f4(u);
        s1 += k * ld_f4(u + 4);
    }
    *(f4*)s = s0;
    *(f4*)(s + 4) = s1;
}

hipError_t launch_gdn_tree_commit(const float* x, int xts, int K, float* cst, float* state, const uint64_t* anc,
                                  int leaf, int nt, int nv, int nk, const float* trace, hipStream_t st) {
    const int cd = (2 * nk + nv) * S;
    gdn_tree_commit_kernel<<<8 * nv + (cd + 255) / 256, 256, 0, st>>>(x, xts, K, cst, state, anc, leaf, nt, nv, nk, trace);
    return hipGetLastError();
}

}  // namespace it
