// A drafted token tree: the ancestor masks and positions that the tree calls take, and the cache rows of
// the accepted path. No counterpart in the reference, whose drafts are chains (src/mtp.rs:166-204).
//
// A tree is up to 64 nodes in topological order; anc[t] is the 64-bit mask of node t and its ancestors
// (0: a padding node), so a node's path is the set bits of its mask in ascending order.
#include "common.h"
#include "internal.h"

namespace it {

// One wave, lane = node. The masks grow by pointer doubling: after round r a node's mask holds its
// nearest 2^r - 1 ancestors and itself, and `up` the ancestor 2^r levels above (64 levels in 6 rounds). A
// parent outside -1 .. t-1 makes a padding node, and so does a padding ancestor. 1.5 us for 64 nodes, a launch.
__global__ __launch_bounds__(64) void tree_plan_kernel(const int* __restrict__ parent, int nt, int p0,
                                                       uint64_t* __restrict__ anc, int* __restrict__ pos) {
    const int t = threadIdx.x, p = t < nt ? parent[t] : -2;
    int dead = p < -1 || p >= t, up = dead ? -1 : p;
    uint64_t m = (uint64_t)1 << t;
#pragma unroll
    for (int r = 0; r < 6; ++r) {
        const int a = up < 0 ? t : up;   // (every lane takes part in the exchanges)
        m |= (uint64_t)(uint32_t)__shfl((int)(uint32_t)m, a) | (uint64_t)(uint32_t)__shfl((int)(m >> 32), a) << 32;
        dead |= __shfl(dead, a);
        const int next = __shfl(up, a);
        up = up < 0 ? -1 : next;
    }
    if (t < nt) {
        anc[t] = dead ? 0 : m;
        if (pos) pos[t] = p0 + (dead ? 0 : (int)__popcll(m) - 1);
    }
}

hipError_t launch_tree_plan(const int* parent, int nt, int p0, uint64_t* anc, int* pos, hipStream_t st) {
    tree_plan_kernel<<<1, 64, 0, st>>>(parent, nt, p0, anc, pos);
    return hipGetLastError();
}

// Rows pos0 + path[i] -> pos0 + i of both caches, path = the set bits of anc[leaf] up to leaf. A workgroup
// owns 64 bytes of every row: one 16-byte piece of one path row a thread, all loaded before any is stored,
// so the rows may overlap and one memory round trip serves the whole path. grid (row pieces / 4, 2 caches).
// A launch and that round trip: 2.2 us for 7 rows of 512 values, 2.6 for 64 rows of 1024.
__global__ __launch_bounds__(256) void kv_tree_commit_kernel(u4* kc, u4* vc, int pieces, int pos0,
                                                             const uint64_t* __restrict__ anc, int leaf) {
    __shared__ int path[64];
    const int tid = threadIdx.x, i = tid >> 2, c = 4 * blockIdx.x + (tid & 3);
    uint64_t m = anc[leaf] & (~(uint64_t)0 >> (63 - leaf));
    if (!(m >> leaf & 1)) m = 0;   // a padding node, as the recurrent layer's commit takes it
    if (tid < 64 && (m >> tid & 1)) path[__popcll(m & (((uint64_t)1 << tid) - 1))] = tid;
    __syncthreads();
    u4* cache = (blockIdx.y ? vc : kc) + (size_t)pos0 * pieces + c;
    const bool moves = i < (int)__popcll(m) && c < pieces && path[i] != i;
    u4 x = {};
    if (moves) x = cache[(size_t)path[i] * pieces];
    IT_WAIT_VMCNT(0);   // the piece is here before any wave passes the barrier and overwrites its row
    __syncthreads();
    if (moves) cache[(size_t)i * pieces] = x;
}

hipError_t launch_kv_tree_commit(void* kc, void* vc, size_t row_bytes, int pos0, const uint64_t* anc, int leaf,
                                 hipStream_t st) {
    const int pieces = (int)(row_bytes / 16);
    kv_tree_commit_kernel<<<dim3((pieces + 3) / 4, 2), 256, 0, st>>>((u4*)kc, (u4*)vc, pieces, pos0, anc, leaf);
    return hipGetLastError();
}

}  // namespace it
