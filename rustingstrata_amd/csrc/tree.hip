// Trees of drafted tokens: their positions and ancestor masks (strata_tree_step) and the path that the model's choices confirm
// (strata_tree_accept). All integers. A sequence's rows are its tree's nodes, a parent before its children; a sequence of more
// rows than the masks have bits is a plain line of tokens.
#include "branch.h"

namespace strata {

struct TreeSeq {
    int q0, n, len, base;  // rows, own cached positions with them and before them
};
__device__ __forceinline__ TreeSeq tree_seq(const int* q_start, const int* len, int s, int t) {
    TreeSeq r;
    r.q0 = min(max(sload(q_start + s), 0), t);
    r.n = min(max(sload(q_start + s + 1), r.q0), t) - r.q0;
    r.len = sload(len + s);
    r.base = max(r.len - r.n, 0);
    return r;
}

// Node i's mask is its parent's and its own bit, its depth the number of its ancestors. By doubling: after round r the mask holds
// the 2^r nearest of the line upwards and `up` is the node 2^r above, so a tree of depth d takes log2(d) + 1 rounds through LDS.
// A block per sequence, a thread per node. Bound by latency: 512 sequences of up to 64 nodes 2.8 us
// replayed, one of 26 2.4 (a launch's own floor is 1.6).
template <int W>
__global__ __launch_bounds__(W <= 2 ? 64 : 32 * W) void tree_step_kernel(TreeStep a) {
    constexpr int T = W <= 2 ? 64 : 32 * W;
    __shared__ uint32_t bits[W][T];
    __shared__ int ups[T];
    const int s = blockIdx.x, i = threadIdx.x;
    const int P = a.prefix_len ? max(sload(a.prefix_len), 0) : 0;
    if (s == a.nseq) {  // rows behind the last sequence
        for (int r = min(max(sload(a.q_start + a.nseq), 0), a.t) + i; r < a.t; r += T) {
            a.pos[r] = -1;
            for (int w = 0; w < a.words; w++) a.mask[(uint64_t)r * a.words + w] = 0;
        }
        return;
    }
    const TreeSeq q = tree_seq(a.q_start, a.len, s, a.t);
    const long long first = (long long)P + q.base;
    if (q.n > 32 * a.words) {
        for (int r = i; r < q.n; r += T) {
            a.pos[q.q0 + r] = (int)min(first + r, (long long)INT32_MAX);
            for (int w = 0; w < a.words; w++) a.mask[(uint64_t)(q.q0 + r) * a.words + w] = 0;
        }
        return;
    }
    int up = i < q.n ? a.parent[q.q0 + i] : -1;
    const bool bad = up < -1 || up >= i;
    if (bad) up = -1;
    uint32_t m[W];
#pragma unroll
    for (int w = 0; w < W; w++) m[w] = w == i / 32 ? 1u << (i % 32) : 0u;
    while (__syncthreads_or(up >= 0)) {
        ups[i] = up;
#pragma unroll
        for (int w = 0; w < W; w++) bits[w][i] = m[w];
        __syncthreads();
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < W; w++) m[w] |= bits[w][up];
            up = ups[up];
        }
    }
    if (i < q.n) {
        int depth = -1;
#pragma unroll
        for (int w = 0; w < W; w++) {
            depth += __popc(m[w]);
            if (w < a.words) a.mask[(uint64_t)(q.q0 + i) * a.words + w] = m[w];
        }
        a.pos[q.q0 + i] = (int)min(first + depth, (long long)INT32_MAX);
        if (bad && a.err) atomicAdd(a.err, 1);
    }
}

hipError_t launch_tree_step(const TreeStep& a, hipStream_t s) {
    const dim3 grid((unsigned)a.nseq + 1);
    if (a.words <= 1) tree_step_kernel<1><<<grid, dim3(64), 0, s>>>(a);
    else if (a.words <= 2) tree_step_kernel<2><<<grid, dim3(64), 0, s>>>(a);
    else if (a.words <= 4) tree_step_kernel<4><<<grid, dim3(128), 0, s>>>(a);
    else tree_step_kernel<8><<<grid, dim3(256), 0, s>>>(a);
    return hipGetLastError();
}

// The walk from the root: the next node is the first one whose parent is the current node and whose token is the choice after it. A
// wave per sequence holds the nodes in its registers (R a lane), so a step is R comparisons, a ballot and two lane reads; the
// current node's index only grows, so the walk ends. Bound by latency: the nodes' loads, then the path's stores.
template <int R>
__global__ __launch_bounds__(64) void tree_accept_kernel(TreeAccept a) {
    const int s = blockIdx.x, lane = threadIdx.x;
    const TreeSeq q = tree_seq(a.q_start, a.len, s, a.t);
    int* chosen = a.chosen + (uint64_t)s * a.max_path;
    int* runs = a.runs + (uint64_t)s * a.max_path * 3;
    int n = 0, last = -1, keep = q.len, moves = 0;  // moves: path entries whose run has been written
    const bool tree = q.n <= 32 * a.words;
    if (q.n > 0 && sload(a.slots + q.q0) >= 0) {
        if (!tree) {  // a line of tokens: the choice after its last one
            n = 1;
            last = q.q0 + q.n - 1;
            if (lane == 0) chosen[0] = sload(a.ids + last);
        } else {
            int par[R], tok[R], id[R], slot[R];
#pragma unroll
            for (int r = 0; r < R; r++) {
                const int i = 64 * r + lane;
                const bool in = i < q.n;
                par[r] = in ? a.parent[q.q0 + i] : -2;
                tok[r] = in ? a.tokens[q.q0 + i] : -1;
                id[r] = in ? a.ids[q.q0 + i] : -1;
                slot[r] = in ? a.slots[q.q0 + i] : -1;
            }
            auto of = [&](const int (&v)[R], int i) {  // node i's value, i the same in all lanes
                int x = 0;
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (i >> 6 == r) x = __builtin_amdgcn_readlane(v[r], i & 63);
                return x;
            };
            int cur = 0;
            for (;;) {
                const int c = of(id, cur), from = of(slot, cur), to = of(slot, n);  // (lane reads: before the lanes part)
                if (lane == 0) {
                    const bool moved = cur != n;
                    chosen[n] = c;
                    runs[3 * n] = moved ? from : 0;
                    runs[3 * n + 1] = moved ? to : 0;
                    runs[3 * n + 2] = moved;
                }
                last = cur;
                n++;
                if (n == a.max_path || c < 0) break;
                int next = -1;
#pragma unroll
                for (int r = R - 1; r >= 0; r--) {
                    const uint64_t hit = __ballot(par[r] == cur && tok[r] == c && 64 * r + lane > cur);
                    if (hit) next = 64 * r + __builtin_ctzll(hit);
                }
                if (next < 0) break;
                cur = next;
            }
            last += q.q0;
            keep = q.base + n;
            moves = n;
        }
    }
    for (int i = n + lane; i < a.max_path; i += 64) chosen[i] = -1;
    for (int i = 3 * moves + lane; i < 3 * a.max_path; i += 64) runs[i] = 0;
    if (lane == 0) {
        a.n_path[s] = n;
        a.last[s] = last;
        a.keep[s] = keep;
    }
}

hipError_t launch_tree_accept(const TreeAccept& a, hipStream_t s) {
    if (!a.nseq) return hipSuccess;
    const dim3 grid((unsigned)a.nseq);
    if (a.words <= 2) tree_accept_kernel<1><<<grid, dim3(64), 0, s>>>(a);
    else if (a.words <= 4) tree_accept_kernel<2><<<grid, dim3(64), 0, s>>>(a);
    else tree_accept_kernel<4><<<grid, dim3(64), 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace strata
