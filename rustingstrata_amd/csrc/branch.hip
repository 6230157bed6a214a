// Sequences that go on from others (strata_kv_pages_fork) and rows of the caches moved from slot to slot (strata_kv_rows_move).
#include "branch.h"

namespace strata {

// ---------------- forking, cutting and ending ----------------
// Sequence s becomes the first k[s] positions of what sequence u = src[s] held before the call. With full = k / page, rem = k %
// page: its `full` first pages are u's (refs[p], the holders of page p but one, goes up by one for each), and where rem > 0
// the page behind them is
//   taken over, if s is u's heir (u itself, or else the first that goes on from u), nobody else holds the page (refs 0) and no
//   sequence that goes on from u keeps it as a full one;
//   else a new page from the stack, rem rows to be copied (runs[s]).
// Pages that a changed sequence held go down by one each; those that nobody holds any more go on the stack, behind the pages
// taken, in the order (sequence, place in its table) in which they are first met. That order comes from `claim`: the smallest
// s * max_pages + j over a page's releases, so the stack does not depend on the order of atomics.
// Four phases, each after all of the one before: the plan (a block; 4 sequences a thread) beside copies of the tables that others
// go on from and cleared claims; the holders' counts; the pages that go; the stack and tables. Up to FORK_ONE sequences run them
// in one block with a wave a sequence, more in four launches. Bound by latency: every phase is a chain of two or three trips to memory.
constexpr int FORK_ONE = 16;
enum { F_CHANGED = 1, F_OTHER = 2, F_TAKE = 4, F_COPY = 8, F_EMPTY = 16, F_LOST = 32 };

struct ForkPlan {
    int flags, full, pg, fresh;  // pg: the page with the rem rows; fresh: its copy's
    int held, rem, len, pad;     // positions before; rows of pg; the length to report
};
struct ForkScratch {
    int* head;                    // pages on the stack before, pages taken
    ForkPlan* plan;               // [nseq]
    int* gone;                    // [nseq] pages that go back
    unsigned long long* claim;    // [n_pages]
    int* snap;                    // [nseq][max_pages] the pages of src[s]
};
__host__ __device__ static inline ForkScratch fork_scratch(const PagesFork& a) {
    ForkScratch f;
    uint8_t* p = (uint8_t*)a.scratch;
    f.head = (int*)p;
    f.plan = (ForkPlan*)(p + 64);
    f.gone = (int*)(p + 64 + sizeof(ForkPlan) * SERVE_MAX_SEQ);
    f.claim = (unsigned long long*)(p + 64 + (sizeof(ForkPlan) + 4) * SERVE_MAX_SEQ);
    f.snap = (int*)(f.claim + a.n_pages);
    return f;
}
size_t pages_fork_scratch_bytes(const PagesFork& a) {
    return 64 + (sizeof(ForkPlan) + 4) * SERVE_MAX_SEQ + (size_t)a.n_pages * 8 + (a.src ? (size_t)a.nseq * a.max_pages * 4 : 0);
}

struct ForkSeq {
    int src, held, k;  // held: positions before (of s); k: positions that it keeps
    bool ok;           // src is a sequence
};
__device__ __forceinline__ ForkSeq fork_seq(const PagesFork& a, int s) {
    ForkSeq r;
    const int limit = (int)min((long long)a.max_pages << a.page_shift, (long long)INT32_MAX);
    const int u = a.src ? a.src[s] : s;
    r.ok = u >= 0 && u < a.nseq;
    r.src = r.ok ? u : s;
    r.held = min(max(a.len[s], 0), limit);
    const int n = r.src == s ? r.held : min(max(a.len[r.src], 0), limit);
    r.k = r.ok && a.keep ? min(max(a.keep[s], 0), n) : n;
    return r;
}
__device__ __forceinline__ int pages_of(const PagesFork& a, int n) { return (int)(((long long)n + (1 << a.page_shift) - 1) >> a.page_shift); }
__device__ __forceinline__ bool in_pool(const PagesFork& a, int p) { return p >= 0 && p < a.n_pages; }
// Counts that other waves have changed: past this CU's L1.
__device__ __forceinline__ int shared_load(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned long long shared_load(const unsigned long long* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Phase 0a, a block of 1024 threads.
__device__ void fork_plan(const PagesFork& a, const ForkScratch& f) {
    __shared__ int heir[SERVE_MAX_SEQ], most[SERVE_MAX_SEQ], ws[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int s = tid; s < a.nseq; s += 1024) {
        heir[s] = INT32_MAX;
        most[s] = -1;
    }
    const int stack = min(max(*a.n_free, 0), a.n_pages);
    __syncthreads();
    ForkSeq q[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = 4 * tid + i;
        if (s >= a.nseq) continue;
        q[i] = fork_seq(a, s);
        atomicMin(&heir[q[i].src], q[i].src == s ? -1 : s);
        atomicMax(&most[q[i].src], q[i].k >> a.page_shift);
    }
    __syncthreads();
    ForkPlan p[4];
    int need = 0, err = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = 4 * tid + i;
        p[i] = ForkPlan{0, 0, -1, -1, 0, 0, 0, 0};
        if (s >= a.nseq) continue;
        const int full = q[i].k >> a.page_shift, rem = q[i].k & ((1 << a.page_shift) - 1), u = q[i].src;
        err += !q[i].ok;
        p[i].held = q[i].held;
        p[i].len = a.len[s];
        if (u == s && q[i].k == q[i].held) continue;
        p[i].flags = F_CHANGED | (u != s ? F_OTHER : 0);
        p[i].full = full;
        p[i].rem = rem;
        if (rem) {
            p[i].pg = a.tables[(uint64_t)u * a.max_pages + full];
            const bool known = in_pool(a, p[i].pg);
            const bool takes = !known || (heir[u] == (u == s ? -1 : s) && most[u] <= full && a.refs[p[i].pg] == 0);
            p[i].flags |= takes ? F_TAKE : F_COPY;
            need += !takes;
        }
    }
    // the pages wanted before this thread's
    int inc = need;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
    }
    if (lane == 63) ws[wave] = inc;
    __syncthreads();
    int at = inc - need, total = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w < wave) at += ws[w];
        total += ws[w];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = 4 * tid + i;
        if (s >= a.nseq) continue;
        if (p[i].flags & F_CHANGED) {
            bool refused = false;
            if (p[i].flags & F_COPY) {
                refused = at >= stack;
                if (!refused) p[i].fresh = a.free_pages[stack - 1 - at];
                at++;
            }
            if (!refused) {
                p[i].len = q[i].k;
            } else {  // no page: a cut is not made, a sequence that was to become another is empty
                err++;
                p[i].full = p[i].rem = 0;
                if (p[i].flags & F_OTHER) p[i].len = 0;
                p[i].flags = p[i].flags & F_OTHER ? F_CHANGED | F_OTHER : 0;
            }
        }
        f.plan[s] = p[i];
    }
    err = __syncthreads_count(err & 1) + 2 * __syncthreads_count(err & 2) + 4 * __syncthreads_count(err & 4);  // (at most 4)
    if (tid == 0) {
        f.head[0] = stack;
        f.head[1] = min(total, stack);
        if (a.err && err) atomicAdd(a.err, err);
    }
}
// Phase 0b, a wave: the pages of the sequence that s goes on from, and the claims of those that it may let go.
__device__ __forceinline__ void fork_copy(const PagesFork& a, const ForkScratch& f, int s) {
    const int lane = threadIdx.x & 63;
    const ForkSeq q = fork_seq(a, s);
    if (q.src == s && q.k == q.held) return;
    if (q.src != s)
        for (int j = lane; j < pages_of(a, q.k); j += 64) f.snap[(uint64_t)s * a.max_pages + j] = a.tables[(uint64_t)q.src * a.max_pages + j];
    for (int j = (q.src == s ? q.k >> a.page_shift : 0) + lane; j < pages_of(a, q.held); j += 64) {
        const int p = a.tables[(uint64_t)s * a.max_pages + j];
        if (in_pool(a, p)) __hip_atomic_store(f.claim + p, ~0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}
// The places of s's table whose pages it lets go are fork_from .. pages_of(held) - 1, those that it has from another 0 .. fork_kept - 1.
__device__ __forceinline__ int fork_kept(const ForkPlan& p) { return p.full + (p.flags & F_TAKE ? 1 : 0); }
__device__ __forceinline__ int fork_from(const ForkPlan& p) { return p.flags & F_OTHER ? 0 : fork_kept(p); }
// Phase 1, a wave: the holders' counts.
__device__ __forceinline__ void fork_count(const PagesFork& a, const ForkScratch& f, int s) {
    const int lane = threadIdx.x & 63;
    const ForkPlan p = f.plan[s];
    if (!(p.flags & F_CHANGED)) return;
    const uint64_t row = (uint64_t)s * a.max_pages;
    if (p.flags & F_OTHER)
        for (int j = lane; j < fork_kept(p); j += 64) {
            const int pg = f.snap[row + j];
            if (in_pool(a, pg)) atomicAdd(a.refs + pg, 1);
        }
    for (int j = fork_from(p) + lane; j < pages_of(a, p.held); j += 64) {
        const int pg = a.tables[row + j];
        if (in_pool(a, pg)) {
            atomicSub(a.refs + pg, 1);
            atomicMin(f.claim + pg, (unsigned long long)(row + j));
        }
    }
}
__device__ __forceinline__ bool fork_goes(const PagesFork& a, const ForkScratch& f, uint64_t cell, int pg) {
    return in_pool(a, pg) && shared_load(a.refs + pg) < 0 && shared_load(f.claim + pg) == cell;
}
// Phase 2, a wave: how many pages go back.
__device__ __forceinline__ void fork_gone(const PagesFork& a, const ForkScratch& f, int s) {
    const int lane = threadIdx.x & 63;
    const ForkPlan p = f.plan[s];
    const uint64_t row = (uint64_t)s * a.max_pages;
    int n = 0;
    if (p.flags & F_CHANGED) {
        for (int j = fork_from(p) + lane; j < pages_of(a, p.held); j += 64) n += fork_goes(a, f, row + j, a.tables[row + j]);
#pragma unroll
        for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o, 64);
    }
    if (lane == 0) f.gone[s] = n;
}
// Phase 3, a wave: the stack, the table and what the caller reads. (It reads no input that an output may lie over.)
__device__ __forceinline__ void fork_apply(const PagesFork& a, const ForkScratch& f, int s) {
    const int lane = threadIdx.x & 63;
    const ForkPlan p = f.plan[s];
    const int stack = f.head[0], used = f.head[1];
    const uint64_t row = (uint64_t)s * a.max_pages;
    int before = 0, all = 0;  // pages that go back: of the sequences before, of all
    for (int i = lane; i < a.nseq; i += 64) {
        const int n = f.gone[i];
        all += n;
        before += i < s ? n : 0;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        before += __shfl_xor(before, o, 64);
        all += __shfl_xor(all, o, 64);
    }
    if (p.flags & F_CHANGED) {
        int at = stack - used + before;
        const int end = pages_of(a, p.held);
        for (int j0 = fork_from(p); j0 < end; j0 += 64) {
            const int j = j0 + lane, pg = j < end ? a.tables[row + j] : -1;
            const bool goes = fork_goes(a, f, row + j, pg);
            const uint64_t b = __ballot(goes);
            if (goes) {
                const int to = at + __popcll(b & ((1ull << lane) - 1));
                if (to < a.n_pages) a.free_pages[to] = pg;
                __hip_atomic_store(a.refs + pg, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            at += __popcll(b);
        }
        // (the same lane wrote what it read above, or a place that nothing above reads)
        if (p.flags & F_OTHER)
            for (int j = lane; j < fork_kept(p); j += 64) a.tables[row + j] = f.snap[row + j];
        if (lane == 0 && (p.flags & F_COPY)) a.tables[row + p.full] = p.fresh;  // (a page from the stack has no other holder: refs 0)
    }
    if (lane == 0) {
        const bool copy = (p.flags & F_COPY) && in_pool(a, p.fresh);
        a.runs[3 * s] = copy ? p.pg << a.page_shift : 0;
        a.runs[3 * s + 1] = copy ? p.fresh << a.page_shift : 0;
        a.runs[3 * s + 2] = copy ? p.rem : 0;
        a.len_out[s] = p.len;
        if (s == 0) {
            *a.n_free_out = min(stack - used + all, a.n_pages);
            if (a.err && stack - used + all > a.n_pages) atomicAdd(a.err, 1);
        }
    }
}

__global__ __launch_bounds__(1024) void pages_fork_one_kernel(PagesFork a) {
    const ForkScratch f = fork_scratch(a);
    const int s = threadIdx.x >> 6;
    fork_plan(a, f);
    if (s < a.nseq) fork_copy(a, f, s);
    __syncthreads();
    if (s < a.nseq) fork_count(a, f, s);
    __syncthreads();
    if (s < a.nseq) fork_gone(a, f, s);
    __syncthreads();
    if (s < a.nseq) fork_apply(a, f, s);
}
__global__ __launch_bounds__(1024) void pages_fork_plan_kernel(PagesFork a) {
    const ForkScratch f = fork_scratch(a);
    if (blockIdx.x == 0) {
        fork_plan(a, f);
    } else {
        const int s = (blockIdx.x - 1) * 16 + (threadIdx.x >> 6);
        if (s < a.nseq) fork_copy(a, f, s);
    }
}
template <int PHASE>
__global__ __launch_bounds__(256) void pages_fork_kernel(PagesFork a) {
    const ForkScratch f = fork_scratch(a);
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s >= a.nseq) return;
    if constexpr (PHASE == 1) fork_count(a, f, s);
    else if constexpr (PHASE == 2) fork_gone(a, f, s);
    else fork_apply(a, f, s);
}

hipError_t launch_pages_fork(const PagesFork& a, hipStream_t s) {
    if (!a.nseq) return hipSuccess;
    if (a.nseq <= FORK_ONE) {
        pages_fork_one_kernel<<<dim3(1), dim3(1024), 0, s>>>(a);
    } else {
        const dim3 grid((unsigned)(a.nseq + 3) / 4);
        pages_fork_plan_kernel<<<dim3(1 + (unsigned)(a.nseq + 15) / 16), dim3(1024), 0, s>>>(a);
        pages_fork_kernel<1><<<grid, dim3(256), 0, s>>>(a);
        pages_fork_kernel<2><<<grid, dim3(256), 0, s>>>(a);
        pages_fork_kernel<3><<<grid, dim3(256), 0, s>>>(a);
    }
    return hipGetLastError();
}

// ---------------- rows of the caches ----------------
// A block per group and cache takes the group's runs (from, to, n: n consecutive rows) in batches of rows: all of a batch are read
// before any of it is written, and batches follow each other, so rows that move towards the front over rows already read come out
// right (a confirmed path closing up). A row's 16-byte chunks go to `tpr` threads, a power of two from 8 to 256; MOVE_U rows a
// thread are in flight.
constexpr int MOVE_MAX_RUNS = 256, MOVE_U = 8;

__global__ __launch_bounds__(256) void rows_move_kernel(RowsMove a, int tpr_shift) {
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    __shared__ int from[MOVE_MAX_RUNS], to[MOVE_MAX_RUNS], rf[256], rt[256];
    __shared__ long long start[MOVE_MAX_RUNS], ws[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int g = blockIdx.x / a.n_caches, c = blockIdx.x % a.n_caches;
    const uint64_t base = sload(a.caches + c);
    long long n = 0;
    if (tid < a.per) {
        const int* r = a.runs + ((uint64_t)g * a.per + tid) * 3;
        from[tid] = r[0];
        to[tid] = r[1];
        n = r[2];
        // (a run that leaves the caches is left out)
        if (n < 0 || r[0] < 0 || r[1] < 0 || (uint64_t)(r[0] + n) > a.n_slots || (uint64_t)(r[1] + n) > a.n_slots) n = 0;
    }
    long long inc = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
    }
    if (lane == 63) ws[wave] = inc;
    __syncthreads();
    for (int w = 0; w < wave; w++) inc += ws[w];
    const long long total = ws[0] + ws[1] + ws[2] + ws[3];
    if (!total) return;
    start[tid] = inc - n;
    __syncthreads();
    const int tpr = 1 << tpr_shift, rows = 256 >> tpr_shift, batch = rows * MOVE_U, row = tid >> tpr_shift;
    const uint64_t chunks = a.row_bytes / 16;
    for (long long b = 0; b < total; b += batch) {
        const int m = (int)min(total - b, (long long)batch);
        if (tid < m) {  // row b + tid: the last run that begins there or before
            int lo = 0, hi = a.per;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= b + tid) lo = mid;
                else hi = mid;
            }
            const int i = (int)(b + tid - start[lo]);
            rf[tid] = from[lo] + i;
            rt[tid] = to[lo] + i;
        }
        __syncthreads();
        for (uint64_t col = tid & (tpr - 1); col - (tid & (tpr - 1)) < chunks; col += tpr) {
            v4u v[MOVE_U];
#pragma unroll
            for (int u = 0; u < MOVE_U; u++) {
                const int i = u * rows + row;
                if (i < m && col < chunks) v[u] = *gptr<v4u>(base + (uint64_t)rf[i] * a.row_bytes + 16 * col);
            }
            wait_loads();
            __syncthreads();
#pragma unroll
            for (int u = 0; u < MOVE_U; u++) {
                const int i = u * rows + row;
                if (i < m && col < chunks) *(v4u*)(base + (uint64_t)rt[i] * a.row_bytes + 16 * col) = v[u];
            }
        }
        __syncthreads();
    }
}

hipError_t launch_rows_move(const RowsMove& a, hipStream_t s) {
    if (!a.groups || !a.n_caches || !a.per) return hipSuccess;
    int shift = 3;
    while (shift < 8 && (16ull << shift) < a.row_bytes) shift++;
    rows_move_kernel<<<dim3((unsigned)((uint64_t)a.groups * a.n_caches)), dim3(256), 0, s>>>(a, shift);
    return hipGetLastError();
}

}  // namespace strata
