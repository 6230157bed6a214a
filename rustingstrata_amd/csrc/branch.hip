// Sequences that go on from others (strata_kv_pages_fork) and rows of the caches moved from slot to slot (strata_kv_rows_move).
#include "branch.h"

#include <algorithm>

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
// Phases, each after all of the one before: the plan (a block); copies of the tables that others go on from and
// cleared claims; the holders' counts; the pages that go; the stack and tables. Where the tables have few entries one block of 1024
// threads does them all over lists of the entries that are kept and let go, whatever sequence they belong to; else four launches, a wave
// a sequence. Bound by latency: every phase is a chain of trips to memory. Entries are those that the tables have room for (the host knows no
// lengths). Beams, tables of 272 entries 8.8 us in one block and 13.0 in four launches, 1344 11.0 and 13.8, 5376 30 and 16.6. Without src the
// pages let go decide (us in one block / in four launches, pages of 16, 4096, 16384 and 32768 entries of 256 sequences): all cut
// inside their last page 5.8 / 11.4 at each, every 16th ended 8.8 / 12.1, 14.9 / 12.2, 24 / 14, all ended at once 34 / 14, 141 / 16,
// 279 / 21; 32 sequences of 1024 pages 5.5 / 10.2, 24 / 47, 278 / 94. The cuts of every step are what the limit serves; the end of
// everything at once pays for it. (The end of a step of 256 trees over tables of 12: 16.1 us and 20.9.)
constexpr long long FORK_ONE = 1 << 15, FORK_ONE_SRC = 1 << 11;
enum { F_CHANGED = 1, F_OTHER = 2, F_TAKE = 4, F_COPY = 8 };

struct ForkPlan {
    int flags, full, pg, fresh;  // pg: the page with the rem rows; fresh: its copy's
    int held, rem, len, pad;     // positions before; rows of pg; the length to report
};
struct ForkScratch {
    int* head;                    // pages on the stack before, pages taken
    ForkPlan* plan;               // [nseq]
    int* gone;                    // [nseq] pages that go back
    unsigned long long* claim;    // [n_pages]
    int* snap;                    // [nseq][max_pages] the pages of src[s]; of one block its lists
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
    return 64 + (sizeof(ForkPlan) + 4) * SERVE_MAX_SEQ + (size_t)a.n_pages * 8 + std::max(a.src ? (size_t)a.nseq * a.max_pages * 4 : 0, (size_t)FORK_ONE * 12);
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

// Exclusive sums of a value a thread over a block of 1024, and the total. ws: 16 words.
__device__ __forceinline__ int fork_scan(int v, int& total, int* ws) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
    }
    __syncthreads();  // (ws is free)
    if (lane == 63) ws[wave] = inc;
    __syncthreads();
    int at = inc - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w < wave) at += ws[w];
        total += ws[w];
    }
    return at;
}

// Phase 0a, a block of 1024 threads: sequences tid + 1024 i of the thread in p[i] (up to 1024 sequences one a thread: four in a row wait
// for each other's loads, 256 cut sequences 12.3 us for 8.5). heir, most: nseq words of LDS each; ws: 16.
__device__ __forceinline__ void fork_plan(const PagesFork& a, ForkPlan (&p)[4], int& stack, int& used, int* heir, int* most, int* ws) {
    const int tid = threadIdx.x;
    for (int s = tid; s < a.nseq; s += 1024) {
        heir[s] = INT32_MAX;
        most[s] = -1;
    }
    stack = min(max(*a.n_free, 0), a.n_pages);
    __syncthreads();
    ForkSeq q[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = tid + 1024 * i;
        if (s >= a.nseq) continue;
        q[i] = fork_seq(a, s);
        atomicMin(&heir[q[i].src], q[i].src == s ? -1 : s);
        atomicMax(&most[q[i].src], q[i].k >> a.page_shift);
    }
    __syncthreads();
    int need[4] = {0, 0, 0, 0}, err = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = tid + 1024 * i;
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
            need[i] = !takes;
        }
    }
    int wanted = 0;  // pages, by the sequences before
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = tid + 1024 * i;
        if (1024 * i >= a.nseq) break;
        int total, at = wanted + fork_scan(need[i], total, ws);
        wanted += total;
        if (s >= a.nseq || !(p[i].flags & F_CHANGED)) continue;
        const bool refused = (p[i].flags & F_COPY) && at >= stack;
        if (!refused) {
            if (p[i].flags & F_COPY) p[i].fresh = a.free_pages[stack - 1 - at];
            p[i].len = q[i].k;
        } else {  // no page: a cut is not made, a sequence that was to become another is empty
            err++;
            p[i].full = p[i].rem = 0;
            if (p[i].flags & F_OTHER) p[i].len = 0;
            p[i].flags = p[i].flags & F_OTHER ? F_CHANGED | F_OTHER : 0;
        }
    }
    err = __syncthreads_count(err & 1) + 2 * __syncthreads_count(err & 2) + 4 * __syncthreads_count(err & 4);  // (at most 4)
    used = min(wanted, stack);
    if (tid == 0 && a.err && err) atomicAdd(a.err, err);
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
// What the caller reads of sequence s, and its copied page's place.
__device__ __forceinline__ void fork_report(const PagesFork& a, int s, const ForkPlan& p) {
    if (p.flags & F_COPY) a.tables[(uint64_t)s * a.max_pages + p.full] = p.fresh;  // (a page from the stack has no other holder: refs 0)
    const bool copy = (p.flags & F_COPY) && in_pool(a, p.fresh);
    a.runs[3 * s] = copy ? p.pg << a.page_shift : 0;
    a.runs[3 * s + 1] = copy ? p.fresh << a.page_shift : 0;
    a.runs[3 * s + 2] = copy ? p.rem : 0;
    a.len_out[s] = p.len;
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
    }
    if (lane == 0) {
        fork_report(a, s, p);
        if (s == 0) {
            *a.n_free_out = min(stack - used + all, a.n_pages);
            if (a.err && stack - used + all > a.n_pages) atomicAdd(a.err, 1);
        }
    }
}

// The last sequence with v[s] <= x.
__device__ __forceinline__ int fork_find(const int* v, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
__global__ __launch_bounds__(1024) void pages_fork_one_kernel(PagesFork a) {
    __shared__ int heir[SERVE_MAX_SEQ], most[SERVE_MAX_SEQ], first[SERVE_MAX_SEQ], srcs[SERVE_MAX_SEQ], ws[16];
    const ForkScratch f = fork_scratch(a);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    ForkPlan p[4];
    int stack, used;
    fork_plan(a, p, stack, used, heir, most, ws);
    // the lists: entry i of those kept is the first ones of another's table, entry i of those let go at place `first` on
    int *kept0 = heir, *gone0 = most;
    unsigned sums = 0;  // of the sequences before: those kept in the upper half, those let go in the lower one (up to FORK_ONE each)
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = tid + 1024 * i;
        if (1024 * i >= a.nseq) break;
        unsigned n = 0;
        if (s < a.nseq && (p[i].flags & F_CHANGED)) {
            n = max(pages_of(a, p[i].held) - fork_from(p[i]), 0);
            if (p[i].flags & F_OTHER) n += (unsigned)fork_kept(p[i]) << 16;
        }
        int total;
        const unsigned at = sums + (unsigned)fork_scan((int)n, total, ws);  // (its barriers: heir and most have been read)
        sums += (unsigned)total;
        if (s < a.nseq) {
            kept0[s] = at >> 16;
            gone0[s] = at & 0xFFFF;
            first[s] = fork_from(p[i]);
            srcs[s] = a.src ? a.src[s] : s;
        }
    }
    const int n_kept = sums >> 16, n_gone = sums & 0xFFFF;
    __syncthreads();
    int *keep_page = f.snap, *keep_cell = keep_page + FORK_ONE, *gone_page = keep_cell + FORK_ONE;
    for (int i = tid; i < n_kept; i += 1024) {
        const int s = fork_find(kept0, a.nseq, i), j = i - kept0[s], pg = a.tables[(uint64_t)srcs[s] * a.max_pages + j];
        keep_page[i] = pg;
        keep_cell[i] = s * a.max_pages + j;
        if (in_pool(a, pg)) atomicAdd(a.refs + pg, 1);
    }
    for (int i = tid; i < n_gone; i += 1024) {
        const int s = fork_find(gone0, a.nseq, i), j = first[s] + i - gone0[s], pg = a.tables[(uint64_t)s * a.max_pages + j];
        gone_page[i] = pg;
        if (in_pool(a, pg)) __hip_atomic_store(f.claim + pg, ~0ull, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    for (int i = tid; i < n_gone; i += 1024) {
        const int pg = gone_page[i];
        if (in_pool(a, pg)) {
            atomicSub(a.refs + pg, 1);
            atomicMin(f.claim + pg, (unsigned long long)i);
        }
    }
    __syncthreads();
    int at = stack - used;  // the next place on the stack
    for (int i0 = 0; i0 < n_gone; i0 += 1024) {
        const int i = i0 + tid, pg = i < n_gone ? gone_page[i] : -1;
        const bool goes = fork_goes(a, f, i, pg);
        const uint64_t b = __ballot(goes);
        __syncthreads();  // (ws is free)
        if (lane == 0) ws[wave] = __popcll(b);
        __syncthreads();
        int to = at + __popcll(b & ((1ull << lane) - 1));
#pragma unroll
        for (int w = 0; w < 16; w++) {
            if (w < wave) to += ws[w];
            at += ws[w];
        }
        if (goes) {
            if (to < a.n_pages) a.free_pages[to] = pg;
            __hip_atomic_store(a.refs + pg, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    // (all table entries that others go on from, and all that go, have been read)
    for (int i = tid; i < n_kept; i += 1024) a.tables[keep_cell[i]] = keep_page[i];
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (tid + 1024 * i < a.nseq) fork_report(a, tid + 1024 * i, p[i]);
    if (tid == 0) {
        *a.n_free_out = min(at, a.n_pages);
        if (a.err && at > a.n_pages) atomicAdd(a.err, 1);
    }
}
__global__ __launch_bounds__(1024) void pages_fork_plan_kernel(PagesFork a) {
    const ForkScratch f = fork_scratch(a);
    if (blockIdx.x == 0) {
        __shared__ int heir[SERVE_MAX_SEQ], most[SERVE_MAX_SEQ], ws[16];
        ForkPlan p[4];
        int stack, used;
        fork_plan(a, p, stack, used, heir, most, ws);
#pragma unroll
        for (int i = 0; i < 4; i++)
            if ((int)threadIdx.x + 1024 * i < a.nseq) f.plan[threadIdx.x + 1024 * i] = p[i];
        if (threadIdx.x == 0) {
            f.head[0] = stack;
            f.head[1] = used;
        }
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
    if ((long long)a.nseq * a.max_pages <= (a.src ? FORK_ONE_SRC : FORK_ONE)) {
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
// A block takes a group's runs (from, to, n: n consecutive rows) in `cpb` caches, their rows one cache behind the other, in batches:
// all of a batch are read before any of it is written, and batches follow each other, so rows that move towards the front over rows
// already read come out right (a confirmed path closing up). A row's 16-byte chunks go to `tpr` threads, a power of two from 8 to
// 256; MOVE_U rows a thread are in flight. Copies of pages are bound by their bytes (256 groups of 32 rows of 1 KB in 96 caches 311 us,
// 5.2 TB/s), a few rows a group by the chain of a block (the runs, their sums, the rows), hence several caches a block there (256
// confirmed paths in 24 caches 12.8 us with one, 5.6 with six).
constexpr int MOVE_MAX_RUNS = 256, MOVE_U = 8;

__global__ __launch_bounds__(256) void rows_move_kernel(RowsMove a, int tpr_shift, int cpb, unsigned first) {
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    __shared__ int from[MOVE_MAX_RUNS], to[MOVE_MAX_RUNS];
    __shared__ uint64_t rs[256], rd[256];
    __shared__ long long start[MOVE_MAX_RUNS], ws[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int parts = (a.n_caches + cpb - 1) / cpb;
    const unsigned at = first + blockIdx.x;
    const int g = at / parts, c0 = at % parts * cpb, nc = min(cpb, a.n_caches - c0);
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
    for (int o = 1; o < 64 && o < a.per; o <<= 1) {
        const long long u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
    }
    if (lane == min(63, a.per - 1 - 64 * wave)) ws[wave] = inc;
    if (lane == 0 && 64 * wave >= a.per) ws[wave] = 0;
    __syncthreads();
    for (int w = 0; w < wave; w++) inc += ws[w];
    const long long rows = ws[0] + ws[1] + ws[2] + ws[3], total = rows * nc;
    if (!total) return;
    start[tid] = inc - n;
    __syncthreads();
    const int tpr = 1 << tpr_shift, step = 256 >> tpr_shift, batch = step * MOVE_U, row = tid >> tpr_shift;
    const uint64_t chunks = a.row_bytes / 16;
    for (long long b = 0; b < total; b += batch) {
        const int m = (int)min(total - b, (long long)batch);
        if (tid < m) {  // row x of cache c: of the last run that begins there or before
            const long long c = (b + tid) / rows, x = b + tid - c * rows;
            int lo = 0, hi = a.per;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= x) lo = mid;
                else hi = mid;
            }
            const uint64_t base = a.caches[c0 + c];
            const int i = (int)(x - start[lo]);
            rs[tid] = base + (uint64_t)(from[lo] + i) * a.row_bytes;
            rd[tid] = base + (uint64_t)(to[lo] + i) * a.row_bytes;
        }
        __syncthreads();
        for (uint64_t col = tid & (tpr - 1); col - (tid & (tpr - 1)) < chunks; col += tpr) {
            v4u v[MOVE_U];
#pragma unroll
            for (int u = 0; u < MOVE_U; u++) {
                const int i = u * step + row;
                if (i < m && col < chunks) v[u] = *gptr<v4u>(rs[i] + 16 * col);
            }
            wait_loads();
            __syncthreads();
#pragma unroll
            for (int u = 0; u < MOVE_U; u++) {
                const int i = u * step + row;
                if (i < m && col < chunks) *(v4u*)(rd[i] + 16 * col) = v[u];
            }
        }
        __syncthreads();
    }
}

hipError_t launch_rows_move(const RowsMove& a, hipStream_t s) {
    if (!a.groups || !a.n_caches || !a.per) return hipSuccess;
    int shift = 3;
    while (shift < 8 && (16ull << shift) < a.row_bytes) shift++;
    // one cache a block where a group is one run (pages' rows); else caches as leave four blocks a CU
    const int cpb = a.per == 1 ? 1 : (int)std::max<long long>(1, std::min<long long>(8, (long long)a.groups * a.n_caches / 1024));
    // HIP's launches have fewer than 2^32 threads: more blocks go on in further ones (a captured launch of more is refused)
    constexpr uint64_t most = 1 << 23;
    const uint64_t blocks = (uint64_t)a.groups * ((a.n_caches + cpb - 1) / cpb);
    for (uint64_t first = 0; first < blocks; first += most)
        rows_move_kernel<<<dim3((unsigned)std::min(blocks - first, most)), dim3(256), 0, s>>>(a, shift, cpb, (unsigned)first);
    return hipGetLastError();
}

}  // namespace strata
