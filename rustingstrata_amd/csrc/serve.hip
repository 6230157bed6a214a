// Serving a batch of sequences: the step of the page tables (strata_kv_pages_step) and the processing of logits before the
// choice of a token (strata_logits_process). Neither has a counterpart in the reference's Backend trait, which serves one
// sequence with a contiguous cache and samples on the host.
#include "serve.h"

#include <algorithm>

#include "argmax_key.h"
#include "xlane.h"

namespace strata {

// ---------------- page tables and slot maps ----------------
// From the sequences' cached lengths and new tokens, all integers:
//   have[s] = ceil(len / page) pages held, need[s] = ceil((len + add) / page) - have[s] pages wanted;
//   sequences that end (add < 0) push their pages on the stack of free pages in (sequence, page) order;
//   off = exclusive prefix sum of need: page j of sequence s's new ones is the (off + j)-th from the stack's top;
//   q_start = prefix sum of the new tokens, token t at own index i = len + t - q_start[s]: slot = page(i) * page + i % page.
// Sums saturate at SAT (2^30), beyond every limit they are compared with, so no count overflows. One block of 1024 threads:
// a thread sums 4 consecutive sequences, the waves' totals meet in LDS, and the tokens find their sequence by a binary search
// of q_start in LDS. Bound by latency (two rounds of loads and three barriers of scans): 8 sequences, one token each 6.6 us, 512
// with 8192 new tokens 11.6.
// More than PAGES_ONE tokens take a second launch over many blocks that searches q_start in memory (4096 tokens 9.6 us in one block,
// 10.0 in two launches; 2048 7.8 and 9.8; 8192 13.1 and 10.0).
constexpr int PAGES_ONE = 4096;
constexpr unsigned SAT = 1u << 30;
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, SAT); }  // a, b <= SAT

// Exclusive saturating prefix sum of 4 values a thread over a block of 1024 threads; the total to every thread. ws: 17 words.
__device__ __forceinline__ unsigned scan4(const unsigned (&v)[4], unsigned (&ex)[4], unsigned* ws) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned mine = sat_add(sat_add(v[0], v[1]), sat_add(v[2], v[3]));
    unsigned inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(inc, o, 64);
        if (lane >= o) inc = sat_add(inc, u);
    }
    unsigned before = __shfl_up(inc, 1, 64);
    if (lane == 0) before = 0;
    __syncthreads();  // (ws is free: its readers of the scan before are done)
    if (lane == 63) ws[wave] = inc;
    __syncthreads();
    unsigned base = 0, total = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        const unsigned u = ws[w];
        if (w < wave) base = sat_add(base, u);
        total = sat_add(total, u);
    }
    base = sat_add(base, before);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        ex[k] = base;
        base = sat_add(base, v[k]);
    }
    return total;
}

// The last i in 0 .. n - 1 with a[i] <= v (a[0] <= v, a not decreasing).
template <typename P>
__device__ __forceinline__ int last_le(P a, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Token t of sequence s: its position and slot, and the table entry of a page that it opens. len: the cached tokens before
// this step; refused: the sequence gets nothing.
__device__ __forceinline__ void place_token(const PagesStep& a, int t, int s, int start, int len, bool refused, int off, int top, int P) {
    const long long i = (long long)len + (t - start);
    a.pos[t] = (int)min(P + i, (long long)INT32_MAX);
    int slot = -1;
    if (!refused) {
        const int page = 1 << a.page_shift, have = (int)(((long long)len + page - 1) >> a.page_shift), pi = (int)(i >> a.page_shift);
        int* cell = a.tables + (uint64_t)s * a.max_pages + pi;
        int pg;
        if (pi >= have) {
            pg = a.free_pages[top - 1 - (off + pi - have)];
            if ((i & (page - 1)) == 0) *cell = pg;
        } else {
            pg = *cell;
        }
        if (pg >= 0 && pg < a.n_pages) slot = (pg << a.page_shift) + (int)(i & (page - 1));
    }
    a.slots[t] = slot;
}

// st[s]: the cached length before the step, or ~length of a refused sequence.
template <bool ONE>
__global__ __launch_bounds__(1024) void pages_plan_kernel(PagesStep a) {
    __shared__ int qs[SERVE_MAX_SEQ], po[SERVE_MAX_SEQ], st[SERVE_MAX_SEQ];
    __shared__ unsigned ws[17];
    const int tid = threadIdx.x, page = 1 << a.page_shift;
    const int limit = (int)min((long long)a.max_pages << a.page_shift, (long long)INT32_MAX);
    int add[4], len[4];
    unsigned v[4], ex[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int s = 4 * tid + k;
        add[k] = s < a.nseq ? a.add[s] : 0;
        len[k] = s < a.nseq ? a.len[s] : 0;
        v[k] = add[k] < 0 && len[k] > 0 ? (unsigned)((min(len[k], limit) + (long long)page - 1) >> a.page_shift) : 0u;
    }
    const int held = min(max(*a.n_free, 0), a.n_pages), P = a.prefix_len ? max(*a.prefix_len, 0) : 0;
    // sequences that end: their pages on the stack, entry i by thread i
    const unsigned back = scan4(v, ex, ws);
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (4 * tid + k < a.nseq) po[4 * tid + k] = (int)ex[k];
    __syncthreads();
    const int top = min(held + (int)back, a.n_pages);
    for (int i = tid; i < top - held; i += 1024) {
        const int s = last_le(po, a.nseq, i);
        a.free_pages[held + i] = a.tables[(uint64_t)s * a.max_pages + (i - po[s])];
    }
    // new tokens, then the pages that they need
    unsigned start[4];
    bool bad[4];
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = add[k] > 0 ? min((unsigned)add[k], SAT) : 0u;
    const unsigned total = scan4(v, start, ws);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const long long end = (long long)len[k] + add[k];
        bad[k] = add[k] > 0 && (len[k] < 0 || end > limit || sat_add(start[k], v[k]) > (unsigned)a.t_max);
        v[k] = add[k] > 0 && !bad[k] ? (unsigned)(((end + page - 1) >> a.page_shift) - (((long long)len[k] + page - 1) >> a.page_shift)) : 0u;
    }
    scan4(v, ex, ws);  // (its barriers: the pushed pages are written, po has been read)
    int refused = back > (unsigned)(a.n_pages - held) ? 1 : 0;
    refused = tid ? 0 : refused;  // (a stack that overflows counts once)
    unsigned used = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const int s = 4 * tid + k;
        if (v[k] && sat_add(ex[k], v[k]) > (unsigned)top) bad[k] = true;
        if (!bad[k] && v[k]) used = ex[k] + v[k];  // (the sequences that get pages come before all that do not)
        refused += bad[k];
        if (s < a.nseq) {
            qs[s] = (int)min(start[k], (unsigned)a.t_max);
            po[s] = (int)ex[k];
            st[s] = bad[k] ? ~max(len[k], 0) : max(len[k], 0);
            a.q_start[s] = qs[s];
            a.len_out[s] = add[k] < 0 ? 0 : bad[k] || add[k] == 0 ? len[k] : len[k] + add[k];
            if constexpr (!ONE) {
                a.scratch[4 + s] = po[s];
                a.scratch[4 + SERVE_MAX_SEQ + s] = st[s];
            }
        }
    }
    // the pages taken (the largest `used`) and the sequences refused, over the block
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        used = max(used, (unsigned)__shfl_xor((int)used, o, 64));
        refused += __shfl_xor(refused, o, 64);
    }
    __shared__ unsigned us[16];
    __shared__ int rs[16];
    if ((tid & 63) == 0) {
        us[tid >> 6] = used;
        rs[tid >> 6] = refused;
    }
    __syncthreads();
    const int rows = (int)min(total, (unsigned)a.t_max);
    if (tid == 0) {
        for (int w = 1; w < 16; w++) {
            used = max(used, us[w]);
            refused += rs[w];
        }
        a.q_start[a.nseq] = rows;
        *a.n_free_out = top - (int)used;
        if (a.err && refused) *a.err += refused;
        if constexpr (!ONE) {
            a.scratch[0] = rows;
            a.scratch[1] = top;
            a.scratch[2] = P;
        }
    }
    if constexpr (ONE) {
        for (int t = tid; t < a.t_max; t += 1024) {
            if (t < rows) {
                const int s = last_le(qs, a.nseq, t), f = st[s];
                place_token(a, t, s, qs[s], f < 0 ? ~f : f, f < 0, po[s], top, P);
            } else {
                a.pos[t] = a.slots[t] = -1;
            }
        }
    }
}

__global__ __launch_bounds__(256) void pages_place_kernel(PagesStep a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= a.t_max) return;
    if (t < a.scratch[0]) {
        const int s = last_le(a.q_start, a.nseq, t), f = a.scratch[4 + SERVE_MAX_SEQ + s];
        place_token(a, t, s, a.q_start[s], f < 0 ? ~f : f, f < 0, a.scratch[4 + s], a.scratch[1], a.scratch[2]);
    } else {
        a.pos[t] = a.slots[t] = -1;
    }
}

size_t pages_scratch_bytes(int) { return (4 + 2 * SERVE_MAX_SEQ) * sizeof(int); }

hipError_t launch_pages_step(const PagesStep& a, hipStream_t s) {
    if (a.t_max <= PAGES_ONE) {
        pages_plan_kernel<true><<<dim3(1), dim3(1024), 0, s>>>(a);
    } else {
        pages_plan_kernel<false><<<dim3(1), dim3(1024), 0, s>>>(a);
        pages_place_kernel<<<dim3((unsigned)((a.t_max + 255) / 256)), dim3(256), 0, s>>>(a);
    }
    return hipGetLastError();
}

// ---------------- penalties, biases and masks on logits ----------------
// For token v of a row, with c its count among the history's tokens at index >= from and seen whether the history (its last
// `last` tokens) holds it:
//   y = x; seen: y = y > 0 ? y / rep : y * rep; y = y - freq * c; c > 0: y = y - pres; y = y + bias; not allowed: -inf
// one rounding a step, in this order. A block takes 4 NU tokens a thread of a row. One table of a word a token in LDS serves
// twice (a table each left half the waves: 27.5 us for the 22 below): first the biases (of a token's the largest index counts),
// which go to the registers of the token's thread, then the history's counts (integer atomics, so the order does not matter);
// then one pass over the logits, which were requested at the start. Every block of a row reads the row's history again, from
// L2. 64 rows of 151936 from x into out, histories of 4096, 100 biases and a mask: 22 us, 3.6 TB/s; one row, bound by the chain
// of its loads: 4.4 us. The rows' choices follow in logits_choose_kernel (4.0 and 1.5 us).
constexpr int LP_T = 512;
constexpr uint32_t LP_SEEN = 0x80000000u;

// NU: tokens a thread / 4. VEC: rows that are 16-byte aligned in x and out, 4 consecutive tokens a load; else a token a load.
template <int NU, bool VEC>
__global__ __launch_bounds__(LP_T) void logits_process_kernel(LogitsProcess a) {
    constexpr int CHUNK = 4 * NU * LP_T;
    __shared__ __align__(16) uint32_t tab[CHUNK];
    __shared__ uint64_t sk[LP_T / 64];
    const int r = blockIdx.y, base = blockIdx.x * CHUNK, tid = threadIdx.x, m = min(CHUNK, a.n - base);
    const float* x = a.x + (uint64_t)r * a.x_stride + base;
    float* out = a.out + (uint64_t)r * a.out_stride + base;
    // this thread's tokens: at(u, e) of the chunk
    auto at = [&](int u, int e) { return VEC ? 4 * (u * LP_T + tid) + e : (4 * u + e) * LP_T + tid; };
    float y[NU][4];
    uint32_t mw[NU][VEC ? 1 : 4];
    const uint32_t* mask = a.mask ? a.mask + (uint64_t)r * a.mask_stride : nullptr;
#pragma unroll
    for (int u = 0; u < NU; u++) {
        if constexpr (VEC) {
            const int i = at(u, 0);
            if (i + 4 <= m) {
                const float4 v = *(const float4*)(x + i);
                y[u][0] = v.x; y[u][1] = v.y; y[u][2] = v.z; y[u][3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) y[u][e] = i + e < m ? x[i + e] : 0.0f;
            }
            mw[u][0] = mask && i < m ? mask[(base + i) >> 5] >> ((base + i) & 31) : 0xFu;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = at(u, e);
                y[u][e] = i < m ? x[i] : 0.0f;
                mw[u][e] = mask && i < m ? mask[(base + i) >> 5] >> ((base + i) & 31) : 1u;
            }
        }
    }
    int h0 = 0, h1 = 0, from = 0, b0 = 0, b1 = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.pen) {
        h1 = (int)min((uint64_t)max(a.hist_len[r], 0), a.hist_stride);
        h0 = a.last > 0 ? max(h1 - a.last, 0) : 0;
        from = a.hist_from ? a.hist_from[r] : 0;
        rep = a.pen[3 * r];
        freq = a.pen[3 * r + 1];
        pres = a.pen[3 * r + 2];
    }
    if (a.bias_start) {
        b0 = min(max(a.bias_start[r], 0), a.n_bias);
        b1 = min(max(a.bias_start[r + 1], b0), a.n_bias);
    }
    const bool pen = h1 > h0, bias = b1 > b0;
    const int* hr = a.hist + (uint64_t)r * a.hist_stride;
    constexpr int HU = 8;  // history loads in flight
    int tok[HU];
    auto history = [&](int i0) {
#pragma unroll
        for (int k = 0; k < HU; k++) tok[k] = i0 + k * LP_T < h1 ? hr[i0 + k * LP_T] : -1;
    };
    if (pen) history(h0 + tid);
    auto clear = [&] {  // this thread's words
#pragma unroll
        for (int u = 0; u < NU; u++) {
            if constexpr (VEC) *(uint4*)&tab[at(u, 0)] = make_uint4(0, 0, 0, 0);
            else
#pragma unroll
                for (int e = 0; e < 4; e++) tab[at(u, e)] = 0;
        }
    };
    auto words = [&](int u, uint32_t (&w)[4]) {
        if constexpr (VEC) *(uint4*)w = *(const uint4*)&tab[at(u, 0)];
        else
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = tab[at(u, e)];
    };
    uint32_t bv[NU][4] = {};
    if (pen || bias) {
        clear();
        __syncthreads();
    }
    if (bias) {
        for (int e = b0 + tid; e < b1; e += LP_T) {
            const unsigned v = (unsigned)a.bias_ids[e] - (unsigned)base;
            if (v < (unsigned)m) atomicMax(&tab[v], (uint32_t)(e + 1));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NU; u++) words(u, bv[u]);
        if (pen) {
            clear();  // (the words that this thread has just read)
            __syncthreads();
        }
    }
    if (pen) {
        for (int i0 = h0 + tid;;) {
#pragma unroll
            for (int k = 0; k < HU; k++) {
                const unsigned v = (unsigned)tok[k] - (unsigned)base;
                if (v < (unsigned)m) {  // (no id below 0: base + m is at most 2^31 - 1)
                    if (i0 + k * LP_T >= from) atomicAdd(&tab[v], 1u);
                    else atomicOr(&tab[v], LP_SEEN);
                }
            }
            i0 += HU * LP_T;
            if (i0 >= h1) break;
            history(i0);
        }
        __syncthreads();
    }
    const bool place = x == out;
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < NU; u++) {
        uint32_t cv[4] = {};
        if (pen) words(u, cv);
        bool changed = !place;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float x0 = y[u][e];
            float v = x0;
            if (cv[e]) v = v > 0.0f ? v / rep : v * rep;
            const uint32_t k = cv[e] & ~LP_SEEN;
            if (k) {
                v = v - freq * (float)k;
                v = v - pres;
            }
            if (bv[u][e]) v = v + a.bias_vals[bv[u][e] - 1];
            const bool ok = VEC ? (mw[u][0] >> e) & 1u : mw[u][VEC ? 0 : e] & 1u;
            if (!ok) v = -INFINITY;
            changed |= __float_as_uint(v) != __float_as_uint(x0);
            y[u][e] = v;
            if (ok && at(u, e) < m) {
                const uint64_t key = amax_key(v, base + at(u, e));
                best = key > best ? key : best;
            }
        }
        if (VEC && at(u, 0) + 4 <= m) {
            if (changed) *(float4*)(out + at(u, 0)) = make_float4(y[u][0], y[u][1], y[u][2], y[u][3]);
        } else if (changed) {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (at(u, e) < m) out[at(u, e)] = y[u][e];
        }
    }
    if (!a.ids) return;
    best = wave_max_u64(best);
    if ((tid & 63) == 0) sk[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < LP_T / 64; w++) best = sk[w] > best ? sk[w] : best;
        a.keys[(uint64_t)r * gridDim.x + blockIdx.x] = best;
    }
}

// A row's choice from its chunks' keys (a key is 0 only where no token of the chunk is allowed), and the history's next token.
__global__ __launch_bounds__(64) void logits_choose_kernel(LogitsProcess a, int parts) {
    const int r = blockIdx.x, lane = threadIdx.x, k = a.append ? a.hist_len[r] : -1;  // (waits with the keys)
    uint64_t best = 0;
    for (int i = lane; i < parts; i += 64) {
        const uint64_t key = a.keys[(uint64_t)r * parts + i];
        best = key > best ? key : best;
    }
    best = wave_max_u64(best);
    if (lane == 0) {
        const int id = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : -1;
        a.ids[r] = id;
        if (id >= 0 && k >= 0 && (uint64_t)k < a.hist_stride) {
            a.hist[(uint64_t)r * a.hist_stride + k] = id;
            a.hist_len[r] = k + 1;
        }
    }
}

static int logits_parts(int n, int nu) { return (int)(((long long)n + 4 * nu * LP_T - 1) / (4 * nu * LP_T)); }
// Tokens a block: 4096, or 2048 where the larger blocks would be fewer than two a CU (64 rows of 151936: 22.0 against 26.2 us; one
// row 5.2 against 4.3).
static int logits_nu(int n, int rows) { return (long long)rows * logits_parts(n, 2) >= 512 ? 2 : 1; }
size_t logits_key_bytes(int n, int rows) { return (size_t)rows * logits_parts(n, logits_nu(n, rows)) * sizeof(uint64_t); }

hipError_t launch_logits_process(const LogitsProcess& a, hipStream_t s) {
    const int nu = logits_nu(a.n, a.rows), parts = logits_parts(a.n, nu);
    const dim3 grid((unsigned)parts, (unsigned)a.rows);
    const bool vec = ((uintptr_t)a.x | (uintptr_t)a.out) % 16 == 0 && (a.rows == 1 || (a.x_stride | a.out_stride) % 4 == 0);
    if (nu == 2 && vec) logits_process_kernel<2, true><<<grid, dim3(LP_T), 0, s>>>(a);
    else if (nu == 2) logits_process_kernel<2, false><<<grid, dim3(LP_T), 0, s>>>(a);
    else if (vec) logits_process_kernel<1, true><<<grid, dim3(LP_T), 0, s>>>(a);
    else logits_process_kernel<1, false><<<grid, dim3(LP_T), 0, s>>>(a);
    if (a.ids) logits_choose_kernel<<<dim3((unsigned)a.rows), dim3(64), 0, s>>>(a, parts);
    return hipGetLastError();
}

}  // namespace strata
