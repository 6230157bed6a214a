// Attention of a ragged batch over a paged f16 KV cache (strata_attn_paged; no counterpart in the reference, whose attention
// serves one sequence with a contiguous cache: src/backend.rs:337-343, 383-410). The batch's t query rows belong to nseq
// sequences, sequence s's to rows q_start[s] .. q_start[s + 1] - 1; row r sits at position pos[r]. A sequence's own key j
// (position P + j, j < len[s]) is cached at row tables[s][j / page] page + j % page; the P keys of the prefix, which every
// sequence sees as its first, at prefix[j / page] page + j % page. Row r, query head h:
//   out = sum_k exp(s_k - M) v_k / (sum_k exp(s_k - M) + exp(sink_h - M)) * sigmoid(gate),  s_k = q . k scale,
// over the keys at positions <= pos[r] (with a window the last `win` of them). A row that sees no key gives 0; a page outside
// 0 .. n_pages - 1 holds no keys.
//
// Three kernels: attn_paged_dec_kernel takes the sequences of few rows (a decode step: bound by their K and V bytes),
// attn_paged_tile_kernel the keys that many rows share (the prefix for all rows, or a prompt chunk's own keys: bound by the
// matrix cores), and attn_paged_merge_kernel joins their softmax sums. Numerics as in attn.hip: q and the softmax weights as
// f16 hi + lo parts, K and V exact in f16, all sums in f32, log2 units.
#include <algorithm>
#include <climits>

#include "attn_dev.h"
#include "serve.h"

namespace strata {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// A call's workspace and split plan (launch_attn_paged).
struct PagedWs {
    int2* map;     // [nseq nkv] first block and pieces of a decode sequence's KV head
    float2* dml;   // [slots][dr] max and sum of a piece's rows
    float* dacc;   // [slots][dr][hd]
    float2* pml;   // [t nh][nsp]: the prefix's splits
    float* pacc;   // [t nh][nsp][hd]
    float2* tml;   // [t nh][nst]: the splits of a long sequence's own keys
    float* tacc;
    int dblocks, nct, dr, nsp, nst;  // decode blocks, their column tiles; rows (tokens x G) up to which a sequence decodes; splits
    bool final_tiles;              // the tile kernel writes out itself (one split, no prefix)
};

// ---------------- sequences ----------------
constexpr int DEC_CHUNK = 128;  // 32 keys a wave
struct SeqInfo {
    int q0, qn;   // query rows
    int len;      // own keys
    int c0, nc;   // the first chunk of DEC_CHUNK own keys that a row sees, and how many (decode sequences)
};
__device__ __forceinline__ int prefix_len(const PagedAttn& a) { return a.prefix_len ? min(max(sload(a.prefix_len), 0), a.max_prefix) : 0; }
// UNI: s is the same in the whole wave (scalar loads, so that what follows from them stays in scalar registers).
template <bool UNI>
__device__ __forceinline__ SeqInfo seq_info(const PagedAttn& a, int s, int G, int dr, int P) {
    auto ld = [](const int* p) { return UNI ? sload(p) : *p; };
    SeqInfo r;
    r.q0 = min(max(ld(a.q_start + s), 0), a.t);
    r.qn = min(max(ld(a.q_start + s + 1), r.q0), a.t) - r.q0;
    r.len = (int)min((long long)max(ld(a.len + s), 0), (long long)a.max_pages << a.page_shift);
    r.c0 = r.nc = 0;
    if (r.qn > 0 && r.qn * G <= dr) {
        if (a.win > 0) {
            int first = INT_MAX;  // (a window hides keys before the first row's)
            for (int i = 0; i < r.qn; i++) first = min(first, ld(a.pos + r.q0 + i));
            r.c0 = (int)(max((long long)first + 1 - a.win - P, 0ll) / DEC_CHUNK);
        }
        r.nc = max((int)(((long long)r.len + DEC_CHUNK - 1) / DEC_CHUNK) - r.c0, 0);
    }
    return r;
}
// Own keys that row r of a sequence sees: lo .. hi (inclusive; none if hi < lo). Keys of the prefix: the same with P for len
// and 0 for P's part of the position.
__device__ __forceinline__ void own_range(const PagedAttn& a, int pos, int len, int P, int& lo, int& hi) {
    hi = (int)min((long long)pos - P, (long long)len - 1);
    lo = a.win > 0 ? (int)max((long long)pos + 1 - a.win - P, 0ll) : 0;
}

// One query row again by a wave in float32 over the keys lo .. hi alone, for rows near a value that is not finite: acc, max and
// sum of its softmax (the max in log2 units). Built for few registers, not for speed.
template <int HD>
__device__ void paged_row_again(const PagedAttn& a, const float* q, int g, const int* table, int lo, int hi, float (&acc)[HD / 64],
                                float& m, float& l) {
    const int lane = threadIdx.x & 63;
    const uint64_t kvd = (uint64_t)a.nkv * HD;
    auto row = [&](int j) {  // the key's cache row, or -1
        const int pg = table[j >> a.page_shift];
        return pg >= 0 && pg < a.n_pages ? ((int64_t)pg << a.page_shift) + (j & ((1 << a.page_shift) - 1)) : (int64_t)-1;
    };
    auto score = [&](int j) {
        const int64_t r = row(j);
        if (r < 0) return -INFINITY;
        float s = 0.0f;
#pragma unroll 1
        for (int c = 0; c < HD; c += 8) {
            const h8 kv = *(const h8*)(a.kc + (uint64_t)r * kvd + g * HD + c);
#pragma unroll
            for (int e = 0; e < 8; e++) s += q[c + e] * (float)kv[e];
        }
        return s * (a.scale * LOG2E);
    };
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int c = 0; c < HD / 64; c++) acc[c] = 0.0f;
#pragma unroll 1
    for (int j = lo + lane; j <= hi; j += 64) m = fmaxf(m, score(j));
    m = wave_max64(m);
    if (m == -INFINITY) return;
#pragma unroll 1
    for (int k0 = lo; k0 <= hi; k0 += 64) {
        const float p = k0 + lane <= hi ? exp2_hw(score(k0 + lane) - m) : 0.0f;
        l += p;
#pragma unroll 1
        for (int e = 0; e < 64 && k0 + e <= hi; e++) {
            const float pe = __shfl(p, e, 64);
            const int64_t r = row(k0 + e);
            if (r < 0) continue;
#pragma unroll
            for (int c = 0; c < HD / 64; c++) acc[c] += pe * h2f(a.vc[(uint64_t)r * kvd + g * HD + lane + 64 * c]);
        }
    }
    l = wave_sum64(l);
}

// The exclusive prefix sums of f(s), s < n <= SERVE_MAX_SEQ, into cum by a block of 256 threads; the total (and the largest
// f(s)) to every thread. cum[n - 1] + f(n - 1) is the total.
template <typename F>
__device__ __forceinline__ int scan_seqs(int n, F&& f, int* cum, int* ws, int& largest) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per = (n + 255) / 256;
    int sum = 0, big = 0;
    for (int i = 0; i < per; i++) {
        const int s = tid * per + i;
        if (s < n) {
            const int v = f(s);
            cum[s] = sum;
            sum += v;
            big = max(big, v);
        }
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(inc, o, 64);
        if (lane >= o) inc += u;
        big = max(big, __shfl_xor(big, o, 64));
    }
    if (lane == 63) {
        ws[wave] = inc;
        ws[4 + wave] = big;
    }
    __syncthreads();
    int base = inc - sum, total = 0;
    largest = 0;
#pragma unroll
    for (int w = 0; w < 4; w++) {
        if (w < wave) base += ws[w];
        total += ws[w];
        largest = max(largest, ws[4 + w]);
    }
    for (int i = 0; i < per; i++)
        if (tid * per + i < n) cum[tid * per + i] += base;
    __syncthreads();
    return total;
}
// The last i < n with cum[i] <= v.
__device__ __forceinline__ int seq_of(const int* cum, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cum[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The scaled hi and lo f16 parts of 8 query values.
__device__ __forceinline__ void split_q8(const f4& x0, const f4& x1, float up, h8& hi, h8& lo) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float x = (e < 4 ? x0[e & 3] : x1[e & 3]) * up;
        hi[e] = (_Float16)x;
        lo[e] = (_Float16)(x - (float)hi[e]);
    }
}

// The A fragment of V^T for 16 dims a 16-lane group from V rows as they are in memory: each group of 16 lanes reads 4 rows x
// 16 columns (lane i: row i / 4, columns 4 (i % 4) ..) and lane i gets column i of the 4 rows.
__device__ __forceinline__ h4 read_tr(const uint16_t* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p));
}

// ---------------- few rows a sequence ----------------
// The work is the list of all (sequence, KV head, chunk of DEC_CHUNK own keys), chunk fastest; a block takes an equal run of
// it, so contexts of any lengths load the CUs evenly. A run covers pieces of one or more (sequence, KV head) pairs; block b's
// piece of pair i leaves its softmax sums at slot b + i (along the list either b or i goes up by one, so slots are distinct).
// The block that holds a pair's first chunk notes which blocks follow.
// Inside a piece, wave w takes keys 32 w .. 32 w + 31 of each chunk with its own online softmax for all rows (16 NT columns:
// token c / G, head c % G), on f16 MFMA with f32 accuracy:
//   S^T (2 tiles of 16 keys x 16 columns) = K Q^T (v_mfma_f32_16x16x32_f16; A: the key rows, read straight from memory in the
//   fragments' layout, 16 rows x 64 bytes a load; B: q's hi and lo parts);
//   O^T (16 dims x 16 columns, DT tiles) += V^T P^T (K = 32; B: the lane's own 8 weights, hi and lo; A: V's rows through the
//   wave's LDS, read transposed).
// The next chunk's V is requested when this one's has gone to LDS, its K when the scores are done: both fly during the softmax
// and the V products without more registers. The four waves meet in LDS at the piece's end.
template <int HD>
struct PagedDec {
    static constexpr int VP = HD + 16;             // halves a V row in LDS (32 bytes on: the transposed reads' 16 rows spread)
    static constexpr int WAVE = 32 * VP * 2;
    static constexpr int MERGE = DEC_WAVES * (HD * 16 + 32) * 4;
    static constexpr int BYTES = DEC_WAVES * WAVE > MERGE ? DEC_WAVES * WAVE : MERGE;
};
template <int HD, int NT>
__global__ __launch_bounds__(256, NT == 1 ? 2 : 1) void attn_paged_dec_kernel(PagedAttn a, PagedWs w) {
    using L = PagedDec<HD>;
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    constexpr int KS = HD / 32, DT = HD / 16, LPR = HD / 8, RPI = 64 / LPR, NV = 32 / RPI;  // lanes a V row, rows a load, loads
    __shared__ __align__(16) uint8_t lds[L::BYTES];
    __shared__ int ws[8];
    __shared__ SeqInfo sq;
    __shared__ int sb[2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    const int G = a.nh / a.nkv, P = prefix_len(a), b = blockIdx.x;
    // this block's run of the list: the thread that holds the sequence of its start says which it is
    int W0, W1, share;
    {
        const int per = (a.nseq + 255) / 256;
        SeqInfo mine{};
        int sum = 0, big = 0;
        for (int i = 0; i < per; i++)
            if (tid * per + i < a.nseq) {
                mine = seq_info<false>(a, tid * per + i, G, w.dr, P);
                sum += mine.nc;
                big = max(big, mine.nc);
            }
        int at = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(at, o, 64);
            if (lane >= o) at += u;
            big = max(big, __shfl_xor(big, o, 64));
        }
        if (lane == 63) {
            ws[wave] = at;
            ws[4 + wave] = big;
        }
        __syncthreads();
        int total = 0;
        at -= sum;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            if (v < wave) at += ws[v];
            total += ws[v];
            big = max(big, ws[4 + v]);
        }
        total *= a.nkv;
        // (at most 128 pieces a pair: the merge's work)
        share = max((total + (int)gridDim.x - 1) / (int)gridDim.x, (big + 127) / 128);
        W0 = (int)min((long long)b * share, (long long)total);
        W1 = (int)min((long long)W0 + share, (long long)total);
        if (W0 >= W1) return;
        if (W0 >= at * a.nkv && W0 < (at + sum) * a.nkv)
            for (int i = 0; i < per && tid * per + i < a.nseq; i++) {
                const SeqInfo q = per == 1 ? mine : seq_info<false>(a, tid * per + i, G, w.dr, P);
                if (W0 >= at * a.nkv && W0 < (at + q.nc) * a.nkv) {
                    sq = q;
                    sb[0] = tid * per + i;
                    sb[1] = at * a.nkv;
                }
                at += q.nc;
            }
        __syncthreads();
    }
    auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    SeqInfo q{uni(sq.q0), uni(sq.qn), uni(sq.len), uni(sq.c0), uni(sq.nc)};
    int s = uni(sb[0]), base = uni(sb[1]);
    W0 = uni(W0), W1 = uni(W1), share = uni(share);
    uint16_t* vs = (uint16_t*)(lds + wave * L::WAVE);
    const uint32_t kvd2 = 2 * a.nkv * HD;
    const int vr = lane / LPR, vcol = 8 * (lane % LPR);
    const uint32_t vcol2 = 2 * vcol;
    for (int at = W0; at < W1;) {
        while (at - base >= q.nc * a.nkv) {  // the next sequence that has work
            base += q.nc * a.nkv;
            if (++s >= a.nseq) return;
            q = seq_info<true>(a, s, G, w.dr, P);
        }
        const int g = (at - base) / q.nc, f = (at - base) % q.nc, n = min(q.nc - f, W1 - at);
        const int pair = s * a.nkv + g;
        if (f == 0 && tid == 0) w.map[pair] = make_int2(b, (at + q.nc - 1) / share - b + 1);
        at += n;
        const int* table = a.tables + (uint64_t)s * a.max_pages;
        const uint64_t kg = (uint64_t)(a.kc + g * HD), vg = (uint64_t)(a.vc + g * HD);
        // The wave's two groups of 16 keys of chunk c (each in one page): their cache rows; ok: bit t where group t has keys. A
        // group without keys reads the other's rows.
        struct Rows {
            uint64_t at[2];  // bytes into either cache
            int last[2], ok;
        };
        auto pages = [&](int c, int (&pg)[2]) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; t++) pg[t] = sload(table + (min(DEC_CHUNK * c + 32 * wave + 16 * t, q.len - 1) >> a.page_shift));
        };
        auto rows = [&](int c, const int (&pg)[2]) __attribute__((always_inline)) {
            Rows r;
            r.ok = 0;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int k0 = DEC_CHUNK * c + 32 * wave + 16 * t;
                r.at[t] = (((uint64_t)(uint32_t)pg[t] << a.page_shift) + (k0 & ((1 << a.page_shift) - 1))) * kvd2;
                r.last[t] = min(q.len - 1 - k0, 15);
                r.ok |= (r.last[t] >= 0 && (uint32_t)pg[t] < (uint32_t)a.n_pages) << t;
            }
            if (r.ok == 1) r.at[1] = r.at[0], r.last[1] = r.last[0];
            if (r.ok == 2) r.at[0] = r.at[1], r.last[0] = r.last[1];
            return r;
        };
        // (a group's rows: a scalar base and a lane's 32-bit offset)
        v4u kf[2][KS], vb[NV];
        auto load_v = [&](const Rows& r) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < NV; u++) {
                const int t = u * RPI / 16, k = (u * RPI) % 16 + vr;  // key k of group t
                const uint32_t off = __umul24(min(k, r.last[t]), kvd2) + vcol2;
                vb[u] = *gptr<v4u>(vg + r.at[t] + off);
            }
        };
        auto load_k = [&](const Rows& r) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t off = __umul24(min(l16, r.last[t]), kvd2) + 16 * lg;
#pragma unroll
                for (int k = 0; k < KS; k++) kf[t][k] = *gptr<v4u>(kg + r.at[t] + off + 64 * k);
            }
        };
        const int c0 = q.c0 + f, c1 = c0 + n;
        int pg[2];
        pages(c0, pg);
        Rows cur = rows(c0, pg);
        if (cur.ok) {
            load_v(cur);
            load_k(cur);
        }
        if (n > 1) pages(c0 + 1, pg);
        // the rows' queries and the keys they see
        h8 qh[NT][KS], ql[NT][KS];
        float usc[NT], m[NT], l[NT];
        int lo[NT], hi[NT];
        f4 o[NT][DT];
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const int c = 16 * u + l16, tok = c / G, h = g * G + c % G;
            const bool live = tok < q.qn;
            f4 qv[2 * KS];
            float mx = 0.0f;
            const float* qr = a.q + ((uint64_t)(q.q0 + (live ? tok : 0)) * a.nh + h) * HD;
            const int pos = a.pos[q.q0 + (live ? tok : 0)];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    qv[2 * k + e] = *(const f4*)(qr + 32 * k + 8 * lg + 4 * e);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        qv[2 * k + e][i] = live ? qv[2 * k + e][i] : 0.0f;
                        mx = fmaxf(mx, fabsf(qv[2 * k + e][i]));
                    }
                }
            lo[u] = 1;
            hi[u] = 0;
            if (live) own_range(a, pos, q.len, P, lo[u], hi[u]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            int ex = 0;
            if (mx > 0.0f) (void)frexpf(mx, &ex);
            const float up = ldexpf(1.0f, 14 - ex);
            usc[u] = ldexpf(a.scale * LOG2E, ex - 14);
#pragma unroll
            for (int k = 0; k < KS; k++) split_q8(qv[2 * k], qv[2 * k + 1], up, qh[u][k], ql[u][k]);
            m[u] = -INFINITY;
            l[u] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[u][d] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
        }
        for (int c = c0; c < c1; c++) {
            const Rows r = cur;
            if (r.ok) {
#pragma unroll
                for (int u = 0; u < NV; u++) *(v4u*)&vs[(u * RPI + vr) * L::VP + vcol] = vb[u];
            }
            __builtin_amdgcn_wave_barrier();
            const bool more = c + 1 < c1;
            if (more) {
                cur = rows(c + 1, pg);
                if (cur.ok) load_v(cur);
            }
            f4 sv[NT][2];
            if (r.ok) {
#pragma unroll
                for (int u = 0; u < NT; u++)
#pragma unroll
                    for (int t = 0; t < 2; t++) sv[u][t] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KS; k++)
#pragma unroll
                    for (int u = 0; u < NT; u++)
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            const h8 kv = __builtin_bit_cast(h8, kf[t][k]);
                            sv[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, qh[u][k], sv[u][t], 0, 0, 0);
                            sv[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv, ql[u][k], sv[u][t], 0, 0, 0);
                        }
            }
            if (more) {
                if (cur.ok) load_k(cur);
                if (c + 2 < c1) pages(c + 2, pg);
            }
            if (!r.ok) continue;
            const int k0 = DEC_CHUNK * c + 32 * wave;
            h8 ph[NT], pl[NT];
#pragma unroll
            for (int u = 0; u < NT; u++) {
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = k0 + 16 * t + 4 * lg + i;
                        if (j < lo[u] || j > hi[u] || !((r.ok >> t) & 1)) sv[u][t][i] = -INFINITY;
                        mx = fmaxf(mx, sv[u][t][i]);
                    }
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float mxs = mx * usc[u];  // (a positive factor keeps the order)
                if (__ballot(mxs > m[u] + 1.0f)) {  // (m follows the maximum when a weight would pass 2, column by column)
                    const float mnew = mxs > m[u] + 1.0f ? mxs : m[u], alpha = m[u] == -INFINITY ? 0.0f : exp2_hw(m[u] - mnew);
                    l[u] *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[u][d] *= alpha;
                    m[u] = mnew;
                }
                const float mref = m[u] == -INFINITY ? 0.0f : m[u];
                float p[8];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        p[4 * t + i] = exp2_hw(__builtin_fmaf(sv[u][t][i], usc[u], -mref));
                        l[u] += p[4 * t + i];
                    }
                split_w8(p, ph[u], pl[u]);
            }
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const uint16_t* vp = &vs[(4 * lg + (l16 >> 2)) * L::VP + 16 * d + 4 * (l16 & 3)];
                const h4 v0 = read_tr(vp), v1 = read_tr(vp + 16 * L::VP);
                const h8 vf = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    o[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, ph[u], o[u][d], 0, 0, 0);
                    o[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[u], o[u][d], 0, 0, 0);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int u = 0; u < NT; u++) {
            l[u] += __shfl_xor(l[u], 16, 64);
            l[u] += __shfl_xor(l[u], 32, 64);
        }
        // the waves' sums meet in LDS, 16 rows at a time
        float* ow = (float*)lds;
        float* mw = ow + DEC_WAVES * HD * 16;
        float* lw = mw + DEC_WAVES * 16;
#pragma unroll
        for (int u = 0; u < NT; u++) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) ow[(wave * HD + 16 * d + 4 * lg + i) * 16 + l16] = o[u][d][i];
            if (lg == 0) {
                mw[wave * 16 + l16] = m[u];
                lw[wave * 16 + l16] = l[u];
            }
            __syncthreads();
            constexpr int DPT = HD / 16;
            const int rr = tid >> 4, dd0 = (tid & 15) * DPT, c = 16 * u + rr;
            const bool live = c < q.qn * G;
            const uint64_t at_row = (uint64_t)(b + pair) * w.dr + c;
            float M = -INFINITY, e[DEC_WAVES], sum = 0.0f, acc[DPT], nf = 0.0f;
#pragma unroll
            for (int v = 0; v < DEC_WAVES; v++) M = fmaxf(M, mw[v * 16 + rr]);
#pragma unroll
            for (int v = 0; v < DEC_WAVES; v++) {
                e[v] = mw[v * 16 + rr] == -INFINITY ? 0.0f : exp2_hw(mw[v * 16 + rr] - M);
                sum += lw[v * 16 + rr] * e[v];
            }
#pragma unroll
            for (int d = 0; d < DPT; d++) {
                acc[d] = 0.0f;
#pragma unroll
                for (int v = 0; v < DEC_WAVES; v++) acc[d] += ow[(v * HD + dd0 + d) * 16 + rr] * e[v];
                nf = __builtin_fmaf(acc[d], 0.0f, nf);
            }
            if (live) {
#pragma unroll
                for (int d = 0; d < DPT; d++) w.dacc[at_row * HD + dd0 + d] = acc[d] * (1.0f / PF_SCALE);
                if ((tid & 15) == 0) w.dml[at_row] = make_float2(M, sum);
            }
            // A row with finite scores whose sums are not may owe it to a key that it does not see (0 times a value that is not
            // finite): again, over its own keys alone
            for (uint64_t bad = __ballot(live && nf != 0.0f && sum - sum == 0.0f); bad;) {
                const int ln = __builtin_ctzll(bad), rb = (64 * wave + ln) >> 4, cb = 16 * u + rb, tok = cb / G;
                bad &= ~(0xFFFFull << (ln & 48));
                int klo, khi;
                own_range(a, a.pos[q.q0 + tok], q.len, P, klo, khi);
                float ac[HD / 64], mm, ll;
                paged_row_again<HD>(a, a.q + ((uint64_t)(q.q0 + tok) * a.nh + g * G + cb % G) * HD, g, table, max(klo, DEC_CHUNK * c0),
                                    min(khi, DEC_CHUNK * c1 - 1), ac, mm, ll);
                const uint64_t r = (uint64_t)(b + pair) * w.dr + cb;
#pragma unroll
                for (int d = 0; d < HD / 64; d++) w.dacc[r * HD + lane + 64 * d] = ac[d];
                if (lane == 0) w.dml[r] = make_float2(mm, ll);
            }
        }
        __syncthreads();  // the tiles are rewritten by the next piece
    }
}

// ---------------- many rows over the same keys ----------------
// A block of 4 waves takes 128 query rows of one KV head (128 / G tokens x G heads, 32 rows a wave) over a split of the keys
// that they see, in tiles of 64 keys as attn_prefill_kernel of attn.hip does, on v_mfma_f32_32x32x16_f16. PRE: tiles of the
// call's rows whatever their sequence, over the prefix's keys: K and V of the prefix are read once a tile of 128 / G tokens
// rather than once a token. Else: tiles of the rows of each sequence that is too long for the decode kernel, over its own
// keys. Blocks are numbered so that the tiles over the same keys run on one XCD (its L2 holds a split's K and V).
template <int HD, bool PRE>
__global__ __launch_bounds__(256, 2) void attn_paged_tile_kernel(PagedAttn a, PagedWs w, int tiles) {
    using L = PfLayout<HD>;
    constexpr int KS = HD / 16, DT = HD / 32, ND = HD / 8, BK = 64;
    constexpr int KB = BK * L::KP * 2, VB = HD * L::VP * 2;
    static_assert(KB + VB >= SERVE_MAX_SEQ * 4, "the prefix sums use the tiles' LDS");
    __shared__ __align__(16) uint8_t lds[KB + VB];
    __shared__ int ws[8];
    uint16_t* ks = (uint16_t*)lds;
    uint16_t* vs = (uint16_t*)(lds + KB);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
    const int G = a.nh / a.nkv, gs = 31 - __builtin_clz(G), TT = 128 >> gs, P = prefix_len(a);
    const int ns = PRE ? w.nsp : w.nst, nc = a.nkv * ns;
    // block x: combination (KV head, split) c on XCD c % 8, tile tt
    const int x = blockIdx.x, c = (x & 7) + 8 * ((x >> 3) / tiles);
    int tt = (x >> 3) % tiles;
    if (c >= nc) return;
    const int g = c % a.nkv, split = c / a.nkv;
    // the tile's first row, its tokens, the keys' table and number
    int t0, nt, len;
    const int* table;
    if constexpr (PRE) {
        t0 = tt * TT;
        nt = min(TT, min(max(a.q_start[a.nseq], 0), a.t) - t0);
        len = P;
        table = a.prefix;
        if (nt <= 0) return;
    } else {
        int* cum = (int*)lds;
        int largest;
        const int total = scan_seqs(a.nseq, [&](int i) {
            const SeqInfo q = seq_info<false>(a, i, G, w.dr, P);
            return q.qn * G > w.dr ? (q.qn + TT - 1) / TT : 0;
        }, cum, ws, largest);
        tt = total - 1 - tt;  // (a sequence's last, longest tiles first)
        if (tt < 0) return;
        const int s = seq_of(cum, a.nseq, tt);
        const int j = tt - cum[s];
        __syncthreads();
        const SeqInfo q = seq_info<true>(a, __builtin_amdgcn_readfirstlane(s), G, w.dr, P);
        t0 = q.q0 + j * TT;
        nt = min(TT, q.qn - j * TT);
        len = q.len;
        table = a.tables + (uint64_t)s * a.max_pages;
    }
    // this lane's row (a query column), the keys it sees, and those that the wave's and the block's rows see
    const int r = 32 * wave + l32, tok = r >> gs, h = g * G + (r & (G - 1));
    const bool live = tok < nt;
    int lo = INT_MAX, hi = -1;
    if (live) own_range(a, a.pos[t0 + tok], len, PRE ? 0 : P, lo, hi);
    if (hi < lo) hi = -1, lo = INT_MAX;
    int wlo = lo, whi = hi, maxlo = hi < 0 ? -1 : lo, minhi = live ? hi : INT_MAX;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        wlo = min(wlo, __shfl_xor(wlo, o, 64));
        whi = max(whi, __shfl_xor(whi, o, 64));
        maxlo = max(maxlo, __shfl_xor(maxlo, o, 64));
        minhi = min(minhi, __shfl_xor(minhi, o, 64));
    }
    wlo = __builtin_amdgcn_readfirstlane(wlo);
    whi = __builtin_amdgcn_readfirstlane(whi);
    maxlo = __builtin_amdgcn_readfirstlane(maxlo);
    minhi = __builtin_amdgcn_readfirstlane(minhi);
    if (lane == 0) {
        ws[wave] = wlo;
        ws[4 + wave] = whi;
    }
    __syncthreads();
    const int blo = min(min(ws[0], ws[1]), min(ws[2], ws[3])), bhi = max(max(ws[4], ws[5]), max(ws[6], ws[7]));
    // the split's tiles of 64 keys: kb .. ke - 1
    const int kt0 = bhi < 0 ? 0 : blo / BK, kt1 = bhi < 0 ? 0 : bhi / BK + 1, per = (kt1 - kt0 + ns - 1) / ns;
    const int kb = min(kt0 + split * per, kt1), ke = min(kb + per, kt1);
    h8 qh[KS], ql[KS];
    float usc;
    const float* qr = a.q + ((uint64_t)(t0 + (live ? tok : 0)) * a.nh + h) * HD;
    {
        f4 v[2 * KS];
        float mx = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                v[2 * k + e] = *(const f4*)(qr + 16 * k + 8 * hf + 4 * e);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[2 * k + e][i] = live ? v[2 * k + e][i] : 0.0f;
                    mx = fmaxf(mx, fabsf(v[2 * k + e][i]));
                }
            }
        mx = max_half(mx);
        int ex = 0;
        if (mx > 0.0f) (void)frexpf(mx, &ex);
        const float up = ldexpf(1.0f, 14 - ex);
        usc = ldexpf(a.scale * LOG2E, ex - 14);
#pragma unroll
        for (int k = 0; k < KS; k++) split_q8(v[2 * k], v[2 * k + 1], up, qh[k], ql[k]);
    }
    f16v o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    constexpr int NPK = BK * ND / 256, NPV = BK / 2 * ND / 256;
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    v4u kr[NPK], vr[NPV][2];
    const int kk = tid / ND, kcol = 8 * (tid % ND);
    const int vk = 2 * (((tid >> 3) & 7) + 8 * (wave / (ND / 8))), vcol = 8 * ((tid & 7) + 8 * (wave % (ND / 8)));
    constexpr int KST = 256 / ND, VST = 64 / (ND / 8);
    const uint64_t kvd2 = 2 * (uint64_t)a.nkv * HD;
    const uint32_t kc2 = 2 * (g * HD + kcol), vc2 = 2 * (g * HD + vcol);
    // Pages of a tile's four groups of 16 keys (a group lies in one page); past the last key its group's, a page outside the
    // pool is read as page 0 and its keys hidden.
    auto pages = [&](int k0, int (&pg)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; u++) pg[u] = sload(table + (min(k0 + 16 * u, (len - 1) & ~15) >> a.page_shift));
    };
    auto fetch = [&](int k0, const int (&pg)[4]) __attribute__((always_inline)) {
        const int lim = len - 1 - k0;  // (keys past the last read its row)
        auto at = [&](int i, int grp, uint32_t col) __attribute__((always_inline)) {  // cache bytes of key min(i, lim), in group grp
            const int g16 = min(16 * grp, lim & ~15), p = grp == 0 ? pg[0] : grp == 1 ? pg[1] : grp == 2 ? pg[2] : pg[3];
            const uint64_t row = ((uint64_t)(p >= 0 && p < a.n_pages ? p : 0) << a.page_shift) + ((k0 + g16) & ((1 << a.page_shift) - 1));
            return row * kvd2 + (__umul24((uint32_t)(min(i, lim) - g16), (uint32_t)kvd2) + col);
        };
#pragma unroll
        for (int u = 0; u < NPK; u++) kr[u] = *gptr<v4u>((uint64_t)a.kc + at(KST * u + kk, ND == 16 ? u : 2 * u + (wave >> 1), kc2));
#pragma unroll
        for (int u = 0; u < NPV; u++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                vr[u][e] = *gptr<v4u>((uint64_t)a.vc + at(VST * u + e + vk, ND == 16 ? 2 * u + (wave >> 1) : wave, vc2));
    };
    int pg[4], pn[4];
    if (kb < ke) {
        pages(BK * kb, pg);
        fetch(BK * kb, pg);
        pages(min(BK * (kb + 1), (len - 1) & ~63), pn);
    }
    for (int kt = kb; kt < ke; kt++) {
        const int k0 = BK * kt;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < NPK; u++) *(v4u*)&ks[(kk + KST * u) * L::KP + kcol] = kr[u];
#pragma unroll
        for (int u = 0; u < NPV; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t va = vr[u][0][e], vb = vr[u][1][e];
                *(uint32_t*)&vs[(vcol + 2 * e) * L::VP + vk + VST * u] = __builtin_amdgcn_perm(vb, va, 0x05040100u);
                *(uint32_t*)&vs[(vcol + 2 * e + 1) * L::VP + vk + VST * u] = __builtin_amdgcn_perm(vb, va, 0x07060302u);
            }
        __syncthreads();
        int hole = 0;  // groups without a page
#pragma unroll
        for (int u = 0; u < 4; u++) hole |= (pg[u] < 0 || pg[u] >= a.n_pages) << u;
        if (kt + 1 < ke) {
#pragma unroll
            for (int u = 0; u < 4; u++) pg[u] = pn[u];
            fetch(k0 + BK, pg);
            pages(min(k0 + 2 * BK, (len - 1) & ~63), pn);
        }
        if (k0 > whi || k0 + BK - 1 < wlo) continue;
        f16v s[2], z;
#pragma unroll
        for (int i = 0; i < 16; i++) z[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const h8 k0f = *(const h8*)&ks[l32 * L::KP + 16 * k + 8 * hf], k1f = *(const h8*)&ks[(32 + l32) * L::KP + 16 * k + 8 * hf];
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0f, qh[k], k ? s[0] : z, 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1f, qh[k], k ? s[1] : z, 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0f, ql[k], s[0], 0, 0, 0);
            s[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1f, ql[k], s[1], 0, 0, 0);
        }
        if (k0 + BK - 1 > minhi || k0 < maxlo || hole) {
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int kp = 32 * mt + 8 * (i >> 2) + 4 * hf + (i & 3);
                    if (k0 + kp > hi || k0 + kp < lo || ((hole >> (kp >> 4)) & 1)) s[mt][i] = -INFINITY;
                }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, s[mt][i]);
        mx = max_half(mx);
        const float mxs = mx * usc;
        if (__ballot(mxs > m + 1.0f)) {  // (m follows the maximum when a weight would pass 2, column by column)
            const float mnew = mxs > m + 1.0f ? mxs : m, alpha = m == -INFINITY ? 0.0f : exp2_hw(m - mnew);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= alpha;
            m = mnew;
        }
        const float mref = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p = exp2_hw(__builtin_fmaf(s[mt][i], usc, -mref));
                s[mt][i] = p;
                sum += p;
            }
        l += sum;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) p[e] = s[mt][8 * u + e];
                h8 ph, pl;
                split_w8(p, ph, pl);
                h8 vf[DT];
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    const uint16_t* vp = &vs[(32 * d + l32) * L::VP + 32 * mt + 16 * u + 4 * hf];
                    const uint2 a0 = *(const uint2*)vp, a1 = *(const uint2*)(vp + 8);
                    vf[d] = __builtin_bit_cast(h8, make_uint4(a0.x, a0.y, a1.x, a1.y));
                }
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], ph, o[d], 0, 0, 0);
#pragma unroll
                for (int d = 0; d < DT; d++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], pl, o[d], 0, 0, 0);
            }
    }
    l += __shfl_xor(l, 32, 64);
    // rows with finite scores whose sums are not finite: again, over the keys that they see alone
    float nf = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) nf = __builtin_fmaf(o[d][i], 0.0f, nf);
    const uint64_t nfb = __ballot(nf != 0.0f && l - l == 0.0f && live);
    uint32_t again = (uint32_t)nfb | (uint32_t)(nfb >> 32);
    const uint64_t row = (uint64_t)(t0 + tok) * a.nh + h;
    const bool fin = !PRE && w.final_tiles;
    float2* ml = PRE ? w.pml : w.tml;
    float* accp = PRE ? w.pacc : w.tacc;
    // the scale that turns sums into an output (final: normalized by the sum and the sink), and its gate
    auto norm = [&](int hh, float mm, float ll) {
        const float sk = a.sink ? a.sink[hh] * LOG2E : -INFINITY, M = fmaxf(mm, sk);
        const float sc = mm == -INFINITY ? 0.0f : exp2_hw(mm - M);
        const float den = ll * sc + (sk == -INFINITY ? 0.0f : exp2_hw(sk - M));
        return den == 0.0f ? 0.0f : sc / den;  // (not a number where a score is)
    };
    if (live && !((again >> l32) & 1)) {
        const float f = (fin ? norm(h, m, l) : 1.0f) * (1.0f / PF_SCALE);
        float* dst = fin ? a.out + row * HD : accp + (row * ns + split) * HD;
        const float* gate = fin && a.qg ? a.qg + row * 2 * HD + HD : nullptr;
        if (fin || m != -INFINITY) {
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int col = 32 * d + 8 * j + 4 * hf;
                    float4 v = make_float4(o[d][4 * j] * f, o[d][4 * j + 1] * f, o[d][4 * j + 2] * f, o[d][4 * j + 3] * f);
                    if (gate) {
                        v.x *= sigmoid_f(gate[col]); v.y *= sigmoid_f(gate[col + 1]);
                        v.z *= sigmoid_f(gate[col + 2]); v.w *= sigmoid_f(gate[col + 3]);
                    }
                    *(float4*)(dst + col) = v;
                }
        }
        if (!fin && hf == 0) ml[row * ns + split] = make_float2(m, l);
    }
    for (; again; again &= again - 1) {
        const int rb = 32 * wave + __builtin_ctz(again), hb = g * G + (rb & (G - 1)), tb = t0 + (rb >> gs);
        const uint64_t rowb = (uint64_t)tb * a.nh + hb;
        int klo, khi;
        own_range(a, a.pos[tb], len, PRE ? 0 : P, klo, khi);
        float ac[HD / 64], mm, ll;
        paged_row_again<HD>(a, a.q + rowb * HD, g, table, max(klo, BK * kb), min(khi, BK * ke - 1), ac, mm, ll);
        const float f = fin ? norm(hb, mm, ll) : 1.0f;
        float* dst = fin ? a.out + rowb * HD : accp + (rowb * ns + split) * HD;
#pragma unroll
        for (int d = 0; d < HD / 64; d++) {
            const int col = lane + 64 * d;
            const float v = ac[d] * f;
            dst[col] = fin && a.qg ? v * sigmoid_f(a.qg[rowb * 2 * HD + HD + col]) : v;
        }
        if (!fin && lane == 0) ml[rowb * ns + split] = make_float2(mm, ll);
    }
}

// ---------------- the join ----------------
// The sequence of row r < q_start[nseq]: the last s with q_start[s] <= r, by a wave in rounds of 64 loads (q_start does not
// decrease; nseq <= 4096).
__device__ __forceinline__ int row_seq(const PagedAttn& a, int r) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.nseq;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const uint64_t le = __ballot(i < n && a.q_start[lo + i] <= r);
        const int k = le ? 63 - __builtin_clzll(le) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

// Row r, query head h from its partial sums: out = sum_i acc_i 2^(m_i - M) / (sum_i l_i 2^(m_i - M) + 2^(sink - M)). Block
// (x, heads y) of MW waves a head: wave v of a head takes partials v, v + MW, .. (the prefix's splits, then the own keys'
// pieces or splits), their maxima a lane each, then the weighted rows with the loads of 8 in flight. DEC: x is row x % per of
// sequence x / per, the sequences of the decode kernel; else x is a row, those of the tile kernel.
template <int HD, int MW, bool DEC>
__global__ __launch_bounds__(256) void attn_paged_merge_kernel(PagedAttn a, PagedWs w, int per) {
    constexpr int DL = HD / 64, HPB = 4 / MW;
    __shared__ float sm[HPB][MW], sl[HPB][MW], so[HPB][MW][HD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int G = a.nh / a.nkv, P = prefix_len(a);
    int s, r;
    if constexpr (DEC) {
        s = blockIdx.x / per;
    } else {
        r = blockIdx.x;
        if (r >= a.q_start[a.nseq]) return;
        s = __builtin_amdgcn_readfirstlane(row_seq(a, r));
    }
    const SeqInfo q = seq_info<true>(a, s, G, w.dr, P);
    if constexpr (DEC) r = q.q0 + blockIdx.x % per;
    const bool dec = q.qn * G <= w.dr;
    if (r < q.q0 || r >= q.q0 + q.qn || dec != DEC) return;
    const int hi = wave / MW, v = wave % MW;
    for (int h = blockIdx.y * HPB + hi; h < a.nh; h += gridDim.y * HPB) {
        const int g = h / G;
        const uint64_t row = (uint64_t)r * a.nh + h;
        const int np = P > 0 ? w.nsp : 0;
        int no = 0;
        uint64_t first = 0, step = 1;  // partial i >= np: row first + (i - np) step of (ml, acc)
        const float2* oml = DEC ? w.dml : w.tml;
        const float* oacc = DEC ? w.dacc : w.tacc;
        if constexpr (DEC) {
            if (q.nc > 0) {
                const int2 mp = w.map[s * a.nkv + g];
                no = mp.y;
                first = (uint64_t)(mp.x + s * a.nkv + g) * w.dr + (r - q.q0) * G + h % G;
                step = w.dr;
            }
        } else {
            no = w.nst;
            first = row * w.nst;
        }
        const int n = np + no;
        float M = -INFINITY, L = 0.0f, acc[DL];
#pragma unroll
        for (int d = 0; d < DL; d++) acc[d] = 0.0f;
        for (int i0 = v; i0 < n; i0 += 64 * MW) {
            const int i = i0 + MW * lane;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (i < n) ml = i < np ? w.pml[row * np + i] : oml[first + (uint64_t)(i - np) * step];
            const float mnew = fmaxf(M, wave_max64(ml.x));
            const float e = ml.x == -INFINITY ? 0.0f : exp2_hw(ml.x - mnew), f = M == -INFINITY ? 0.0f : exp2_hw(M - mnew);
            L = L * f + wave_sum64(ml.y * e);
#pragma unroll
            for (int d = 0; d < DL; d++) acc[d] *= f;
            M = mnew;
            const uint64_t some = __ballot(ml.x != -INFINITY);
            const int cnt = some ? 64 - __builtin_clzll(some) : 0;
            for (int j0 = 0; j0 < cnt; j0 += 8) {
                float av[8][DL];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int ii = i0 + MW * (j0 + j);
                    const bool has = j0 + j < 64 && ((some >> ((j0 + j) & 63)) & 1);
                    const float* src = ii < np ? w.pacc + (row * np + ii) * HD : oacc + (first + (uint64_t)(ii - np) * step) * HD;
#pragma unroll
                    for (int d = 0; d < DL; d++) av[j][d] = has ? src[DL * lane + d] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float es = __shfl(e, (j0 + j) & 63, 64);
#pragma unroll
                    for (int d = 0; d < DL; d++) acc[d] += av[j][d] * es;
                }
            }
        }
        if constexpr (MW > 1) {
            if (lane == 0) {
                sm[hi][v] = M;
                sl[hi][v] = L;
            }
#pragma unroll
            for (int d = 0; d < DL; d++) so[hi][v][DL * lane + d] = acc[d];
            __syncthreads();
            float Mb = -INFINITY;
#pragma unroll
            for (int u = 0; u < MW; u++) Mb = fmaxf(Mb, sm[hi][u]);
            L = 0.0f;
#pragma unroll
            for (int d = 0; d < DL; d++) acc[d] = 0.0f;
#pragma unroll
            for (int u = 0; u < MW; u++) {
                const float f = sm[hi][u] == -INFINITY ? 0.0f : exp2_hw(sm[hi][u] - Mb);
                L += sl[hi][u] * f;
#pragma unroll
                for (int d = 0; d < DL; d++) acc[d] += so[hi][u][DL * lane + d] * f;
            }
            M = Mb;
            __syncthreads();
        }
        if (MW == 1 || v == 0) {
            const float sk = a.sink ? a.sink[h] * LOG2E : -INFINITY, Ms = fmaxf(M, sk);
            const float sc = M == -INFINITY ? 0.0f : exp2_hw(M - Ms);
            const float den = L * sc + (sk == -INFINITY ? 0.0f : exp2_hw(sk - Ms)), f = den == 0.0f ? 0.0f : sc / den;
#pragma unroll
            for (int d = 0; d < DL; d++) {
                float x = acc[d] * f;
                if (a.qg) x *= sigmoid_f(a.qg[row * 2 * HD + HD + DL * lane + d]);
                a.out[row * HD + DL * lane + d] = x;
            }
        }
    }
}

// ---------------- launches ----------------
static int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// The split plan and the workspace's layout from `at`; the end of the layout in *end.
static PagedWs plan(const PagedAttn& a, uint8_t* at, size_t* end) {
    PagedWs w{};
    const int G = a.nh / a.nkv;
    const long long rows = (long long)a.t * G;
    // a sequence decodes up to 16 rows (one column tile), up to 32 where the longest has no more
    const long long most_rows = (long long)a.max_q * G;
    w.nct = most_rows > 16 && most_rows <= 32 ? 2 : 1;
    w.dr = (int)std::min<long long>(16 * w.nct, most_rows);
    const long long most = (long long)a.nseq * a.nkv * (((long long)a.max_pages << a.page_shift) / DEC_CHUNK + 1);
    w.dblocks = (int)std::min<long long>(most, w.nct == 1 ? 512 : 256);  // the blocks that run at once
    // splits of the tile kernels: enough blocks for two a CU
    auto splits = [&](long long tiles, long long keys) {
        const long long blocks = tiles * a.nkv, want = div_up(512, std::max(blocks, 1ll));
        return (int)std::max<long long>(1, std::min<long long>({want, (keys + 127) / 128, 64}));
    };
    w.nsp = splits(div_up(rows, 128), a.max_prefix);
    const bool tiles = most_rows > w.dr;
    w.nst = splits(div_up(rows, 128), (long long)a.max_pages << a.page_shift);
    w.final_tiles = w.nst == 1 && !a.max_prefix;
    size_t o = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = at + o;
        o += (bytes + 255) & ~(size_t)255;
        return (void*)p;
    };
    const size_t slots = (size_t)w.dblocks + (size_t)a.nseq * a.nkv, out_rows = (size_t)a.t * a.nh;
    w.map = (int2*)take((size_t)a.nseq * a.nkv * sizeof(int2));
    w.dml = (float2*)take(slots * w.dr * sizeof(float2));
    w.dacc = (float*)take(slots * w.dr * a.hd * sizeof(float));
    if (a.max_prefix) {
        w.pml = (float2*)take(out_rows * w.nsp * sizeof(float2));
        w.pacc = (float*)take(out_rows * w.nsp * a.hd * sizeof(float));
    }
    if (tiles && !w.final_tiles) {
        w.tml = (float2*)take(out_rows * w.nst * sizeof(float2));
        w.tacc = (float*)take(out_rows * w.nst * a.hd * sizeof(float));
    }
    *end = o;
    return w;
}

size_t paged_attn_ws_bytes(const PagedAttn& a) {
    size_t n;
    plan(a, nullptr, &n);
    return n;
}

template <int HD>
static void launch_t(const PagedAttn& a, const PagedWs& w, hipStream_t s) {
    const int G = a.nh / a.nkv, TT = 128 / G;
    auto grid = [&](int tiles, int ns) { return dim3((unsigned)(8 * div_up((long long)a.nkv * ns, 8) * (long long)tiles)); };
    if (a.max_prefix) {
        const int tiles = div_up(a.t, TT);
        attn_paged_tile_kernel<HD, true><<<grid(tiles, w.nsp), dim3(256), 0, s>>>(a, w, tiles);
    }
    if ((long long)a.max_q * G > w.dr) {
        // tiles of the long sequences: each has more than dr / G rows
        const int tiles = (int)std::min<long long>((long long)a.t / TT + std::min<long long>(a.nseq, a.t / (w.dr / G + 1)), INT_MAX);
        attn_paged_tile_kernel<HD, false><<<grid(std::max(tiles, 1), w.nst), dim3(256), 0, s>>>(a, w, std::max(tiles, 1));
    }
    if (w.nct == 2)
        attn_paged_dec_kernel<HD, 2><<<dim3((unsigned)w.dblocks), dim3(256), 0, s>>>(a, w);
    else
        attn_paged_dec_kernel<HD, 1><<<dim3((unsigned)w.dblocks), dim3(256), 0, s>>>(a, w);
    const int per = w.dr / G;
    attn_paged_merge_kernel<HD, 4, true><<<dim3((unsigned)(a.nseq * per), (unsigned)a.nh), dim3(256), 0, s>>>(a, w, per);
    if (w.tml) attn_paged_merge_kernel<HD, 1, false><<<dim3((unsigned)a.t, (unsigned)((a.nh + 3) / 4)), dim3(256), 0, s>>>(a, w, 0);
}

hipError_t launch_attn_paged(const PagedAttn& a, hipStream_t s) {
    size_t n;
    const PagedWs w = plan(a, (uint8_t*)a.ws, &n);
    if (a.hd == 128) launch_t<128>(a, w, s);
    else launch_t<64>(a, w, s);
    return hipGetLastError();
}

}  // namespace strata
