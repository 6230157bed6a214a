// Attention of a ragged batch over a paged f16 KV cache (strata_attn_paged; no counterpart in the reference, whose attention
// serves one sequence with a contiguous cache: src/backend.rs:337-343, 383-410). The batch's t query rows belong to nseq
// sequences, sequence s's to rows q_start[s] .. q_start[s + 1] - 1; row r sits at position pos[r]. A sequence's own key j
// (position P + j, j < len[s]) is cached at row tables[s][j / page] page + j % page; the P keys of the prefix, which every
// sequence sees as its first, at prefix[j / page] page + j % page. Row r, query head h:
//   out = sum_k exp(s_k - M) v_k / (sum_k exp(s_k - M) + exp(sink_h - M)) * sigmoid(gate),  s_k = q . k scale,
// over the keys at positions <= pos[r] (with a window the last `win` of them). A row that sees no key gives 0; a page outside
// 0 .. n_pages - 1 holds no keys.
//
// One launch does the work in blocks of three kinds (attn_paged_kernel), a second one joins its partial sums:
//   dec_block     the own keys of sequences of few rows (a decode step): bound by their K and V bytes;
//   prefix_block  the prefix for those sequences' rows, whatever their sequence: K and V read once a tile of rows;
//   tile_block    the prefix and own keys of sequences of many rows (prompt chunks), from attn_paged_plan_kernel's list of their
//                 tiles: bound by the matrix cores and the softmax's vector instructions, which add up.
// The prefix and the own keys are bound by different things and run beside each other (in launches of their own: 64 sequences over a
// prefix of 16000 71 us a call for 59, 24 of 4 tokens over one of 6001 35 for 22). Beside tiles, whose blocks come first and fill the
// CUs, they start as those end (2500 tokens of three chunks over a prefix of 16000 1265 us, with 60 decoding sequences 1293). Numerics as in attn.hip: q and the softmax weights as f16 hi
// + lo parts (2^-22 of a value), K and V exact in f16, all sums in f32, log2 units.
#include <algorithm>
#include <climits>

#include "attn_dev.h"
#include "serve.h"

namespace strata {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// A call's workspace and split plan (plan() below).
struct PagedWs {
    int2* map;     // decode sequences: [nseq nkv] first block and pieces of a KV head; direct: [dblocks] the (sequence, KV head)
                   // that begins in a block and goes on past it, and its pieces (0: none)
    float2* dml;   // [slots][dr] max and sum of a piece's rows
    float* dacc;   // [slots][dr][hd]
    float2* pml;   // [prows nh][nsp]: the prefix's splits, of the rows of decode sequences (without a plan: of all rows)
    float* pacc;   // [prows nh][nsp][hd]
    int* plan;     // long sequences (null: none): PlanHead, then a Tile each
    int* drows;    // with a plan and a prefix: the rows of decode sequences, one sequence's behind the other's
    int* dstart;   // and where sequence s's begin in that list
    int4* cut;     // [tblocks] KV head and tile that block b's run cuts, and the last block of its pieces (below 0: none)
    float2* tml;   // [2 tblocks][128]: the pieces of tiles that more than one block computes
    float* tacc;   // [2 tblocks][128][hd]
    int direct;    // a (sequence, KV head) that one block holds is finished there, and the join takes those that a block cuts
    int dblocks, nct, dr, nsp, prows, tblocks;  // decode blocks, their column tiles; rows (tokens x G) up to which a sequence decodes
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

// The keys of a sequence as one list: virtual key v < 64 np lies in the prefix (key v, none from P on), v >= 64 np is own key
// v - 64 np, np = ceil(P / 64) tiles of 64.
struct Keys {
    const int* prefix;
    const int* own;
    int P, np, len;
};
// Virtual keys that a row at position pos sees: lo .. hi (none: hi = -1, lo past it).
__device__ __forceinline__ void row_range(const PagedAttn& a, const Keys& k, int pos, int& lo, int& hi) {
    const long long own = min((long long)pos - k.P, (long long)k.len - 1);
    const int first = a.win > 0 ? (int)max((long long)pos + 1 - a.win, 0ll) : 0;
    hi = own >= 0 ? 64 * k.np + (int)own : min(pos, k.P - 1);
    lo = first < k.P ? first : 64 * k.np + (first - k.P);
    if (hi < lo) hi = -1, lo = INT_MAX;
}

// One query row again by a wave in float32 over the virtual keys lo .. hi alone, for rows near a value that is not finite: acc,
// max and sum of its softmax (the max in log2 units). Built for few registers, not for speed.
template <int HD>
__device__ void paged_row_again(const PagedAttn& a, const Keys& ks, const float* q, int g, int lo, int hi, float (&acc)[HD / 64],
                                float& m, float& l) {
    const int lane = threadIdx.x & 63;
    const uint64_t kvd = (uint64_t)a.nkv * HD;
    auto row = [&](int v) {  // the key's cache row, or -1
        const bool pre = v < 64 * ks.np;
        const int j = pre ? v : v - 64 * ks.np;
        if (pre && j >= ks.P) return (int64_t)-1;
        const int pg = (pre ? ks.prefix : ks.own)[j >> a.page_shift];
        return pg >= 0 && pg < a.n_pages ? ((int64_t)pg << a.page_shift) + (j & ((1 << a.page_shift) - 1)) : (int64_t)-1;
    };
    auto score = [&](int v) {
        const int64_t r = row(v);
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
    for (int v = lo + lane; v <= hi; v += 64) m = fmaxf(m, score(v));
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

// The factor that turns a row's sums into its output: over the sum and the sink (0 for a row without keys, not a number where a
// score is not).
__device__ __forceinline__ float out_factor(const PagedAttn& a, int h, float m, float l) {
    const float sk = a.sink ? a.sink[h] * LOG2E : -INFINITY, M = fmaxf(m, sk);
    const float sc = m == -INFINITY ? 0.0f : exp2_hw(m - M);
    const float den = l * sc + (sk == -INFINITY ? 0.0f : exp2_hw(sk - M));
    return den == 0.0f ? 0.0f : sc / den;
}

// ---------------- few rows a sequence ----------------
// The work is the list of all (sequence, KV head, chunk of DEC_CHUNK own keys), chunk fastest; a block takes an equal run of
// it, so contexts of any lengths load the CUs evenly. A run covers pieces of one or more (sequence, KV head) pairs; block b's
// piece of pair i leaves its softmax sums at slot b + i (along the list either b or i goes up by one, so slots are distinct).
// The block that holds a pair's first chunk notes which blocks follow; with many pairs (DIRECT) one that holds a whole pair
// finishes its rows.
// Inside a piece, wave w takes keys 32 w .. 32 w + 31 of each chunk with its own online softmax for all rows (16 NT columns:
// token c / G, head c % G), on f16 MFMA with f32 accuracy:
//   S^T (2 tiles of 16 keys x 16 columns) = K Q^T (v_mfma_f32_16x16x32_f16; A: the key rows, read straight from memory in the
//   fragments' layout, 16 rows x 64 bytes a load; B: q's hi and lo parts);
//   O^T (16 dims x 16 columns, DT tiles) += V^T P^T (K = 32; B: the lane's own 8 weights, hi and lo; A: V's rows through the
//   wave's LDS, read transposed).
// The next chunk's V (the next piece's, at the end of one) is requested when this one's has gone to LDS, its K when the scores are
// done: both fly during the softmax and the V products without more registers. The four waves meet in LDS at the piece's end,
// while the next one's queries arrive.
// 64 sequences of 100 to 24000 keys (32 heads of 128 over 4, 539 MB): 112 us, 4.8 TB/s, a copy's rate; 1000 of 300 138 us, 4.5 TB/s; one of 550 keys 9 us, a chain
// of the run's search (2), the loads (2.5), the products (1.2) and the waves' meeting (2).
template <int HD>
struct PagedDec {
    static constexpr int VP = HD + 16;             // halves a V row in LDS (32 bytes on: the transposed reads' 16 rows spread)
    static constexpr int WAVE = 32 * VP * 2;
    static constexpr int MERGE = DEC_WAVES * (HD * 17 + 32) * 4;
    static constexpr int BYTES = DEC_WAVES * WAVE > MERGE ? DEC_WAVES * WAVE : MERGE;
};
template <int HD, int NT, bool DIRECT>
__device__ __forceinline__ void dec_block(const PagedAttn& a, const PagedWs& w, int b, uint8_t* lds) {
    using L = PagedDec<HD>;
    typedef unsigned v4u __attribute__((ext_vector_type(4)));
    constexpr int KS = HD / 32, DT = HD / 16, LPR = HD / 8, RPI = 64 / LPR, NV = 32 / RPI;  // lanes a V row, rows a load, loads
    __shared__ int ws[8];
    __shared__ SeqInfo sq;
    __shared__ int sb[2];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
    const int G = a.nh / a.nkv, P = prefix_len(a);
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
        // (at most 128 pieces a pair, the join's work: 131072 keys over one KV head 29 us, up to 64 40; up to 256, joined by two waves, 38 for 33)
        share = max((total + w.dblocks - 1) / w.dblocks, (big + 127) / 128);
        W0 = (int)min((long long)b * share, (long long)total);
        W1 = (int)min((long long)W0 + share, (long long)total);
        if (DIRECT && tid == 0) w.map[b] = make_int2(0, 0);
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
    const uint64_t kb = (uint64_t)a.kc, vb0 = (uint64_t)a.vc;
    // a piece: chunks c0 .. c1 - 1 of sequence s and KV head g
    struct Piece {
        SeqInfo q;
        int s, g, c0, c1, head;  // head: if it holds the pair's first chunk, the blocks that share the pair (else 0)
    };
    int at = W0;
    auto next_piece = [&](Piece& p) __attribute__((always_inline)) {
        if (at >= W1) return false;
        while (at - base >= q.nc * a.nkv) {  // the next sequence that has work
            base += q.nc * a.nkv;
            if (++s >= a.nseq) return false;
            q = seq_info<true>(a, s, G, w.dr, P);
        }
        const int g = (at - base) / q.nc, f = (at - base) % q.nc, n = min(q.nc - f, W1 - at);
        p = Piece{q, s, g, q.c0 + f, q.c0 + f + n, f == 0 ? (at + q.nc - 1) / share - b + 1 : 0};
        at += n;
        return true;
    };
    // The wave's two groups of 16 keys of chunk c (each in one page): their cache rows; ok: bit t where group t has keys. A
    // group without keys reads the other's rows.
    struct Rows {
        uint64_t at[2];  // bytes into either cache
        int last[2], ok;
    };
    auto pages = [&](const Piece& p, int c, int (&pg)[2]) __attribute__((always_inline)) {
        const int* table = a.tables + (uint64_t)p.s * a.max_pages;
#pragma unroll
        for (int t = 0; t < 2; t++) pg[t] = sload(table + (min(DEC_CHUNK * c + 32 * wave + 16 * t, p.q.len - 1) >> a.page_shift));
    };
    auto rows = [&](const Piece& p, int c, const int (&pg)[2]) __attribute__((always_inline)) {
        Rows r;
        r.ok = 0;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int k0 = DEC_CHUNK * c + 32 * wave + 16 * t;
            r.at[t] = (((uint64_t)(uint32_t)pg[t] << a.page_shift) + (k0 & ((1 << a.page_shift) - 1))) * kvd2 + 2 * HD * p.g;
            r.last[t] = min(p.q.len - 1 - k0, 15);
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
            vb[u] = *gptr<v4u>(vb0 + r.at[t] + off);
        }
    };
    auto load_k = [&](const Rows& r) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t off = __umul24(min(l16, r.last[t]), kvd2) + 16 * lg;
#pragma unroll
            for (int k = 0; k < KS; k++) kf[t][k] = *gptr<v4u>(kb + r.at[t] + off + 64 * k);
        }
    };
    // a piece's queries and positions, row 16 u + l16
    f4 qv[NT][2 * KS];
    int qpos[NT];
    auto load_q = [&](const Piece& p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const int c = 16 * u + l16, tok = c / G < p.q.qn ? c / G : 0, h = p.g * G + c % G;
            const float* qr = a.q + ((uint64_t)(p.q.q0 + tok) * a.nh + h) * HD;
            qpos[u] = a.pos[p.q.q0 + tok];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int e = 0; e < 2; e++) qv[u][2 * k + e] = *(const f4*)(qr + 32 * k + 8 * lg + 4 * e);
        }
    };
    Piece pc, nx;
    if (!next_piece(pc)) return;
    int pg[2];
    pages(pc, pc.c0, pg);
    Rows cur = rows(pc, pc.c0, pg);
    if (cur.ok) {
        load_v(cur);
        load_k(cur);
    }
    load_q(pc);
    for (bool more_pieces = true; more_pieces; pc = nx) {
        const int c0 = pc.c0, c1 = pc.c1, pair = pc.s * a.nkv + pc.g;
        const bool whole = DIRECT && pc.head == 1;  // no other partial sums: this block writes the rows
        if (pc.head && !whole && tid == 0) w.map[DIRECT ? b : pair] = make_int2(DIRECT ? pair : b, pc.head);
        more_pieces = next_piece(nx);
        if (c0 + 1 < c1) pages(pc, c0 + 1, pg);
        else if (more_pieces) pages(nx, nx.c0, pg);
        // the rows' queries and the keys they see
        h8 qh[NT][KS], ql[NT][KS];
        float usc[NT], m[NT], l[NT];
        int lo[NT], hi[NT];
        f4 o[NT][DT];
#pragma unroll
        for (int u = 0; u < NT; u++) {
            const bool live = (16 * u + l16) / G < pc.q.qn;
            float mx = 0.0f;
#pragma unroll
            for (int k = 0; k < 2 * KS; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    qv[u][k][i] = live ? qv[u][k][i] : 0.0f;
                    mx = fmaxf(mx, fabsf(qv[u][k][i]));
                }
            lo[u] = 1;
            hi[u] = 0;
            if (live) own_range(a, qpos[u], pc.q.len, P, lo[u], hi[u]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            float up;
            query_scale(mx, a.scale, up, usc[u]);
            usc[u] = fmaxf(usc[u], USC_MIN);
#pragma unroll
            for (int k = 0; k < KS; k++) split_q8(qv[u][2 * k], qv[u][2 * k + 1], up, qh[u][k], ql[u][k]);
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
            const bool same = c + 1 < c1, more = same || more_pieces;  // the next chunk: of this piece, or the next one's first
            if (more) {
                cur = same ? rows(pc, c + 1, pg) : rows(nx, nx.c0, pg);
                if (cur.ok) load_v(cur);
            }
            f4 sv[NT][2];
            if (r.ok) {
#pragma unroll
                for (int u = 0; u < NT; u++)
#pragma unroll
                    for (int t = 0; t < 2; t++) sv[u][t] = (f4){0.0f, 0.0f, 0.0f, 0.0f};
                // (the lo parts first: their sums are small, so only the hi parts' steps round at the score's size)
#pragma unroll
                for (int k = 0; k < 2 * KS; k++)
#pragma unroll
                    for (int u = 0; u < NT; u++)
#pragma unroll
                        for (int t = 0; t < 2; t++)
                            sv[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, kf[t][k % KS]), k < KS ? ql[u][k % KS] : qh[u][k % KS],
                                                                              sv[u][t], 0, 0, 0);
            }
            if (more) {
                if (cur.ok) load_k(cur);
                if (c + 2 < c1) pages(pc, c + 2, pg);
                else if (same && more_pieces) pages(nx, nx.c0, pg);
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
        if (more_pieces) load_q(nx);
#pragma unroll
        for (int u = 0; u < NT; u++) {
            l[u] += __shfl_xor(l[u], 16, 64);
            l[u] += __shfl_xor(l[u], 32, 64);
        }
        // the waves' sums meet in LDS, 16 rows at a time (a dim's 16 rows 17 words apart: the reads of 4 rows x 64 dims hit all
        // banks once)
        float* ow = (float*)lds;
        float* mw = ow + DEC_WAVES * HD * 17;
        float* lw = mw + DEC_WAVES * 16;
#pragma unroll
        for (int u = 0; u < NT; u++) {
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) ow[(wave * HD + 16 * d + 4 * lg + i) * 17 + l16] = o[u][d][i];
            if (lg == 0) {
                mw[wave * 16 + l16] = m[u];
                lw[wave * 16 + l16] = l[u];
            }
            __syncthreads();
            constexpr int DPT = HD / 16;
            const int rr = tid >> 4, d4 = 4 * (tid & 15), c = 16 * u + rr;  // dims d4 .. d4 + 3 of each 64
            const bool live = c < pc.q.qn * G;
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
                for (int v = 0; v < DEC_WAVES; v++) acc[d] += ow[(v * HD + (d & ~3) * 16 + d4 + (d & 3)) * 17 + rr] * e[v];
                nf = __builtin_fmaf(acc[d], 0.0f, nf);
            }
            if (live) {
                const int h = pc.g * G + c % G;
                const uint64_t row = (uint64_t)(pc.q.q0 + c / G) * a.nh + h;
                const float f = (whole ? out_factor(a, h, M, sum) : 1.0f) * (1.0f / PF_SCALE);
                float* dst = whole ? a.out + row * HD : w.dacc + at_row * HD;
#pragma unroll
                for (int d = 0; d < DPT; d += 4) {
                    float4 x = make_float4(acc[d] * f, acc[d + 1] * f, acc[d + 2] * f, acc[d + 3] * f);
                    if (whole && a.qg) {
                        const float4 gt = *(const float4*)(a.qg + row * 2 * HD + HD + 16 * d + d4);
                        x.x *= sigmoid_f(gt.x); x.y *= sigmoid_f(gt.y); x.z *= sigmoid_f(gt.z); x.w *= sigmoid_f(gt.w);
                    }
                    *(float4*)(dst + 16 * d + d4) = x;
                }
                if (!whole && (tid & 15) == 0) w.dml[at_row] = make_float2(M, sum);
            }
            // A row with finite scores whose sums are not may owe it to a key that it does not see (0 times a value that is not
            // finite): again, over its own keys alone
            for (uint64_t bad = __ballot(live && nf != 0.0f && sum - sum == 0.0f); bad;) {
                const int ln = __builtin_ctzll(bad), rb = (64 * wave + ln) >> 4, cb = 16 * u + rb, tok = cb / G;
                bad &= ~(0xFFFFull << (ln & 48));
                int klo, khi;
                own_range(a, a.pos[pc.q.q0 + tok], pc.q.len, P, klo, khi);
                float ac[HD / 64], mm, ll;
                paged_row_again<HD>(a, Keys{nullptr, a.tables + (uint64_t)pc.s * a.max_pages, 0, 0, pc.q.len},
                                    a.q + ((uint64_t)(pc.q.q0 + tok) * a.nh + pc.g * G + cb % G) * HD, pc.g, max(klo, DEC_CHUNK * c0),
                                    min(khi, DEC_CHUNK * c1 - 1), ac, mm, ll);
                const uint64_t r = (uint64_t)(b + pair) * w.dr + cb, row = (uint64_t)(pc.q.q0 + tok) * a.nh + pc.g * G + cb % G;
                const float f = whole ? out_factor(a, pc.g * G + cb % G, mm, ll) : 1.0f;
                float* dst = whole ? a.out + row * HD : w.dacc + r * HD;
#pragma unroll
                for (int d = 0; d < HD / 64; d++) {
                    const int col = lane + 64 * d;
                    dst[col] = whole && a.qg ? ac[d] * f * sigmoid_f(a.qg[row * 2 * HD + HD + col]) : ac[d] * f;
                }
                if (!whole && lane == 0) w.dml[r] = make_float2(mm, ll);
            }
        }
        __syncthreads();  // the tiles are rewritten by the next piece
    }
}

// ---------------- many rows over the same keys ----------------
// A block of 4 waves takes 128 query rows of one KV head (128 / G tokens x G heads, 32 rows a wave) over tiles of 64 keys, on
// v_mfma_f32_32x32x16_f16 as attn_prefill_kernel of attn.hip does: S^T (32 keys x 32 rows, two sub-tiles) = K Q^T hi and lo,
// an online softmax a column, O^T (32 dims x 32 rows) += V^T P^T hi and lo with V's rows read transposed from LDS.
// The scores of a tile are computed beside the softmax of the one before, whose vector instructions fill the matrix
// instructions' shadow; a tile costs one barrier. K and V go from memory straight to LDS (no registers hold them), two buffers
// each: while tile t's V and tile t + 1's K are used, the next of each land.
// 1024 rows over 16384 keys (32 heads of 128 over 4): 500 us, 533 TFLOP/s of the formula's operations, twice that on the matrix
// cores for the hi and lo parts. A wave's tile costs its 64 matrix instructions and about 270 vector ones and 33 exps one after
// the other (each part left out alone saves its own share); without loads or over one page it takes as long.
// Rows in LDS are HD halves apart without padding; 16-byte chunk c of row r sits at c ^ swz(r), which spreads both the score
// fragments' reads (a chunk of 32 rows) and the transposed reads (4 chunks of 8 rows) over all banks.
template <int HD>
struct PagedTile {
    static constexpr int BK = 64, ROW = 2 * HD, KB = BK * ROW, BUF = 2 * KB;  // bytes a row, of K's (or V's) tile, of both
    __device__ static __forceinline__ int swz(int r) { return HD == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3); }
};

// The softmax sums of a lane's row (column l32 of wave `wave`) over key tiles kb .. ke - 1; o and l times TILE_SCALE.
constexpr float TILE_SCALE = 16384.0f;
template <int HD>
struct TileSums {
    f16v o[HD / 32];
    float m, l;
};
// live: the lane has a row; qr: its query; pos: its position.
template <int HD>
__device__ __forceinline__ void tile_run(const PagedAttn& a, const Keys& keys, uint8_t* lds, int g, int kb, int ke, bool live, const float* qr,
                                         int pos, TileSums<HD>& r) {
    using L = PagedTile<HD>;
    constexpr int KS = HD / 16, DT = HD / 32, BK = 64, LPR = HD / 8, RPI = 64 / LPR, NJ = 16 / RPI;  // lanes a row, rows a load, loads
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
    const uint32_t kvd2 = 2 * a.nkv * HD;
    const uint64_t kg = (uint64_t)(a.kc + g * HD), vg = (uint64_t)(a.vc + g * HD);
    // Pages of a tile's four groups of 16 keys (a group lies in one page); past the last key its group's; a page outside the
    // pool is read as page 0 and its keys hidden.
    auto pages = [&](int kt, int (&pg)[4]) __attribute__((always_inline)) {
        kt = min(kt, ke - 1);
        const bool pre = kt < keys.np;
        const int k0 = BK * (pre ? kt : kt - keys.np), n = pre ? keys.P : keys.len;
        const int* table = pre ? keys.prefix : keys.own;
#pragma unroll
        for (int u = 0; u < 4; u++) pg[u] = sload(table + (min(k0 + 16 * u, (n - 1) & ~15) >> a.page_shift));
    };
    auto holes = [&](const int (&pg)[4]) __attribute__((always_inline)) {
        int h = 0;
#pragma unroll
        for (int u = 0; u < 4; u++) h |= ((uint32_t)pg[u] >= (uint32_t)a.n_pages) << u;
        return h;
    };
    // A tile's rows of K (or V) into LDS: this wave its 16-key group `wave`, load j rows RPI j .. of it; past the last key its
    // row. Rows RPI j further on, a chunk's place differs by the bits of swz(RPI j) alone (row addresses are multiples of 64 bytes).
    auto load = [&](int kt, const int (&pg)[4], uint64_t src, uint8_t* dst) __attribute__((always_inline)) {
        const bool pre = kt < keys.np;
        const int k0 = BK * (pre ? kt : kt - keys.np), lim = (pre ? keys.P : keys.len) - 1 - k0, g16 = min(16 * wave, lim & ~15);
        const int p = wave == 0 ? pg[0] : wave == 1 ? pg[1] : wave == 2 ? pg[2] : pg[3];
        const uint64_t at = src + (((uint64_t)((uint32_t)p < (uint32_t)a.n_pages ? p : 0) << a.page_shift) + ((k0 + g16) & ((1 << a.page_shift) - 1))) * kvd2;
        uint32_t ln = lane;
        asm volatile("" : "+v"(ln));
        const uint32_t c16 = 16 * ((ln % LPR) ^ L::swz(ln / LPR));
        if (lim >= BK - 1) {
            const uint32_t off = __umul24(ln / LPR, kvd2) + c16;
#pragma unroll
            for (int j = 0; j < NJ; j++) load_lds16_so(at + RPI * j * kvd2, off ^ (16 * L::swz(RPI * j)), dst + (16 * wave + RPI * j) * L::ROW);
        } else {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int row = RPI * j + ln / LPR;  // of the group
                load_lds16_so(at, __umul24(min(16 * wave + row, lim) - g16, kvd2) + (c16 ^ (16 * L::swz(RPI * j))), dst + (16 * wave + RPI * j) * L::ROW);
            }
        }
    };
    // (the query's loads before the tiles', which the loop's first wait covers)
    f4 qv[2 * KS];
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int e = 0; e < 2; e++) qv[2 * k + e] = *(const f4*)(qr + 16 * k + 8 * hf + 4 * e);
    uint8_t *kbuf = lds, *vbuf = lds + L::BUF;
    int pg[4], hole = 0, hole1 = 0;  // pg: of the next tile to request; holes of the tiles whose scores are next, and after it
    if (kb < ke) {
        pages(kb, pg);
        load(kb, pg, kg, kbuf);
        load(kb, pg, vg, vbuf);
        hole = holes(pg);
        if (kb + 1 < ke) {
            pages(kb + 1, pg);
            load(kb + 1, pg, kg, kbuf + L::KB);
            hole1 = holes(pg);
        }
    }
    int lo, hi;  // the virtual keys that the lane's row sees
    row_range(a, keys, pos, lo, hi);
    h8 qh[KS], ql[KS];
    float usc;
    {
        float mx = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * KS; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                qv[k][i] = live ? qv[k][i] : 0.0f;
                mx = fmaxf(mx, fabsf(qv[k][i]));
            }
        mx = max_half(mx);
        float up;
        query_scale(mx, a.scale, up, usc);
        usc = fmaxf(usc, USC_MIN);
#pragma unroll
        for (int k = 0; k < KS; k++) split_q8(qv[2 * k], qv[2 * k + 1], up, qh[k], ql[k]);
    }
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) r.o[d][i] = 0.0f;
    float m = -INFINITY, l = 0.0f, one = 1.0f;
    asm("" : "+s"(one));  // (a product with it stays a mixed-precision multiply-add)
    // this lane's addresses: K's fragment of sub-tile 0, k-step 0, V's transposed reads of dim tile 0 (opaque in each tile, so
    // that the exclusive-ors of the other steps' are not kept in registers)
    auto opaque = [](uint32_t v) __attribute__((always_inline)) {
        asm volatile("" : "+v"(v));
        return v;
    };
    const uint32_t kf0 = l32 * L::ROW + 16 * (hf ^ L::swz(l32));
    const int i16 = lane & 15;
    const uint32_t vf0 = (4 * hf + (i16 >> 2)) * L::ROW + 16 * ((((lane & 16) >> 3) + ((i16 & 3) >> 1)) ^ L::swz(4 * hf + (i16 >> 2))) + 8 * (i16 & 1);
    // all of the wave's rows see keys maxlo .. minhi (both halves of a wave hold the same rows)
    int maxlo = live && hi >= 0 ? lo : -1, minhi = live ? hi : INT_MAX;
    static_for<0, 5>([&](auto S) {
        constexpr int st = decltype(S)::value;
        maxlo = max(maxlo, xl32<st>(maxlo));
        minhi = min(minhi, xl32<st>(minhi));
    });
    maxlo = __builtin_amdgcn_readfirstlane(maxlo);
    minhi = __builtin_amdgcn_readfirstlane(minhi);
    f16v s[2];
    float mx = -INFINITY;
    auto scores = [&](int buf, f16v (&x)[2]) __attribute__((always_inline)) {
        const uint8_t* kt = kbuf + buf * L::KB;
        const uint32_t kf0o = opaque(kf0);
        f16v z;
#pragma unroll
        for (int i = 0; i < 16; i++) z[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const h8 f0 = *(const h8*)(kt + (kf0o ^ (32 * k))), f1 = *(const h8*)(kt + 32 * L::ROW + (kf0o ^ (32 * k)));
            x[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f0, qh[k], k ? x[0] : z, 0, 0, 0);
            x[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1, qh[k], k ? x[1] : z, 0, 0, 0);
            x[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f0, ql[k], x[0], 0, 0, 0);
            x[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f1, ql[k], x[1], 0, 0, 0);
        }
    };
    // keys that a row does not see (where a tile has such), and the column's largest score
    auto mask = [&](int kt, int hole, f16v (&x)[2]) __attribute__((always_inline)) {
        const int k0 = BK * kt;
        const bool tail = kt < keys.np && k0 + BK > keys.P;  // (the prefix's last tile, where it is not whole)
        if (k0 + BK - 1 > minhi || k0 < maxlo || hole || tail) {
            const int top = tail ? min(hi, keys.P - 1) : hi;
            // (one unsigned comparison a key: 0 <= key - lo <= top - lo)
            const uint32_t from = k0 + 4 * hf - (top < lo ? INT_MAX : lo), span = top < lo ? 0 : top - lo;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int i = 0; i < 16; i++) x[mt][i] = from + (32 * mt + 8 * (i >> 2) + (i & 3)) <= span ? x[mt][i] : -INFINITY;
            if (hole)
#pragma unroll
                for (int v = 0; v < 32; v++)
                    if ((hole >> (v >> 3)) & 1) x[v >> 4][v & 15] = -INFINITY;
        }
    };
    auto largest = [&](const f16v (&x)[2]) __attribute__((always_inline)) {
        float v = -INFINITY;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int i = 0; i < 16; i++) v = fmaxf(v, x[mt][i]);
        return max_half(v);
    };
    // one tile: its softmax beside the next one's scores, then its V products; NEXT: there is a next one
    auto tile = [&](int kt, auto NEXT) __attribute__((always_inline)) {
        constexpr bool next = decltype(NEXT)::value;
        const int buf = (kt - kb) & 1;
        if constexpr (next) {
            // (pg: tile kt + 1's pages; its V, and the K of the one after)
            load(kt + 1, pg, vg, vbuf + (buf ^ 1) * L::KB);
            if (kt + 2 < ke) {
                pages(kt + 2, pg);
                load(kt + 2, pg, kg, kbuf + buf * L::KB);
            }
        }
        const float mxs = mx * usc;
        if (__ballot(mxs > m + 1.0f)) {  // (m follows the maximum when a weight would pass 2, column by column)
            const float mnew = mxs > m + 1.0f ? mxs : m, alpha = m == -INFINITY ? 0.0f : exp2_hw(m - mnew);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) r.o[d] *= alpha;
            m = mnew;
        }
        const float mref = (m == -INFINITY ? 0.0f : m) - 14.0f;  // (the weights times TILE_SCALE)
        // the softmax of this tile's 32 values, 32 / KS a step, beside the four matrix instructions of a step of the next one's
        // scores, whose fragments are read a step ahead
        f16v x[2];
        h8 ph[4], pl[4], kf[2][2];
        const uint8_t* kn = kbuf + (buf ^ 1) * L::KB;
        const uint32_t kf0o = opaque(kf0);
        auto frag = [&](int k) __attribute__((always_inline)) {
            kf[k & 1][0] = *(const h8*)(kn + (kf0o ^ (32 * k)));
            kf[k & 1][1] = *(const h8*)(kn + 32 * L::ROW + (kf0o ^ (32 * k)));
        };
        if constexpr (next) {
            frag(0);
#pragma unroll
            for (int i = 0; i < 16; i++) x[0][i] = x[1][i] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < KS; k++) {
            if constexpr (next) {
                if (k + 1 < KS) frag(k + 1);
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][0], qh[k], x[0], 0, 0, 0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][1], qh[k], x[1], 0, 0, 0);
                x[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][0], ql[k], x[0], 0, 0, 0);
                x[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[k & 1][1], ql[k], x[1], 0, 0, 0);
            }
#pragma unroll
            for (int v = 32 / KS * k; v < 32 / KS * (k + 1); v += 2) {
                const int b = v >> 3, e = v & 7;
                const float p0 = exp2_hw(__builtin_fmaf(s[b >> 1][8 * (b & 1) + e], usc, -mref));
                const float p1 = exp2_hw(__builtin_fmaf(s[b >> 1][8 * (b & 1) + e + 1], usc, -mref));
                l += p0;
                l += p1;
                const auto h = __builtin_amdgcn_cvt_pkrtz(p0, p1);
                ph[b][e] = (_Float16)h[0];
                ph[b][e + 1] = (_Float16)h[1];
                pl[b][e] = (_Float16)__builtin_fmaf(p0, one, -(float)h[0]);
                pl[b][e + 1] = (_Float16)__builtin_fmaf(p1, one, -(float)h[1]);
            }
        }
        const uint8_t* vt = vbuf + buf * L::KB;
        const uint32_t vf0o = opaque(vf0);
#pragma unroll
        for (int b = 0; b < 4; b++) {
            h8 vf[DT];
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const h4 v0 = read_tr((const uint16_t*)(vt + 16 * b * L::ROW + (vf0o ^ (64 * d))));
                const h4 v1 = read_tr((const uint16_t*)(vt + (16 * b + 8) * L::ROW + (vf0o ^ (64 * d) ^ 32)));
                vf[d] = __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7);
            }
#pragma unroll
            for (int d = 0; d < DT; d++) r.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], ph[b], r.o[d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < DT; d++) r.o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[d], pl[b], r.o[d], 0, 0, 0);
        }
        if constexpr (next) {
            s[0] = x[0];
            s[1] = x[1];
            wait_loads();
            lds_barrier();
            mask(kt + 1, hole1, s);
            hole1 = holes(pg);
            mx = largest(s);
        }
    };
    if (kb < ke) {
        wait_loads();
        lds_barrier();
        scores(0, s);
        mask(kb, hole, s);
        mx = largest(s);
        // (the K of tile kb has been read by all waves before tile kb + 2's may land on it)
        lds_barrier();
        for (int kt = kb; kt + 1 < ke; kt++) tile(kt, std::integral_constant<bool, true>{});
        tile(ke - 1, std::integral_constant<bool, false>{});
        lds_barrier();  // (the buffers are free for what comes next)
    }
    r.l = l + __shfl_xor(l, 32, 64);
    r.m = m;
}

// The rows of a wave whose sums may owe a value that is not finite to a key that they do not see (finite scores, sums that are
// not): bit l32.
template <int HD>
__device__ __forceinline__ uint32_t tile_again(const TileSums<HD>& r, bool live) {
    float nf = 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) nf = __builtin_fmaf(r.o[d][i], 0.0f, nf);
    const uint64_t b = __ballot(nf != 0.0f && r.l - r.l == 0.0f && live);
    return (uint32_t)b | (uint32_t)(b >> 32);
}
// The wave's rows times their factors f, from the fragments' layout (16 bytes of a row a lane) through LDS (free of tiles) to
// whole rows: row r (0 .. 31, a bit of `rows`) to dst(r), through gate(r) where there is one. Chunk c of row r sits at c ^ r.
template <int HD, typename D, typename G>
__device__ __forceinline__ void tile_store(const TileSums<HD>& r, int tid, float f, uint8_t* lds, uint32_t rows, D&& dst, G&& gate) {
    constexpr int NC = HD / 4, RPL = 64 / NC;  // chunks a row, rows a load
    const int lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
    uint8_t* mine = lds + (tid >> 6) * (32 * 4 * HD);
#pragma unroll
    for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int j = 0; j < 4; j++)
            *(float4*)(mine + l32 * 4 * HD + 16 * ((8 * d + 2 * j + hf) ^ (l32 & (NC - 1)))) =
                make_float4(r.o[d][4 * j] * f, r.o[d][4 * j + 1] * f, r.o[d][4 * j + 2] * f, r.o[d][4 * j + 3] * f);
    __builtin_amdgcn_wave_barrier();
#pragma unroll 4
    for (int i = 0; i < 32 / RPL; i++) {
        const int row = RPL * i + lane / NC, c = (lane % NC) ^ (row & (NC - 1));
        if ((rows >> row) & 1) {
            float4 v = *(const float4*)(mine + row * 4 * HD + 16 * (lane % NC));
            if (const float* gt = gate(row)) {
                const float4 x = *(const float4*)(gt + 4 * c);
                v.x *= sigmoid_f(x.x); v.y *= sigmoid_f(x.y); v.z *= sigmoid_f(x.z); v.w *= sigmoid_f(x.w);
            }
            *(float4*)(dst(row) + 4 * c) = v;
        }
    }
    __builtin_amdgcn_wave_barrier();
}

// The prefix for the rows of decode sequences: tiles of the call's rows (of the plan's list of them, where there is a plan)
// whatever their sequence, so that the prefix's K and V are read once a tile of 128 / G tokens rather than once a token; a
// block takes a split of the prefix's keys. Blocks are numbered so that the tiles over the same keys run on one XCD (its L2
// holds a split's K and V). 64 rows of 32 heads over 16000 keys, own keys beside them: 52 us.
template <int HD>
__device__ __forceinline__ void prefix_block(const PagedAttn& a, const PagedWs& w, int x, int tiles, uint8_t* lds) {
    __shared__ int ws[8];
    int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.nh / a.nkv, gs = 31 - __builtin_clz(G), TT = 128 >> gs, ns = w.nsp;
    const Keys keys{a.prefix, nullptr, prefix_len(a), (prefix_len(a) + 63) / 64, 0};
    // block x: combination (KV head, split) c on XCD c % 8, tile tt
    const int c = (x & 7) + 8 * ((x >> 3) / tiles), tt = (x >> 3) % tiles;
    if (c >= a.nkv * ns || !keys.P) return;
    const int g = c % a.nkv, split = c / a.nkv;
    const int nrows = w.drows ? sload(w.plan + 2) : min(max(sload(a.q_start + a.nseq), 0), a.t), nt = min(TT, nrows - tt * TT);
    if (nt <= 0) return;
    auto tok_of = [&](int i) { return (32 * wave + i) >> gs; };  // of the wave's row i, and its head
    auto head_of = [&](int i) { return g * G + (i & (G - 1)); };
    auto row_of = [&](int t) { return w.drows ? w.drows[tt * TT + t] : tt * TT + t; };
    auto sums_of = [&](int i) { return ((uint64_t)(tt * TT + tok_of(i)) * a.nh + head_of(i)) * ns + split; };
    const int t = row_of(tok_of(tid & 31) < nt ? tok_of(tid & 31) : 0), pos = a.pos[t];
    int lo, hi;
    row_range(a, keys, pos, lo, hi);
    // the tiles that the block's rows see
    int blo = tok_of(tid & 31) < nt ? lo : INT_MAX, bhi = tok_of(tid & 31) < nt ? hi : -1;
    static_for<0, 5>([&](auto S) {
        constexpr int st = decltype(S)::value;
        blo = min(blo, xl32<st>(blo));
        bhi = max(bhi, xl32<st>(bhi));
    });
    if ((tid & 63) == 0) {
        ws[wave] = blo;
        ws[4 + wave] = bhi;
    }
    __syncthreads();
    blo = __builtin_amdgcn_readfirstlane(min(min(ws[0], ws[1]), min(ws[2], ws[3])));
    bhi = __builtin_amdgcn_readfirstlane(max(max(ws[4], ws[5]), max(ws[6], ws[7])));
    const int kt0 = bhi < 0 ? 0 : blo / 64, kt1 = bhi < 0 ? 0 : bhi / 64 + 1, per = (kt1 - kt0 + ns - 1) / ns;
    const int kb = min(kt0 + split * per, kt1), ke = min(kb + per, kt1);
    TileSums<HD> r;
    tile_run<HD>(a, keys, lds, g, kb, ke, tok_of(tid & 31) < nt, a.q + ((uint64_t)t * a.nh + head_of(tid & 31)) * HD, pos, r);
    asm volatile("" : "+v"(tid));  // (nothing of this lane's row waits in registers while the tiles run)
    const int lane = tid & 63, l32 = lane & 31;
    const bool live = tok_of(l32) < nt;
    uint32_t again = tile_again<HD>(r, live);
    const uint32_t rows = (uint32_t)__ballot(live) & ~again;
    tile_store<HD>(r, tid, 1.0f / TILE_SCALE, lds, rows, [&](int i) { return w.pacc + sums_of(i) * HD; }, [](int) { return (const float*)nullptr; });
    if (lane < 32 && ((rows >> l32) & 1)) w.pml[sums_of(l32)] = make_float2(r.m, r.l * (1.0f / TILE_SCALE));
    for (; again; again &= again - 1) {
        const int i = __builtin_ctz(again), tb = row_of(tok_of(i));
        row_range(a, keys, a.pos[tb], lo, hi);
        float ac[HD / 64], mm, ll;
        paged_row_again<HD>(a, keys, a.q + ((uint64_t)tb * a.nh + head_of(i)) * HD, g, max(lo, 64 * kb), min(hi, 64 * ke - 1), ac, mm, ll);
#pragma unroll
        for (int d = 0; d < HD / 64; d++) w.pacc[sums_of(i) * HD + lane + 64 * d] = ac[d];
        if (lane == 0) w.pml[sums_of(i)] = make_float2(mm, ll);
    }
}

// Long sequences. The plan: for each tile of 128 / G tokens of each of them its rows and the tiles of 64 virtual keys that they
// see, and the prefix sums of those; the work is the list of all (KV head, tile, key tile), key tile fastest, and a block takes
// an equal run of it, so chunks at any depth of their contexts load the CUs evenly. A tile that lies in one run is finished by
// its block; of one cut by a run's end each block leaves its sums (the piece from a tile's start at slot 2 b + 1, one that goes
// on from the run before at 2 b), and attn_paged_join_kernel joins them.
struct PlanTile {
    int s, t0, nt, len;  // sequence, first row, rows, own keys
    int kt0, nkt, cum, pad;  // first key tile, key tiles; work of the tiles before
};
constexpr int PLAN_HEAD = 4;  // tiles, their work, rows of decode sequences
// A tile's work in key tiles: those it has, and what it takes to begin and end one (9 + 4 us beside 4 a key tile). With 0 here
// chunks of 2501 tokens take 174 us for 132, long contexts the same.
constexpr int TILE_EXTRA = 3;

// One block of 1024 threads: the sequences' tiles by a scan in LDS, then the tiles' keys and their scan, 1024 tiles at a time.
__global__ __launch_bounds__(1024) void attn_paged_plan_kernel(PagedAttn a, PagedWs w, int tiles) {
    __shared__ int start[SERVE_MAX_SEQ], dstart[SERVE_MAX_SEQ], row0[SERVE_MAX_SEQ + 1], ws[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, G = a.nh / a.nkv, TT = 128 / G, P = prefix_len(a), np = (P + 63) / 64;
    auto scan = [&](int v, int& total) {  // exclusive, over the block
        int inc = v;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(inc, o, 64);
            if (lane >= o) inc += u;
        }
        __syncthreads();
        if (lane == 63) ws[wave] = inc;
        __syncthreads();
        int before = inc - v;
        total = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            if (i < wave) before += ws[i];
            total += ws[i];
        }
        return before;
    };
    int nt[4], nd[4], q[5], sum = 0, dsum = 0, ntiles, ndec = 0;
#pragma unroll
    for (int i = 0; i < 5; i++) q[i] = 4 * tid + i <= a.nseq ? a.q_start[4 * tid + i] : 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = 4 * tid + i, q0 = min(max(q[i], 0), a.t), qn = s < a.nseq ? min(max(q[i + 1], q0), a.t) - q0 : 0;
        const bool dec = qn * G <= w.dr;
        nt[i] = dec ? 0 : (qn + TT - 1) / TT;
        nd[i] = dec ? qn : 0;
        if (s <= a.nseq) row0[s] = q0;
        sum += nt[i];
        dsum += nd[i];
    }
    if (tid == 1023 && a.nseq == SERVE_MAX_SEQ) row0[SERVE_MAX_SEQ] = min(max(q[4], 0), a.t);
    int at = scan(sum, ntiles), dat = w.drows ? scan(dsum, ndec) : 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (4 * tid + i < a.nseq) {
            start[4 * tid + i] = at;
            dstart[4 * tid + i] = dat;
            if (w.drows) w.dstart[4 * tid + i] = dat;
        }
        at += nt[i];
        dat += nd[i];
    }
    __syncthreads();
    auto find = [&](const int* v, int x) {  // the last sequence with v[s] <= x
        int lo = 0, hi = a.nseq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (v[mid] <= x) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    ntiles = min(ntiles, tiles);
    ndec = min(ndec, a.t);
    if (w.drows)
        for (int i = tid; i < ndec; i += 1024) {
            const int s = find(dstart, i);
            w.drows[i] = min(row0[s] + i - dstart[s], a.t - 1);
        }
    PlanTile* plan = (PlanTile*)(w.plan + PLAN_HEAD);
    int cum = 0;
    for (int i0 = 0; i0 < ntiles; i0 += 1024) {
        const int i = i0 + tid;
        PlanTile p{};
        if (i < ntiles) {
            p.s = find(start, i);
            const int q0 = row0[p.s], q1 = max(row0[p.s + 1], q0);
            p.t0 = q0 + (i - start[p.s]) * TT;
            p.nt = min(TT, q1 - p.t0);
            p.len = (int)min((long long)max(a.len[p.s], 0), (long long)a.max_pages << a.page_shift);
            const Keys keys{nullptr, nullptr, P, np, p.len};
            int first = INT_MAX, last = -1;
            for (int t = 0; t < p.nt; t += 16) {
                int pos[16];
#pragma unroll
                for (int e = 0; e < 16; e++) pos[e] = a.pos[p.t0 + min(t + e, p.nt - 1)];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    int lo, hi;
                    row_range(a, keys, pos[e], lo, hi);
                    first = min(first, lo);
                    last = max(last, hi);
                }
            }
            p.kt0 = last < 0 ? 0 : first / 64;
            p.nkt = last < 0 ? 1 : last / 64 + 1 - p.kt0;  // (rows without keys are written too: a tile that nothing of is computed)
        }
        int total;
        p.cum = cum + scan(i < ntiles ? p.nkt + TILE_EXTRA : 0, total);
        cum += total;
        if (i < ntiles) plan[i] = p;
    }
    if (tid == 0) {
        w.plan[0] = ntiles;
        w.plan[1] = cum;
        w.plan[2] = ndec;
    }
}

// The tile whose work holds x (0 <= x < all), by a wave in rounds of 64 loads.
__device__ __forceinline__ int tile_of(const PlanTile* plan, int n, int x) {
    const int lane = threadIdx.x & 63;
    int lo = 0;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const uint64_t le = __ballot(i < n && plan[lo + min(i, n - 1)].cum <= x);
        const int k = le ? 63 - __builtin_clzll(le) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return __builtin_amdgcn_readfirstlane(lo);
}
__device__ __forceinline__ PlanTile plan_tile(const PlanTile* p) {
    return PlanTile{sload(&p->s), sload(&p->t0), sload(&p->nt), sload(&p->len), sload(&p->kt0), sload(&p->nkt), sload(&p->cum), 0};
}
// Where block b's run of the list begins: at b times an equal share of the work, moved to the tile's border where one key tile, and
// no more than an eighth of the share, lies between: a tile that is not cut costs no sums, but the run becomes longer (up to 3 key
// tiles: chunks of 2501 tokens 132 us for 130, up to 5 134).
struct RunAt {
    long long at;  // in the list of all tiles' work
    int g, i, f;   // the KV head, the tile, the key tile of it
    long long share;
    int near;
};
__device__ __forceinline__ RunAt run_at(const PlanTile* plan, int n, int cost, int nkv, int b, int blocks) {
    const long long all = (long long)cost * nkv, share = max((all + blocks - 1) / blocks, 2ll);
    const int near = (int)min(share / 8, 1ll);
    RunAt r{min(b * share, all), nkv, 0, 0, share, near};
    if (r.at == all) return r;
    r.g = (int)(r.at / cost);
    const int x = (int)(r.at - (long long)r.g * cost);
    r.i = tile_of(plan, n, x);
    const int cum = sload(&plan[r.i].cum), nkt = sload(&plan[r.i].nkt), f = x - cum - TILE_EXTRA;
    if (f <= near) {
        r.at -= x - cum;
    } else if (nkt - f <= near) {
        r.at += cum + TILE_EXTRA + nkt - x;
        if (++r.i == n) r.i = 0, r.g++;
    } else {
        r.f = f;
    }
    return r;
}

template <int HD>
__device__ __forceinline__ void tile_block(const PagedAttn& a, const PagedWs& w, int x, uint8_t* lds) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int G = a.nh / a.nkv, gs = 31 - __builtin_clz(G), P = prefix_len(a);
    const PlanTile* plan = (const PlanTile*)(w.plan + PLAN_HEAD);
    const int n = sload(w.plan), cost = sload(w.plan + 1);
    // the b-th run; neighbours in the list, which share keys, run on one XCD
    const int b = (x & 7) * (w.tblocks / 8) + (x >> 3);
    if (!n) {
        if (threadIdx.x == 0) w.cut[b] = make_int4(0, 0, -1, 0);
        return;
    }
    const RunAt from = run_at(plan, n, cost, a.nkv, b, w.tblocks), to = run_at(plan, n, cost, a.nkv, b + 1, w.tblocks);
    if (threadIdx.x == 0) {
        // the tile that begins in this run and goes on past it: the last block of its pieces (run_at's borders)
        int last = -1;
        if (to.f && (from.g != to.g || from.i != to.i || !from.f)) {
            const PlanTile p = plan_tile(plan + to.i);
            const long long end = (long long)cost * to.g + p.cum + TILE_EXTRA + p.nkt;
            last = (int)min((end - to.near - 1) / to.share, (long long)w.tblocks - 1);
        }
        w.cut[b] = make_int4(to.g, to.i, last, 0);
    }
    for (int g = from.g, i = from.i, f = from.f; g < to.g || (g == to.g && (i < to.i || (i == to.i && f < to.f)));) {
        const PlanTile p = plan_tile(plan + i);
        const int k = (g == to.g && i == to.i ? to.f : p.nkt) - f;
        const bool whole = k == p.nkt;
        const Keys keys{a.prefix, a.tables + (uint64_t)p.s * a.max_pages, P, (P + 63) / 64, p.len};
        const int kb = p.kt0 + f, ke = keys.P || keys.len ? kb + k : kb;
        TileSums<HD> r;
        {
            const int rr = 32 * wave + (threadIdx.x & 31), tok = rr >> gs, h = g * G + (rr & (G - 1)), t = p.t0 + (tok < p.nt ? tok : 0);
            tile_run<HD>(a, keys, lds, g, kb, ke, tok < p.nt, a.q + ((uint64_t)t * a.nh + h) * HD, a.pos[t], r);
        }
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));  // (nothing of this lane's row waits in registers while the tiles run)
        const int lane = tid & 63, l32 = lane & 31, rr = 32 * wave + l32, h = g * G + (rr & (G - 1));
        const bool live = (rr >> gs) < p.nt;
        uint32_t again = tile_again<HD>(r, live);
        const uint64_t slot = (uint64_t)(2 * b + (f == 0)) * 128;
        const uint32_t rows = (uint32_t)__ballot(live) & ~again;
        auto row_at = [&](int i) { return (uint64_t)(p.t0 + ((32 * wave + i) >> gs)) * a.nh + g * G + (i & (G - 1)); };
        tile_store<HD>(r, tid, (whole ? out_factor(a, h, r.m, r.l * (1.0f / TILE_SCALE)) : 1.0f) * (1.0f / TILE_SCALE), lds, rows,
                       [&](int i) { return whole ? a.out + row_at(i) * HD : w.tacc + (slot + 32 * wave + i) * HD; },
                       [&](int i) { return whole && a.qg ? a.qg + row_at(i) * 2 * HD + HD : (const float*)nullptr; });
        if (!whole && lane < 32 && ((rows >> l32) & 1)) w.tml[slot + rr] = make_float2(r.m, r.l * (1.0f / TILE_SCALE));
        for (; again; again &= again - 1) {
            const int rb = 32 * wave + __builtin_ctz(again), tb = p.t0 + (rb >> gs), hb = g * G + (rb & (G - 1));
            const uint64_t rowb = (uint64_t)tb * a.nh + hb;
            int lo, hi;
            row_range(a, keys, a.pos[tb], lo, hi);
            float ac[HD / 64], mm, ll;
            paged_row_again<HD>(a, keys, a.q + rowb * HD, g, max(lo, 64 * kb), min(hi, 64 * ke - 1), ac, mm, ll);
            const float fo = whole ? out_factor(a, hb, mm, ll) : 1.0f;
            float* dst = whole ? a.out + rowb * HD : w.tacc + (slot + rb) * HD;
#pragma unroll
            for (int d = 0; d < HD / 64; d++) {
                const int col = lane + 64 * d;
                dst[col] = whole && a.qg ? ac[d] * fo * sigmoid_f(a.qg[rowb * 2 * HD + HD + col]) : ac[d] * fo;
            }
            if (!whole && lane == 0) w.tml[slot + rb] = make_float2(mm, ll);
        }
        f += k;
        if (f == p.nkt) {
            f = 0;
            if (++i == n) i = 0, g++;
        }
        lds_barrier();  // (the rows have left LDS)
    }
}

// A tile that begins in block b's run and goes on past it, joined: the pieces' sums of its 128 rows, 4 rows a wave at a time
// with their loads in flight together; y of HD / 32 blocks.
template <int HD>
__device__ __forceinline__ void join_block(const PagedAttn& a, const PagedWs& w, int b, int y) {
    constexpr int NC = HD / 4, RPW = 64 / NC, U = 4;  // lanes a row (16 bytes each), rows a wave and load, loads
    const int lane = threadIdx.x & 63, last = sload(&w.cut[b].z);
    if (last < 0) return;
    struct { int g, i; } end{sload(&w.cut[b].x), sload(&w.cut[b].y)};
    const PlanTile p = plan_tile((const PlanTile*)(w.plan + PLAN_HEAD) + end.i);
    const int G = a.nh / a.nkv, gs = 31 - __builtin_clz(G), nr = p.nt * G, col = 4 * (lane % NC);
    const int r0 = (y * 4 + (threadIdx.x >> 6)) * U * RPW + lane / NC;
    float M[U], L[U];
    float4 acc[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        M[u] = -INFINITY;
        L[u] = 0.0f;
        acc[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int c = b; c <= last; c++) {
        float2 ml[U];
        float4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint64_t at = (uint64_t)(2 * c + (c == b)) * 128 + min(r0 + u * RPW, nr - 1);
            ml[u] = w.tml[at];
            v[u] = *(const float4*)(w.tacc + at * HD + col);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float mnew = fmaxf(M[u], ml[u].x), f = M[u] == -INFINITY ? 0.0f : exp2_hw(M[u] - mnew);
            const bool none = ml[u].x == -INFINITY;  // (a piece without a maximum has a sum of 0, or not a number)
            const float e = none ? 0.0f : exp2_hw(ml[u].x - mnew);
            L[u] = L[u] * (M[u] == -INFINITY ? 1.0f : f) + (none ? ml[u].y : ml[u].y * e);
            acc[u].x = acc[u].x * f + (none ? 0.0f : v[u].x * e);
            acc[u].y = acc[u].y * f + (none ? 0.0f : v[u].y * e);
            acc[u].z = acc[u].z * f + (none ? 0.0f : v[u].z * e);
            acc[u].w = acc[u].w * f + (none ? 0.0f : v[u].w * e);
            M[u] = mnew;
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int rr = r0 + u * RPW;
        if (rr >= nr) continue;
        const int h = end.g * G + (rr & (G - 1));
        const uint64_t row = (uint64_t)(p.t0 + (rr >> gs)) * a.nh + h;
        const float f = out_factor(a, h, M[u], L[u]);
        float4 x = make_float4(acc[u].x * f, acc[u].y * f, acc[u].z * f, acc[u].w * f);
        if (a.qg) {
            const float* gt = a.qg + row * 2 * HD + HD + col;
            x.x *= sigmoid_f(gt[0]); x.y *= sigmoid_f(gt[1]); x.z *= sigmoid_f(gt[2]); x.w *= sigmoid_f(gt[3]);
        }
        *(float4*)(a.out + row * HD + col) = x;
    }
}

// ---------------- the join of a decode sequence's rows ----------------
// An item is a row and query head, of all rows or (DIRECT) of the pairs that blocks cut, from its partial sums: out = sum_i acc_i
// 2^(m_i - M) / (sum_i l_i 2^(m_i - M) + 2^(sink - M)), the prefix's splits, then the own keys' pieces. Wave v of an item's MW takes
// partials v, v + MW, .., their maxima a lane each and 4 rows requested together (a launch is a chain of trips to memory: the
// sequence, then these). Two waves an item: 2048 items of 64 sequences of 200 .. 6000 keys 5.7 us (four waves 7.1, one 5.4); 768 of
// 4 .. 16 partials 6.6 us (8.4, 8.2). Four waves up to 512 items (a call with one sequence of 32768 keys and one KV head, 128
// pieces, 17 us, with two 21.5; of 131072 keys and four 52 and 57).
template <int HD, bool DIRECT, int MW>
__device__ __forceinline__ void merge_block(const PagedAttn& a, const PagedWs& w, int x, int per) {
    constexpr int DL = HD / 64, ITEMS = 4 / MW, U = 4;
    __shared__ float sm[ITEMS][MW], sl[ITEMS][MW], so[ITEMS][MW][HD];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), v = wave % MW, it = wave / MW, lane = threadIdx.x & 63;
    const int G = a.nh / a.nkv, P = prefix_len(a);
    const int y = ITEMS * x + it;
    int s = min(y / a.nh / per, a.nseq - 1), h = y % a.nh, i = y / a.nh % per, first, pieces;
    SeqInfo q;
    if constexpr (!DIRECT) {
        const int2* mp = w.map + s * a.nkv + h / G;
        first = sload(&mp->x), pieces = sload(&mp->y);  // (not set, and not used, without own keys)
        q = seq_info<true>(a, s, G, w.dr, P);
    } else {
        if (x < a.nseq) {  // sequence x without own keys: its rows are 0
            q = seq_info<true>(a, x, G, w.dr, P);
            if (q.nc == 0 && q.qn * G <= w.dr)
                for (int j = threadIdx.x; j < q.qn * a.nh * (HD / 4); j += 256)
                    *(float4*)(a.out + (uint64_t)q.q0 * a.nh * HD + 4 * j) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        first = min(y / w.dr, w.dblocks - 1);
        const int pair = sload(&w.map[first].x), c = y % w.dr;
        pieces = sload(&w.map[first].y);
        s = pair / a.nkv, h = pair % a.nkv * G + c % G, i = c / G;
        q = seq_info<true>(a, s, G, w.dr, P);
    }
    const int g = h / G, r = q.q0 + i;
    const bool live = (DIRECT ? pieces > 0 && y < w.dblocks * w.dr : y < a.nseq * per * a.nh) && i < q.qn && q.qn * G <= w.dr;
    const uint64_t row = (uint64_t)r * a.nh + h;
    const int np = P > 0 ? w.nsp : 0, n = live ? np + (q.nc > 0 ? pieces : 0) : 0;
    const uint64_t own = (uint64_t)(first + s * a.nkv + g) * w.dr + (r - q.q0) * G + h % G;  // piece i of the own keys: own + i dr
    // (a place past the list's room belongs to no row that the call's q_start allows)
    const int pr = !DIRECT && w.drows ? min(sload(w.dstart + s) + i, w.prows - 1) : r;
    const uint64_t pre = ((uint64_t)pr * a.nh + h) * np;
    auto at = [&](int i) { return i < np ? pre + i : own + (uint64_t)(i - np) * w.dr; };
    float M = -INFINITY, L = 0.0f, acc[DL], gt[DL];
#pragma unroll
    for (int d = 0; d < DL; d++) {
        acc[d] = 0.0f;
        gt[d] = live && a.qg ? a.qg[row * 2 * HD + HD + DL * lane + d] : 0.0f;
    }
    for (int i0 = v; i0 < n; i0 += 64 * MW) {
        const int i = i0 + MW * lane;
        float2 ml = make_float2(-INFINITY, 0.0f);
        if (i < n) ml = (i < np ? w.pml : w.dml)[at(i)];
        const int cnt = min((n - i0 + MW - 1) / MW, 64);
        for (int j0 = 0; j0 < cnt; j0 += U) {
            float av[U][DL];
#pragma unroll
            for (int j = 0; j < U; j++) {  // (past the last partial: the first one again, with no weight)
                const int ii = j0 + j < cnt ? i0 + MW * (j0 + j) : i0;
                const float* src = (ii < np ? w.pacc : w.dacc) + at(ii) * HD;
#pragma unroll
                for (int d = 0; d < DL; d++) av[j][d] = src[DL * lane + d];
            }
            if (j0 == 0) {
                const float mnew = fmaxf(M, wave_max64(ml.x)), f = M == -INFINITY ? 0.0f : exp2_hw(M - mnew);
                const float e = ml.x == -INFINITY ? 1.0f : exp2_hw(ml.x - mnew);  // (a partial without a maximum has a sum of 0, or not a number)
                L = L * f + wave_sum64(ml.y * e);
#pragma unroll
                for (int d = 0; d < DL; d++) acc[d] *= f;
                M = mnew;
            }
            const float e = exp2_hw(ml.x - M);
            const uint64_t some = __ballot(ml.x != -INFINITY);  // (an empty partial's row is not written)
#pragma unroll
            for (int j = 0; j < U; j++) {
                const float es = __shfl(e, (j0 + j) & 63, 64);
                const bool has = j0 + j < cnt && ((some >> ((j0 + j) & 63)) & 1);
#pragma unroll
                for (int d = 0; d < DL; d++) acc[d] += has ? av[j][d] * es : 0.0f;
            }
        }
    }
    if (lane == 0) {
        sm[it][v] = M;
        sl[it][v] = L;
    }
#pragma unroll
    for (int d = 0; d < DL; d++) so[it][v][DL * lane + d] = acc[d];
    __syncthreads();
    if (v || !live) return;
    M = sm[it][0];
#pragma unroll
    for (int u = 1; u < MW; u++) M = fmaxf(M, sm[it][u]);
    L = 0.0f;
#pragma unroll
    for (int d = 0; d < DL; d++) acc[d] = 0.0f;
#pragma unroll
    for (int u = 0; u < MW; u++) {
        const float f = sm[it][u] == -INFINITY ? 1.0f : exp2_hw(sm[it][u] - M);
        L += sl[it][u] * f;
#pragma unroll
        for (int d = 0; d < DL; d++) acc[d] += so[it][u][DL * lane + d] * f;
    }
    const float f = out_factor(a, h, M, L);
#pragma unroll
    for (int d = 0; d < DL; d++) {
        float o = acc[d] * f;
        if (a.qg) o *= sigmoid_f(gt[d]);
        a.out[row * HD + DL * lane + d] = o;
    }
}

// ---------------- launches ----------------
// The pieces: blocks of the long sequences' tiles (TILE), of the prefix for the rows of decode sequences (PRE) and of their own
// keys, in one launch.
template <int HD, int NT, bool TILE, bool PRE, bool DIRECT>
__global__ __launch_bounds__(256, NT == 1 || HD == 64 ? 2 : 1) void attn_paged_kernel(PagedAttn a, PagedWs w, int pblocks, int tiles) {
    constexpr int TB = TILE || PRE ? 2 * PagedTile<HD>::BUF : 0;
    __shared__ __align__(16) uint8_t lds[PagedDec<HD>::BYTES > TB ? PagedDec<HD>::BYTES : TB];
    int b = blockIdx.x;
    if constexpr (TILE) {
        if (b < w.tblocks) return tile_block<HD>(a, w, b, lds);
        b -= w.tblocks;
    }
    if constexpr (PRE) {
        if (b < pblocks) return prefix_block<HD>(a, w, b, tiles, lds);
        b -= pblocks;
    }
    dec_block<HD, NT, DIRECT>(a, w, b, lds);
}
// The joins: of the tiles in pieces, and of the rows of decode sequences.
template <int HD, bool DIRECT, int MW>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(PagedAttn a, PagedWs w, int jblocks, int per) {
    const int b = blockIdx.x;
    if (b < jblocks) return join_block<HD>(a, w, b / (HD / 32), b % (HD / 32));
    merge_block<HD, DIRECT, MW>(a, w, b - jblocks, per);
}

static int div_up(long long a, long long b) { return (int)((a + b - 1) / b); }

// Tiles of the long sequences at most: each of them has more than dr / G rows.
static int max_tiles(const PagedAttn& a, const PagedWs& w) {
    const int G = a.nh / a.nkv;
    return a.t / (128 / G) + std::min(a.nseq, a.t / (w.dr / G + 1)) + 1;
}

// The split plan and the workspace's layout from `at`; the end of the layout in *end.
static PagedWs plan(const PagedAttn& a, uint8_t* at, size_t* end) {
    PagedWs w{};
    const int G = a.nh / a.nkv;
    // a sequence decodes up to 16 rows (one column tile), up to 32 where the longest has no more (64 sequences of 4 tokens, 8 heads a
    // KV head, over 2048 keys: 70 us, as tiles of 128 rows 97)
    const long long most_rows = (long long)a.max_q * G;
    w.nct = most_rows > 16 && most_rows <= 32 ? 2 : 1;
    w.dr = (int)std::min<long long>(16 * w.nct, most_rows);
    const long long most = (long long)a.nseq * a.nkv * (((long long)a.max_pages << a.page_shift) / DEC_CHUNK + 1);
    // the blocks that run at once: two a CU (64 ragged sequences 117 us against 122, 300 of 700 keys 104 against 116; a few long ones
    // gain 3 to 5% from one), one where two column tiles of 128 values fill a CU's registers (of 64 values two: 100 sequences of 4
    // tokens 169 us against 211) or the prefix's blocks take the other's place (24 of 4 tokens over a prefix 24.2 us against 26.4, 64
    // over one of 4096 33 against 41)
    w.dblocks = (int)std::min<long long>(most, (w.nct == 1 || a.hd == 64) && (!a.max_prefix || most_rows > w.dr) ? 512 : 256);
    // where no more (sequence, KV head) than blocks are there, most are cut and each of their rows is joined (64 sequences of 2000
    // keys over 4 KV heads 49 us, direct 53); else most are not (256: 196 and 187; 1000 of 300 keys 177 and 139)
    w.direct = !a.max_prefix && (long long)a.nseq * a.nkv >= w.dblocks;
    // splits of the prefix, of at least 128 keys: a block a CU (64 sequences over a prefix of 4096 31 us, for two a CU 46; of 16000 56
    // and 59): more of them cost more sums than they hide. The rows that count are those of sequences that may decode (all t rows
    // left the decode rows beside chunks with a few long splits: 512 tokens and 63 decoding sequences over 16000 511 us for 336,
    // 1500 tokens and 4 over 2000 212 for 169)
    w.prows = (int)(most_rows > w.dr ? std::min<long long>(a.t, (long long)a.nseq * (w.dr / G)) : a.t);
    const long long blocks = std::max<long long>((long long)div_up((long long)w.prows * G, 128) * a.nkv, 1);
    w.nsp = (int)std::max<long long>(1, std::min<long long>({div_up(256, blocks), div_up(a.max_prefix, 128), 64}));
    w.tblocks = 512;
    size_t o = 0;
    auto take = [&](size_t bytes) {
        uint8_t* p = at + o;
        o += (bytes + 255) & ~(size_t)255;
        return (void*)p;
    };
    const size_t slots = (size_t)w.dblocks + (size_t)a.nseq * a.nkv, out_rows = (size_t)w.prows * a.nh;
    w.map = (int2*)take(std::max((size_t)a.nseq * a.nkv, (size_t)w.dblocks) * sizeof(int2));
    w.dml = (float2*)take(slots * w.dr * sizeof(float2));
    w.dacc = (float*)take(slots * w.dr * a.hd * sizeof(float));
    if (a.max_prefix) {
        w.pml = (float2*)take(out_rows * w.nsp * sizeof(float2));
        w.pacc = (float*)take(out_rows * w.nsp * a.hd * sizeof(float));
    }
    if (most_rows > w.dr) {
        w.plan = (int*)take((PLAN_HEAD + (size_t)max_tiles(a, w) * (sizeof(PlanTile) / 4)) * 4);
        if (a.max_prefix) {
            w.drows = (int*)take((size_t)a.t * 4);
            w.dstart = (int*)take((size_t)a.nseq * 4);
        }
        w.cut = (int4*)take((size_t)w.tblocks * sizeof(int4));
        w.tml = (float2*)take((size_t)2 * w.tblocks * 128 * sizeof(float2));
        w.tacc = (float*)take((size_t)2 * w.tblocks * 128 * a.hd * sizeof(float));
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
    const int G = a.nh / a.nkv, TT = 128 / G, per = w.dr / G;
    int tiles = 0, pblocks = 0;
    if (w.plan) attn_paged_plan_kernel<<<dim3(1), dim3(1024), 0, s>>>(a, w, max_tiles(a, w));
    if (a.max_prefix) {
        tiles = div_up(w.prows, TT);
        pblocks = 8 * div_up((long long)a.nkv * w.nsp, 8) * tiles;
    }
    const dim3 grid((unsigned)((w.plan ? w.tblocks : 0) + pblocks + w.dblocks)), block(256);
    auto launch = [&](auto NT, auto TILE, auto PRE, auto DIRECT) {
        attn_paged_kernel<HD, decltype(NT)::value, decltype(TILE)::value, decltype(PRE)::value, decltype(DIRECT)::value><<<grid, block, 0, s>>>(a, w, pblocks, tiles);
    };
    constexpr std::integral_constant<int, 1> one;
    constexpr std::integral_constant<int, 2> two;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    if (w.nct == 2) {
        if (a.max_prefix) launch(two, no, yes, no);
        else if (w.direct) launch(two, no, no, yes);
        else launch(two, no, no, no);
    } else if (w.plan) {
        if (a.max_prefix) launch(one, yes, yes, no);
        else if (w.direct) launch(one, yes, no, yes);
        else launch(one, yes, no, no);
    } else {
        if (a.max_prefix) launch(one, no, yes, no);
        else if (w.direct) launch(one, no, no, yes);
        else launch(one, no, no, no);
    }
    const int jblocks = w.plan ? w.tblocks * (HD / 32) : 0;
    const long long items = w.direct ? (long long)w.dblocks * w.dr : (long long)a.nseq * per * a.nh;
    if (w.direct) {
        const dim3 jgrid((unsigned)(jblocks + std::max(div_up(items, 2), a.nseq)));
        attn_paged_join_kernel<HD, true, 2><<<jgrid, block, 0, s>>>(a, w, jblocks, per);
    } else if (items > 512) {
        attn_paged_join_kernel<HD, false, 2><<<dim3((unsigned)(jblocks + div_up(items, 2))), block, 0, s>>>(a, w, jblocks, per);
    } else {
        attn_paged_join_kernel<HD, false, 4><<<dim3((unsigned)(jblocks + items)), block, 0, s>>>(a, w, jblocks, per);
    }
}

hipError_t launch_attn_paged(const PagedAttn& a, hipStream_t s) {
    size_t n;
    const PagedWs w = plan(a, (uint8_t*)a.ws, &n);
    if (a.hd == 128) launch_t<128>(a, w, s);
    else launch_t<64>(a, w, s);
    return hipGetLastError();
}

}  // namespace strata
