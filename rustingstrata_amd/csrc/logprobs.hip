// Log probabilities of given tokens with their ranks, the entropy and the likeliest tokens of rows of logits
// (strata_logits_logprobs). With M the largest logit of a row, S = sum e^(x - M) and W = sum e^(x - M) (x - M):
//   logp(v) = (x_v - M) - ln S,   entropy = ln S - W / S,   rank(v) = 1 + the tokens ordered before v,
// tokens ordered as argmax_key.h orders them (by value, the first of equals).
//
// One pass over the logits, bound by their bytes: 1001 rows of 151936, a given token and 20 alternatives 122 us, 5.0 TB/s. A thread keeps
// its own running maximum and the two sums, in f32, rescaled when a tile of 16 of its values brings a larger maximum; a tile's
// terms are added as a tree. The K likeliest: a wave keeps a list in LDS of keys (value and index in 64 bits) above `thr`, below
// which no key is among the block's K best. The first tile starts from a bound that K of its values reach: of each wave's lanes'
// maxima the largest K / 4 (found bit by bit with ballots; its upper 18 bits are bound enough), of those the least. After 1, 2, 4, ..
// tiles the waves agree on the K best of all their lists, so that of a row's 37 tiles about a third bring a wave a candidate; a
// wave's list of its own K best alone let 30 of them through. A tile without one costs a comparison of the lane's maximum.
// A block takes a row where there are many, else a part of one, and a second launch joins the parts: one row 15 us replayed, the
// chain of a tile's loads, its bound and its list (9), then the join's (5).
#include "argmax_key.h"
#include "attn_dev.h"
#include "branch.h"

#include <algorithm>
#include <climits>

namespace strata {

constexpr int LG_T = 256, LG_W = LG_T / 64, LG_U = 4, LG_TILE = LG_T * 4 * LG_U, LG_LIST = 256;

__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
}

// A wave's list of candidates in LDS.
struct TopList {
    uint64_t* buf;      // LG_LIST keys
    int k, cnt;         // the same in all lanes
    uint64_t thr;       // keys up to it do not count
    float quick;        // values below it do not either, nor later ones up to it once K are in the list
    __device__ __forceinline__ void init(uint64_t* b, int top) {
        buf = b;
        k = top;
        cnt = 0;
        thr = 0;
        quick = -INFINITY;
    }
    __device__ __forceinline__ void set(uint64_t t) {
        thr = t;
        const uint32_t u = (uint32_t)(t >> 32) ^ 0x80000000u;
        const float v = __uint_as_float(u ^ ((uint32_t)((int32_t)u >> 31) >> 1));
        quick = v == 0.0f ? -0x1p-149f : v;  // (of the two zeros one is the larger key)
    }
    // The list cut to its K largest keys, in descending order: a key's place is the number of larger ones. Of more than 64 the bound
    // that K of them reach first, bit by bit (by the values' words; by the indices' too where many are equal).
    __device__ __forceinline__ void cut() {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_wave_barrier();
        if (cnt > 64) {
            constexpr int J = LG_LIST / 64;
            uint32_t hi[J], lo[J];
#pragma unroll
            for (int j = 0; j < J; j++) {
                const uint64_t key = lane + 64 * j < cnt ? buf[lane + 64 * j] : 0;
                hi[j] = (uint32_t)(key >> 32);
                lo[j] = (uint32_t)key;
            }
            uint32_t bh = 0, bl = 0;
            for (int b = 31; b >= 0; b--) {
                const uint32_t c = bh | (1u << b);
                int n = 0;
#pragma unroll
                for (int j = 0; j < J; j++) n += __popcll(__ballot(hi[j] >= c));
                if (n >= k) bh = c;
            }
            int above = 0, equal = 0;
#pragma unroll
            for (int j = 0; j < J; j++) {
                above += __popcll(__ballot(hi[j] > bh));
                equal += __popcll(__ballot(hi[j] == bh));
            }
            if (above + equal > 64)
                for (int b = 31; b >= 0; b--) {
                    const uint32_t c = bl | (1u << b);
                    int n = above;
#pragma unroll
                    for (int j = 0; j < J; j++) n += __popcll(__ballot(hi[j] == bh && lo[j] >= c));
                    if (n >= k) bl = c;
                }
            int n = 0;
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < J; j++) {
                const bool stays = hi[j] > bh || (hi[j] == bh && lo[j] >= bl && lane + 64 * j < cnt);
                const uint64_t m = __ballot(stays);
                if (stays) buf[n + __popcll(m & ((1ull << lane) - 1))] = ((uint64_t)hi[j] << 32) | lo[j];
                n += __popcll(m);
            }
            __builtin_amdgcn_wave_barrier();
            cnt = n;
        }
        const uint64_t key = lane < cnt ? buf[lane] : 0;
        int place = 0;
#pragma unroll 8
        for (int i = 0; i < cnt; i++) place += buf[i] > key;
        __builtin_amdgcn_wave_barrier();
        if (lane < cnt && place < k) buf[place] = key;
        __builtin_amdgcn_wave_barrier();
        if (cnt >= k) {
            cnt = k;
            set(uniform64(buf[k - 1]));
        }
    }
    // Keys of the lanes that have one.
    __device__ __forceinline__ void push(bool has, uint64_t key) {
        has = has && key > thr;
        const uint64_t b = __ballot(has);
        if (!b) return;
        if (has) buf[cnt + __popcll(b & ((1ull << (threadIdx.x & 63)) - 1))] = key;
        cnt += __popcll(b);
        if (cnt > LG_LIST - 64) cut();
    }
};

// The place of key i of wave w's list (sorted, as all are; cnt[u] keys of list u) among all lists' keys.
__device__ __forceinline__ int lg_place(const uint64_t* lists, const int* cnt, int w, int i, uint64_t key) {
    int place = i;
    for (int u = 0; u < LG_W; u++) {
        if (u == w) continue;
        int lo = 0, hi = cnt[u];  // keys of list u before lo are larger
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (lists[u * LG_LIST + mid] > key) lo = mid + 1;
            else hi = mid;
        }
        place += lo;
    }
    return place;
}
// The waves' lists cut to the K best of all of them together, and the bound that follows. shared: a word that the call before did not
// use (a wave may still read that one when this call clears its own; of the call before it, the barriers between have all waves past).
__device__ __forceinline__ void lg_agree(TopList& top, const uint64_t* lists, int* cnt, uint64_t* shared) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    top.cut();
    if (lane == 0) cnt[wave] = top.cnt;
    if (threadIdx.x == 0) *shared = 0;
    __syncthreads();
    const uint64_t key = lane < top.cnt ? lists[wave * LG_LIST + lane] : 0;
    const int place = lane < top.cnt ? lg_place(lists, cnt, wave, lane, key) : INT_MAX;
    if (place == top.k - 1) *shared = key;
    top.cnt = __popcll(__ballot(place < top.k));
    __syncthreads();
    const uint64_t bound = uniform64(*shared);
    if (bound > top.thr) top.set(bound);
}

// The sums of a row or of a part of it.
struct LgSums {
    float m, s, w;
};
// a and b together.
__device__ __forceinline__ LgSums lg_join(const LgSums& a, const LgSums& b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return LgSums{m, a.s + b.s, a.w + b.w};  // (nothing, or not a number)
    const float da = fmaxf(a.m - m, -200.0f), db = fmaxf(b.m - m, -200.0f);  // (e^-200 is 0 here)
    const float fa = exp2_hw(da * LOG2E), fb = exp2_hw(db * LOG2E);
    return LgSums{m, a.s * fa + b.s * fb, (a.w + da * a.s) * fa + (b.w + db * b.s) * fb};
}
__device__ __forceinline__ LgSums lg_wave(LgSums v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = lg_join(v, LgSums{__shfl_xor(v.m, o, 64), __shfl_xor(v.s, o, 64), __shfl_xor(v.w, o, 64)});
    return v;
}

// The scratch of rows in parts.
struct LgScratch {
    LgSums* sums;     // [rows][parts]
    int* before;      // [rows][parts][m]
    uint64_t* keys;   // [rows][parts][k]
};
static inline LgScratch lg_scratch(const Logprobs& a, int parts, size_t* bytes) {
    LgScratch f;
    size_t o = 0;
    auto take = [&](size_t n) {
        void* p = (uint8_t*)a.scratch + o;
        o += (n + 255) & ~(size_t)255;
        return p;
    };
    f.sums = (LgSums*)take((size_t)a.rows * parts * sizeof(LgSums));
    f.before = (int*)take((size_t)a.rows * parts * a.m * sizeof(int));
    f.keys = (uint64_t*)take((size_t)a.rows * parts * a.k * sizeof(uint64_t));
    if (bytes) *bytes = o;
    return f;
}

// What a row gives, by a block: v its sums (in all threads), before[i] the tokens ordered before given token i, lists the waves'
// K best (LDS, [LG_W][LG_LIST], cnt[w] of them).
template <bool TOP>
__device__ __forceinline__ void lg_finish(const Logprobs& a, int r, const LgSums& v, const int* before, const uint64_t* lists, const int* cnt) {
    const int tid = threadIdx.x;
    const float ls = logf(v.s);
    auto logp = [&](float x) { return v.s == 0.0f ? -INFINITY : (x - v.m) - ls; };
    if (tid < a.m) {
        const int id = a.ids[(uint64_t)r * a.m + tid];
        const bool in = id >= 0 && id < a.n;
        if (a.logp) a.logp[(uint64_t)r * a.m + tid] = in ? logp(a.x[(uint64_t)r * a.x_stride + id]) : -INFINITY;
        if (a.rank) a.rank[(uint64_t)r * a.m + tid] = in ? before[tid] + 1 : 0;
    }
    if (tid == 0 && a.entropy) a.entropy[r] = v.s == 0.0f ? 0.0f : ls - v.w / v.s;
    if constexpr (!TOP) return;
    // a key's place: its own list is sorted, of the others those that are larger
    const int w = tid >> 6, i = tid & 63;
    int all = 0;
    for (int u = 0; u < LG_W; u++) all += cnt[u];
    if (i < cnt[w]) {
        const uint64_t key = lists[w * LG_LIST + i];
        const int place = lg_place(lists, cnt, w, i, key);
        if (place < a.k) {
            const int id = (int)(0xFFFFFFFFu - (uint32_t)key);
            if (a.top_ids) a.top_ids[(uint64_t)r * a.k + place] = id;
            if (a.top_logp) a.top_logp[(uint64_t)r * a.k + place] = logp(a.x[(uint64_t)r * a.x_stride + id]);
        }
    }
    if (tid < a.k && tid >= all) {  // a row of fewer tokens
        if (a.top_ids) a.top_ids[(uint64_t)r * a.k + tid] = -1;
        if (a.top_logp) a.top_logp[(uint64_t)r * a.k + tid] = -INFINITY;
    }
}

// RANK: ranks are asked for, TOP: the likeliest are. A given token's rank takes a comparison a value, whose ballots are counted on
// the scalar unit, but for a wave's tiles without a value as large (1001 rows, four tokens: among the ten likeliest 136 us, without
// that rule 168; any four 175 and 174).
template <bool RANK, bool TOP>
__global__ __launch_bounds__(LG_T, 4) void logprobs_kernel(Logprobs a, LgScratch f, int parts, int tiles) {
    __shared__ uint64_t lists[TOP ? LG_W * LG_LIST : 1], shared[2];
    __shared__ LgSums ws[LG_W];
    __shared__ uint32_t wb[LG_W], lim[LOGP_MAX_IDS];
    __shared__ int cnt[LG_W], before[LOGP_MAX_IDS], ids[LOGP_MAX_IDS];
    __shared__ float val[LOGP_MAX_IDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x / parts, part = blockIdx.x % parts;
    const float* x = a.x + (uint64_t)r * a.x_stride;
    // tiles of this part; a tile's chunks of 4 values are 16-byte aligned wherever the row begins: the first tile begins `off` values
    // before it. Values outside the row are -inf.
    const int off = (int)(((uintptr_t)x >> 2) & 3);
    const int t0 = (int)((long long)tiles * part / parts), t1 = (int)((long long)tiles * (part + 1) / parts);
    auto order = [](float v) { return (uint32_t)(amax_key(v, 0) >> 32); };
    const uint32_t none = order(-INFINITY);
    if (RANK && tid < LOGP_MAX_IDS) {
        const int id = tid < a.m ? a.ids[(uint64_t)r * a.m + tid] : -1;
        ids[tid] = id;
        val[tid] = id >= 0 && id < a.n ? x[id] : 0.0f;
        lim[tid] = order(val[tid]);
        before[tid] = 0;
    }
    TopList top;
    if constexpr (TOP) top.init(lists + wave * LG_LIST, a.k);
    LgSums v{-INFINITY, 0.0f, 0.0f};
    float cur[LG_U][4], nxt[LG_U][4];
    auto load = [&](int t, float (&y)[LG_U][4]) __attribute__((always_inline)) {
        const long long first = (long long)t * LG_TILE - off;
        if (first >= 0 && first + LG_TILE <= a.n) {
#pragma unroll
            for (int u = 0; u < LG_U; u++) {
                const float4 q = *(const float4*)(x + first + 4 * (u * LG_T + tid));
                y[u][0] = q.x; y[u][1] = q.y; y[u][2] = q.z; y[u][3] = q.w;
            }
        } else {
#pragma unroll
            for (int u = 0; u < LG_U; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const long long i = first + 4 * (u * LG_T + tid) + e;
                    y[u][e] = i >= 0 && i < a.n ? x[i] : -INFINITY;
                }
        }
    };
    if (t0 < t1) load(t0, cur);
    int id0 = 0, n0 = 0;  // the first given token, in scalar registers
    uint32_t lim0 = 0;
    float val0 = 0.0f;
    if constexpr (RANK) {
        __syncthreads();
        id0 = __builtin_amdgcn_readfirstlane(ids[0]);
        lim0 = __builtin_amdgcn_readfirstlane(lim[0]);
        val0 = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(val[0])));
    }
    for (int t = t0; t < t1; t++) {
        if (t + 1 < t1) load(t + 1, nxt);
        float mx = cur[0][0];
#pragma unroll
        for (int u = 0; u < LG_U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) mx = fmaxf(mx, cur[u][e]);
        if (mx > v.m) {
            const float d = fmaxf(v.m - mx, -200.0f), c = exp2_hw(d * LOG2E);  // (the sums before the first value are 0)
            v.w = (v.w + d * v.s) * c;
            v.s *= c;
            v.m = mx;
        }
        const float ref = v.m == -INFINITY ? 0.0f : v.m;
        float es[LG_U], ys[LG_U];
#pragma unroll
        for (int u = 0; u < LG_U; u++) {
            float e4[4], y4[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float y = cur[u][e] - ref;
                e4[e] = exp2_hw(y * LOG2E);  // (0 of -inf; not a number stays one)
                y4[e] = e4[e] * fmaxf(y, -200.0f);
            }
            es[u] = (e4[0] + e4[1]) + (e4[2] + e4[3]);
            ys[u] = (y4[0] + y4[1]) + (y4[2] + y4[3]);
        }
        v.s += (es[0] + es[1]) + (es[2] + es[3]);
        v.w += (ys[0] + ys[1]) + (ys[2] + ys[3]);
        const long long first = (long long)t * LG_TILE - off;  // the tile's first index
        if constexpr (RANK) {
            const bool odd = __ballot(v.s != v.s);  // (there may be values that are no numbers)
            // this wave's values of the tile that come before token id of key l and value y
            auto count = [&](int id, uint32_t l, float y) __attribute__((always_inline)) {
                int n = 0;
                if (id >= first && id < first + LG_TILE) {  // its own tile: of equals those before it
                    const int at = (int)(id - first) - 4 * tid;
#pragma unroll
                    for (int u = 0; u < LG_U; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint32_t o = order(cur[u][e]);
                            n += __popcll(__ballot(o > l || (o == l && 4 * LG_T * u + e < at)));
                        }
                } else if (odd || y == 0.0f || !(y > -INFINITY)) {
                    // (keys >= from; the largest key, a NaN's, has none above it to count from)
                    const uint32_t from = l + (id < first);
                    if (from >= l) {
#pragma unroll
                        for (int u = 0; u < LG_U; u++)
#pragma unroll
                            for (int e = 0; e < 4; e++) n += __popcll(__ballot(order(cur[u][e]) >= from));
                    }
                } else if (!__ballot(mx >= y)) {  // (a likely token: nothing of most tiles comes before it)
                } else if (id < first) {  // (other numbers compare as their keys do)
#pragma unroll
                    for (int u = 0; u < LG_U; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) n += __popcll(__ballot(cur[u][e] > y));
                } else {
#pragma unroll
                    for (int u = 0; u < LG_U; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) n += __popcll(__ballot(cur[u][e] >= y));
                }
                return n;
            };
            n0 += count(id0, lim0, val0);
            for (int i = 1; i < a.m; i++) {
                const int id = __builtin_amdgcn_readfirstlane(ids[i]);
                const uint32_t l = __builtin_amdgcn_readfirstlane(lim[i]);
                const int n = count(id, l, __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(val[i]))));
                if (lane == 0 && n) atomicAdd(&before[i], n);
            }
        }
        if constexpr (TOP) {
            if (t == t0) {  // of each wave's lanes' maxima the largest K / 4: the least of those is a bound that K values reach
                const uint32_t o = order(mx);
                auto reached = [&](int k) {  // the largest key that k of the wave's lanes reach (its upper bits)
                    uint32_t bound = 0;
                    for (int b = 31; b >= 14; b--) {
                        const uint32_t c = bound | (1u << b);
                        if (__popcll(__ballot(o >= c)) >= k) bound = c;
                    }
                    return bound;
                };
                uint32_t bound = reached((top.k + LG_W - 1) / LG_W);
                if (lane == 0) wb[wave] = bound;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < LG_W; w++) bound = min(bound, wb[w]);
                bound = __builtin_amdgcn_readfirstlane(bound);
                if (bound <= none) bound = reached(top.k);  // (a short tile, which leaves some waves without values)
                if (bound > none) top.set((uint64_t)bound << 32);  // (below, lanes without values may count among them)
            }
            if (t == t0 || top.thr == 0 || __ballot(!(mx <= top.quick) || v.s != v.s)) {
                uint32_t hit = 0;  // this lane's values that may count, a bit each
#pragma unroll
                for (int j = 0; j < 4 * LG_U; j++)
                    if (!(cur[j / 4][j % 4] < top.quick)) hit |= 1u << j;
                while (__ballot(hit != 0)) {
                    const int b = hit ? __builtin_ctz(hit) : 0;
                    const long long at = first + 4 * ((b >> 2) * LG_T + tid) + (b & 3);
                    float x0 = cur[0][0];
#pragma unroll
                    for (int j = 1; j < 4 * LG_U; j++) x0 = b == j ? cur[j / 4][j % 4] : x0;
                    top.push(hit != 0 && at >= 0 && at < a.n, amax_key(x0, (int)at));
                    hit &= hit - 1;
                }
            }
            if (((t - t0 + 1) & (t - t0)) == 0 && t + 1 < t1)  // after 1, 2, 4, .. tiles, the words in turn
                lg_agree(top, lists, cnt, shared + (__builtin_ctz(t - t0 + 1) & 1));
        }
#pragma unroll
        for (int u = 0; u < LG_U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) cur[u][e] = nxt[u][e];
    }
    v = lg_wave(v);
    if constexpr (TOP) top.cut();
    if (lane == 0) {
        if (RANK && n0) atomicAdd(&before[0], n0);
        ws[wave] = v;
        if constexpr (TOP) cnt[wave] = top.cnt;
    }
    __syncthreads();
    v = ws[0];
    for (int w = 1; w < LG_W; w++) v = lg_join(v, ws[w]);
    if (RANK && tid < a.m) {
        // values outside the row are not before anything
        if (t0 == 0 && none >= lim[tid] + (ids[tid] < 0)) before[tid] -= off;
        if (t1 == tiles && none > lim[tid]) before[tid] -= (int)((long long)tiles * LG_TILE - off - a.n);
    }
    if (parts == 1) {
        lg_finish<TOP>(a, r, v, before, lists, cnt);
        return;
    }
    const uint64_t at = (uint64_t)r * parts + part;
    if (tid == 0) f.sums[at] = v;
    if (RANK && tid < a.m) f.before[at * a.m + tid] = before[tid];
    if constexpr (TOP) {
        // the part's K best, in any order
        const int all = cnt[0] + cnt[1] + cnt[2] + cnt[3];
        if (lane < cnt[wave]) {
            const uint64_t key = lists[wave * LG_LIST + lane];
            const int place = lg_place(lists, cnt, wave, lane, key);
            if (place < a.k) f.keys[at * a.k + place] = key;
        }
        if (tid < a.k && tid >= all) f.keys[at * a.k + tid] = 0;
    }
}

// The parts of a row, by a block.
__global__ __launch_bounds__(LG_T) void logprobs_join_kernel(Logprobs a, LgScratch f, int parts) {
    __shared__ uint64_t lists[LG_W * LG_LIST];
    __shared__ LgSums ws[LG_W];
    __shared__ int cnt[LG_W], before[LOGP_MAX_IDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = blockIdx.x;
    LgSums v{-INFINITY, 0.0f, 0.0f};
    for (int i = tid; i < parts; i += LG_T) v = lg_join(v, f.sums[(uint64_t)r * parts + i]);
    v = lg_wave(v);
    TopList top;
    if (a.k) {
        top.init(lists + wave * LG_LIST, a.k);
        const int n = parts * a.k;
        for (int i0 = 64 * wave; i0 < n; i0 += LG_T) {
            const uint64_t key = i0 + lane < n ? f.keys[(uint64_t)r * n + i0 + lane] : 0;
            top.push(key != 0, key);
        }
        top.cut();
    }
    if (lane == 0) {
        ws[wave] = v;
        cnt[wave] = a.k ? top.cnt : 0;
    }
    for (int i = wave; a.rank && i < a.m; i += LG_W) {
        int n = 0;
        for (int p = lane; p < parts; p += 64) n += f.before[((uint64_t)r * parts + p) * a.m + i];
#pragma unroll
        for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o, 64);
        if (lane == 0) before[i] = n;
    }
    __syncthreads();
    v = ws[0];
    for (int w = 1; w < LG_W; w++) v = lg_join(v, ws[w]);
    if (a.k) lg_finish<true>(a, r, v, before, lists, cnt);
    else lg_finish<false>(a, r, v, before, lists, cnt);
}

// Tiles of a row (one more where the rows do not begin at a 16-byte border), and the parts of one: blocks for four a CU, as many as run
// at once (1001 rows in one part each 122 us, in two 165).
static int lg_tiles(const Logprobs& a) { return (int)(((long long)a.n + 3 + LG_TILE - 1) / LG_TILE); }
static int lg_parts(const Logprobs& a) { return (int)std::max(1, std::min<int>(lg_tiles(a), 1024 / a.rows)); }
size_t logprobs_scratch_bytes(const Logprobs& a) {
    const int parts = lg_parts(a);
    if (parts == 1) return 0;
    size_t n;
    lg_scratch(a, parts, &n);
    return n;
}
hipError_t launch_logprobs(const Logprobs& a, hipStream_t s) {
    const int parts = lg_parts(a), tiles = lg_tiles(a);
    const LgScratch f = lg_scratch(a, parts, nullptr);
    const dim3 grid((unsigned)((long long)a.rows * parts)), block(LG_T);
    if (a.rank && a.m) {
        if (a.k) logprobs_kernel<true, true><<<grid, block, 0, s>>>(a, f, parts, tiles);
        else logprobs_kernel<true, false><<<grid, block, 0, s>>>(a, f, parts, tiles);
    } else {
        if (a.k) logprobs_kernel<false, true><<<grid, block, 0, s>>>(a, f, parts, tiles);
        else logprobs_kernel<false, false><<<grid, block, 0, s>>>(a, f, parts, tiles);
    }
    if (parts > 1) logprobs_join_kernel<<<dim3((unsigned)a.rows), block, 0, s>>>(a, f, parts);
    return hipGetLastError();
}

}  // namespace strata
