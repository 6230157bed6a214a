// Log probabilities of given tokens with their ranks, the entropy and the likeliest tokens of rows of logits
// (strata_logits_logprobs). With M the largest logit of a row, S = sum e^(x - M) and W = sum e^(x - M) (x - M):
//   logp(v) = (x_v - M) - ln S,   entropy = ln S - W / S,   rank(v) = 1 + the tokens ordered before v,
// tokens ordered as argmax_key.h orders them (by value, the first of equals).
//
// One pass over the logits. A thread keeps its own running maximum and the two sums, in f32, rescaled when a tile of 16 of its
// values brings a larger maximum; a tile's terms are added as a tree. The K likeliest: a wave keeps a list in LDS of keys (value and
// index in 64 bits) above `thr`, its K-th best so far, and cuts it back to K when it is nearly full. The first tile starts from the
// K-th largest of the lanes' maxima (found bit by bit with ballots), which at least K values reach, so that hardly any value but
// the candidates enters the list; later tiles cost one comparison of a lane's maximum.
// A block takes a row where there are many, else a part of one, and a second launch joins the parts.
#include "argmax_key.h"
#include "attn_dev.h"
#include "branch.h"

#include <algorithm>

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
    // The list cut to its K largest keys, in descending order.
    __device__ void cut() {
        const int lane = threadIdx.x & 63;
        __builtin_amdgcn_wave_barrier();
        if (cnt <= 64) {
            const uint64_t key = lane < cnt ? buf[lane] : 0;
            int rank = 0;
            for (int i = 0; i < cnt; i++) {
                const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(key >> 32), i) << 32) | (uint32_t)__builtin_amdgcn_readlane((uint32_t)key, i);
                rank += o > key;
            }
            __builtin_amdgcn_wave_barrier();
            if (lane < cnt && rank < k) buf[rank] = key;
        } else {
            uint64_t key[LG_LIST / 64];
            int rank[LG_LIST / 64];
#pragma unroll
            for (int j = 0; j < LG_LIST / 64; j++) {
                key[j] = lane + 64 * j < cnt ? buf[lane + 64 * j] : 0;
                rank[j] = 0;
            }
            for (int i = 0; i < cnt; i++) {
                const uint64_t o = buf[i];
#pragma unroll
                for (int j = 0; j < LG_LIST / 64; j++) rank[j] += o > key[j];
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < LG_LIST / 64; j++)
                if (lane + 64 * j < cnt && rank[j] < k) buf[rank[j]] = key[j];
        }
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
    if (!a.k) return;
    // a key's place: its own list is sorted, of the others those that are larger
    const int w = tid >> 6, i = tid & 63;
    int all = 0;
    for (int u = 0; u < LG_W; u++) all += cnt[u];
    if (i < cnt[w]) {
        const uint64_t key = lists[w * LG_LIST + i];
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

// M: given tokens at most (0: no ranks). TOP: the likeliest are asked for.
template <int M, bool TOP>
__global__ __launch_bounds__(LG_T) void logprobs_kernel(Logprobs a, LgScratch f, int parts, int tiles) {
    __shared__ uint64_t lists[TOP ? LG_W * LG_LIST : 1];
    __shared__ LgSums ws[LG_W];
    __shared__ int wc[LG_W][M ? M : 1], cnt[LG_W], before[LOGP_MAX_IDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x / parts, part = blockIdx.x % parts;
    const float* x = a.x + (uint64_t)r * a.x_stride;
    // tiles of this part; chunk c of 4 values holds 4 c - off .. (the rows' chunks are 16-byte aligned wherever the row begins)
    const int off = (int)(((uintptr_t)x >> 2) & 3);
    const int t0 = (int)((long long)tiles * part / parts), t1 = (int)((long long)tiles * (part + 1) / parts);
    uint32_t lim[M ? M : 1];
    int id[M ? M : 1], n_before[M ? M : 1];
    auto order = [](float v) { return (uint32_t)(amax_key(v, 0) >> 32); };
    if constexpr (M > 0) {
#pragma unroll
        for (int i = 0; i < M; i++) {
            id[i] = i < a.m ? sload(a.ids + (uint64_t)r * a.m + i) : -1;
            lim[i] = id[i] >= 0 && id[i] < a.n ? order(sload(x + id[i])) : 0u;
            n_before[i] = 0;
        }
    }
    TopList top;
    if constexpr (TOP) top.init(lists + wave * LG_LIST, a.k);
    LgSums v{-INFINITY, 0.0f, 0.0f};
    float cur[LG_U][4], nxt[LG_U][4];
    auto load = [&](int t, float (&y)[LG_U][4]) {
#pragma unroll
        for (int u = 0; u < LG_U; u++) {
            const long long i = (long long)t * LG_TILE + 4 * (u * LG_T + tid) - off;
            if (i >= 0 && i + 4 <= a.n) {
                const float4 q = *(const float4*)(x + i);
                y[u][0] = q.x; y[u][1] = q.y; y[u][2] = q.z; y[u][3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) y[u][e] = i + e >= 0 && i + e < a.n ? x[i + e] : -INFINITY;
            }
        }
    };
    if (t0 < t1) load(t0, cur);
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
        float es[LG_U], ws4[LG_U];
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
            ws4[u] = (y4[0] + y4[1]) + (y4[2] + y4[3]);
        }
        v.s += (es[0] + es[1]) + (es[2] + es[3]);
        v.w += (ws4[0] + ws4[1]) + (ws4[2] + ws4[3]);
        const long long first = (long long)t * LG_TILE - off;  // the tile's first index
        const bool inner = first >= 0 && first + LG_TILE <= a.n;
        auto index = [&](int u, int e) { return first + 4 * (u * LG_T + tid) + e; };
        if constexpr (M > 0) {
#pragma unroll
            for (int i = 0; i < M; i++) {
                if (M > 1 && i >= a.m) continue;
                if (!inner || (id[i] >= first && id[i] < first + LG_TILE)) {  // a tile of the row's ends, or the token's own
#pragma unroll
                    for (int u = 0; u < LG_U; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const long long at = index(u, e);
                            const uint32_t o = order(cur[u][e]);
                            n_before[i] += at >= 0 && at < a.n && (o > lim[i] || (o == lim[i] && at < id[i]));
                        }
                } else {  // of equals, those of the tiles before the token's
                    const uint32_t from = lim[i] + (id[i] < first);
#pragma unroll
                    for (int u = 0; u < LG_U; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) n_before[i] += order(cur[u][e]) >= from;
                }
            }
        }
        if constexpr (TOP) {
            if (t == t0) {  // the K-th largest of the lanes' maxima
                const uint32_t o = order(mx);
                uint32_t bound = 0;
                for (int b = 31; b >= 0; b--) {
                    const uint32_t c = bound | (1u << b);
                    if (__popcll(__ballot(o >= c)) >= top.k) bound = c;
                }
                if (bound > order(-INFINITY)) top.set((uint64_t)bound << 32);  // (below, lanes without values may count among them)
            }
            if (t == t0 || top.thr == 0 || __ballot(!(mx <= top.quick) || v.s != v.s)) {
                uint32_t hit = 0;  // this lane's values that may count, a bit each
#pragma unroll
                for (int j = 0; j < 4 * LG_U; j++)
                    if (!(cur[j / 4][j % 4] < top.quick) && (inner || (index(j / 4, j % 4) >= 0 && index(j / 4, j % 4) < a.n))) hit |= 1u << j;
                while (__ballot(hit != 0)) {
                    const int b = hit ? __builtin_ctz(hit) : 0;
                    float x0 = cur[0][0];
#pragma unroll
                    for (int j = 1; j < 4 * LG_U; j++) x0 = b == j ? cur[j / 4][j % 4] : x0;
                    top.push(hit != 0, amax_key(x0, (int)index(b / 4, b % 4)));
                    hit &= hit - 1;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < LG_U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) cur[u][e] = nxt[u][e];
    }
    v = lg_wave(v);
    if constexpr (TOP) top.cut();
    if constexpr (M > 0) {
#pragma unroll
        for (int i = 0; i < M; i++) {
#pragma unroll
            for (int o = 32; o; o >>= 1) n_before[i] += __shfl_xor(n_before[i], o, 64);
            if (lane == 0) wc[wave][i] = n_before[i];
        }
    }
    if (lane == 0) {
        ws[wave] = v;
        cnt[wave] = TOP ? top.cnt : 0;
    }
    __syncthreads();
    v = ws[0];
    for (int w = 1; w < LG_W; w++) v = lg_join(v, ws[w]);
    if (M > 0 && tid < a.m) {
        int n = 0;
        for (int w = 0; w < LG_W; w++) n += wc[w][tid < M ? tid : 0];
        before[tid] = n;
    }
    if (parts == 1) return lg_finish(a, r, v, before, lists, cnt);
    const uint64_t at = (uint64_t)r * parts + part;
    if (tid == 0) f.sums[at] = v;
    if (M > 0 && tid < a.m) f.before[at * a.m + tid] = before[tid];
    if constexpr (TOP) {
        for (int i = tid; i < LG_W * 64; i += LG_T) {
            // the part's K best, in any order: key i of list w where its place is below K
            const int w = i >> 6, j = i & 63;
            if (j < cnt[w]) {
                const uint64_t key = lists[w * LG_LIST + j];
                int place = j;
                for (int u = 0; u < LG_W; u++) {
                    if (u == w) continue;
                    int lo = 0, hi = cnt[u];
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (lists[u * LG_LIST + mid] > key) lo = mid + 1;
                        else hi = mid;
                    }
                    place += lo;
                }
                if (place < a.k) f.keys[at * a.k + place] = key;
            }
        }
        const int all = cnt[0] + cnt[1] + cnt[2] + cnt[3];
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
    for (int i = wave; i < a.m; i += LG_W) {
        int n = 0;
        for (int p = lane; p < parts; p += 64) n += f.before[((uint64_t)r * parts + p) * a.m + i];
#pragma unroll
        for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o, 64);
        if (lane == 0) before[i] = n;
    }
    __syncthreads();
    v = ws[0];
    for (int w = 1; w < LG_W; w++) v = lg_join(v, ws[w]);
    lg_finish(a, r, v, before, lists, cnt);
}

// Tiles of a row (one more where the rows do not begin at a 16-byte border), and the parts of one: blocks enough for four a CU.
static int lg_tiles(const Logprobs& a) { return (int)(((long long)a.n + 3 + LG_TILE - 1) / LG_TILE); }
static int lg_parts(const Logprobs& a) { return (int)std::max(1, std::min<int>(lg_tiles(a), (1024 + a.rows - 1) / a.rows)); }
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
    const int m = a.rank ? a.m : 0;
    auto launch = [&](auto M) {
        if (a.k) logprobs_kernel<decltype(M)::value, true><<<grid, block, 0, s>>>(a, f, parts, tiles);
        else logprobs_kernel<decltype(M)::value, false><<<grid, block, 0, s>>>(a, f, parts, tiles);
    };
    if (m == 0) launch(std::integral_constant<int, 0>{});
    else if (m == 1) launch(std::integral_constant<int, 1>{});
    else if (m <= 4) launch(std::integral_constant<int, 4>{});
    else launch(std::integral_constant<int, LOGP_MAX_IDS>{});
    if (parts > 1) logprobs_join_kernel<<<dim3((unsigned)a.rows), block, 0, s>>>(a, f, parts);
    return hipGetLastError();
}

}  // namespace strata
