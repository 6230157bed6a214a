// Device pieces that the attention kernels share (attn.hip: one sequence's contiguous cache; attn_paged.hip: a batch over
// pages): fragment types, wave reductions, the softmax's exp2, the f16 splits of queries and weights.
#pragma once
#include "xlane.h"

namespace strata {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float h2f(uint16_t b) {
    _Float16 h;
    __builtin_memcpy(&h, &b, 2);
    return (float)h;
}
__device__ __forceinline__ float sigmoid_f(float x) { return 1.0f / (1.0f + expf(-x)); }

// Maximum and sum over the 64 lanes of a wave, returned to every lane: DPP and swizzle steps within each half, then
// the two halves' results through scalar lane reads (no LDS round trip per step).
__device__ __forceinline__ float wave_max64(float v) {
    v = fmaxf(v, xl32f<0>(v));
    v = fmaxf(v, xl32f<1>(v));
    v = fmaxf(v, xl32f<2>(v));
    v = fmaxf(v, xl32f<3>(v));
    v = fmaxf(v, xl32f<4>(v));
    return fmaxf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0)),
                 __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32)));
}
__device__ __forceinline__ float wave_sum64(float v) {
    v += xl32f<0>(v);
    v += xl32f<1>(v);
    v += xl32f<2>(v);
    v += xl32f<3>(v);
    v += xl32f<4>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0)) +
           __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32));
}

// 2^x by the hardware's v_exp_f32 (within 1 ulp; 2^-inf = 0). The softmaxes work in log2 units: scores times log2(e)
// (one rounding, relative 2^-24 of the exponent, so about |s| 2^-24 ln 2 of each weight: ~1e-7 for the scores that
// carry the weight), then exp2 of the difference from the running maximum.
constexpr float LOG2E = 1.44269504088896341f;
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

constexpr int DEC_WAVES = 4;  // of a block over few rows

typedef float f16v __attribute__((ext_vector_type(16)));

// A query head, whose largest magnitude is mx, goes to f16 hi and lo parts times `up`, the power of two that puts mx in [2^13,
// 2^14), so that the lo parts stay normal numbers; usc undoes it, times `scale` and log2(e). Below 2^-112 `up` stays at 2^126, as
// 2^127 is the last that float32 has (2^(14 - ex) was infinite for heads below 2^-114, their scores not numbers).
__device__ __forceinline__ void query_scale(float mx, float scale, float& up, float& usc) {
    const int e = max((int)(__float_as_uint(mx) >> 23), 14);  // 2^(e - 127) <= mx, which is not below 0
    up = __uint_as_float((uint32_t)(267 - e) << 23);
    usc = scale * LOG2E * __uint_as_float((uint32_t)(e - 13) << 23);
}
// usc is kept at this at least (for a scale not below 0), so that a masked score of -inf stays one times usc. A score s of the
// scaled parts is below 2^37: with usc at this or less its exp2 is 1.
constexpr float USC_MIN = 0x1p-126f;

// Eight softmax weights p (at most 2) times PF_SCALE as f16 hi and lo parts for the P V MFMA: hi = f16(p c), lo the exact
// remainder p c - hi rounded likewise, both to nearest, so hi + lo carries each weight to 2^-22 of its value and the lo
// parts stay normal f16 numbers for weights down to 2^-17. (2^14 is the largest scale that p = 2 leaves in f16, hence the
// lag of 1: with a lag of 3 and 2^11, rows of weights around 2^-18 beside one of 1 were 1.4e-6 off, 7e-6 around 2^-20; the
// time is the same.) Written so that the compiler selects the mixed-precision multiply-adds, which scale, round and read
// the f16 halves in place (and keeps the wait states between them, the exps before and the MFMAs after, as it could not
// for inline assembly).
constexpr float PF_SCALE = 16384.0f;
__device__ __forceinline__ void split_w8(const float* p, h8& hi, h8& lo) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        hi[e] = (_Float16)__builtin_fmaf(p[e], PF_SCALE, 0.0f);
        lo[e] = (_Float16)__builtin_fmaf(p[e], PF_SCALE, -(float)hi[e]);
    }
}
// The larger of this lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

}  // namespace strata
