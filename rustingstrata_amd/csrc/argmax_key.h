// ops::argmax's order (src/ops.rs:110-112): the largest value under f32::total_cmp, the first index on ties. A value
// and its index pack into one 64-bit key whose unsigned maximum is that choice: the total-order image of the bits
// above, ~index below.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace strata {

__device__ __forceinline__ uint64_t amax_key(float v, int i) {
    const int32_t b = __float_as_int(v);
    const uint32_t u = (uint32_t)(b ^ (int32_t)((uint32_t)(b >> 31) >> 1)) ^ 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t k) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)k, o, 64), hi = __shfl_xor((uint32_t)(k >> 32), o, 64);
        const uint64_t other = ((uint64_t)hi << 32) | lo;
        k = other > k ? other : k;
    }
    return k;
}

}  // namespace strata
