// Paged attention of lines of tokens (strata_attn_paged): attn_paged.h holds the kernels.
#include "attn_paged.h"

namespace strata {

size_t paged_attn_ws_bytes(const PagedAttn& a) {
    size_t n;
    plan(a, nullptr, &n);
    return n;
}
hipError_t launch_attn_paged(const PagedAttn& a, hipStream_t s) { return launch_paged<false>(a, s); }

}  // namespace strata
