// Paged attention of drafted trees (strata_attn_paged_tree): attn_paged.h holds the kernels.
#include "attn_paged.h"
#include "branch.h"

namespace strata {

size_t tree_attn_ws_bytes(const PagedAttn& a) {
    size_t n;
    plan(a, nullptr, &n);
    return n;
}
hipError_t launch_attn_tree(const PagedAttn& a, hipStream_t s) { return launch_paged<true>(a, s); }

}  // namespace strata
