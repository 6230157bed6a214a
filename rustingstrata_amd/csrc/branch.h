// Launchers of the operators for drafted trees and branching sequences over a paged f16 KV cache (tree.hip: positions, ancestor
// masks and the path that the choices confirm; branch.hip: sequences that go on from others, rows of the caches; logprobs.hip:
// log probabilities; attn_tree.hip: attention). Arguments are checked in api.hip.
#pragma once
#include "serve.h"

namespace strata {

// Words of a row's ancestor mask at most: trees of up to 256 nodes.
constexpr int TREE_MAX_WORDS = 8;

// A step's trees (strata_tree_step).
struct TreeStep {
    int nseq = 0; const int* q_start = nullptr; const int* parent = nullptr; const int* len = nullptr; const int* prefix_len = nullptr;
    int t = 0, words = 0; int* pos = nullptr; uint32_t* mask = nullptr; int* err = nullptr;
};
hipError_t launch_tree_step(const TreeStep& a, hipStream_t s);

// The confirmed paths (strata_tree_accept).
struct TreeAccept {
    int nseq = 0; const int* q_start = nullptr; const int* parent = nullptr; const int* tokens = nullptr; const int* ids = nullptr;
    const int* len = nullptr; const int* slots = nullptr; int t = 0, words = 0, max_path = 0;
    int* n_path = nullptr; int* chosen = nullptr; int* last = nullptr; int* keep = nullptr; int* runs = nullptr;
};
hipError_t launch_tree_accept(const TreeAccept& a, hipStream_t s);

// Sequences that go on from others (strata_kv_pages_fork). scratch: pages_fork_scratch_bytes() bytes.
struct PagesFork {
    int nseq = 0; const int* src = nullptr; const int* keep = nullptr; const int* len = nullptr;
    int* tables = nullptr; int max_pages = 0, page_shift = 0;
    int* free_pages = nullptr; int n_pages = 0; const int* n_free = nullptr; int* refs = nullptr;
    int* len_out = nullptr; int* n_free_out = nullptr; int* runs = nullptr; int* err = nullptr; void* scratch = nullptr;
};
size_t pages_fork_scratch_bytes(const PagesFork& a);
hipError_t launch_pages_fork(const PagesFork& a, hipStream_t s);

// Rows of the caches from slot to slot (strata_kv_rows_move).
struct RowsMove {
    const uint64_t* caches = nullptr; int n_caches = 0; uint64_t row_bytes = 0; uint64_t n_slots = 0;
    const int* runs = nullptr; int groups = 0, per = 0;
};
hipError_t launch_rows_move(const RowsMove& a, hipStream_t s);

// Log probabilities (strata_logits_logprobs). scratch: logprobs_scratch_bytes() bytes.
constexpr int LOGP_MAX_TOP = 64, LOGP_MAX_IDS = 16;
struct Logprobs {
    const float* x = nullptr; uint64_t x_stride = 0; int n = 0, rows = 0;
    const int* ids = nullptr; int m = 0; float* logp = nullptr; int* rank = nullptr; float* entropy = nullptr;
    int k = 0; int* top_ids = nullptr; float* top_logp = nullptr; void* scratch = nullptr;
};
size_t logprobs_scratch_bytes(const Logprobs& a);
hipError_t launch_logprobs(const Logprobs& a, hipStream_t s);

// Attention of drafted trees (strata_attn_paged_tree): paged attention with an ancestor mask of `words` words a row.
size_t tree_attn_ws_bytes(const PagedAttn& a);
hipError_t launch_attn_tree(const PagedAttn& a, hipStream_t s);

}  // namespace strata
