// Launchers of the operators that serve a batch of sequences over a paged f16 KV cache (serve.hip: page tables and slot
// maps, penalties, biases and masks on logits; attn_paged.hip: attention). Arguments are checked in api.hip.
#pragma once
#include "common.h"

namespace strata {

// Sequences a call takes: their prefix sums sit in a block's LDS.
constexpr int SERVE_MAX_SEQ = 4096;

// One step of the page tables (strata_kv_pages_step). scratch: pages_scratch_bytes(nseq) bytes.
struct PagesStep {
    int nseq = 0; const int* add = nullptr; const int* len = nullptr;
    int* tables = nullptr; int max_pages = 0, page_shift = 0;
    int* free_pages = nullptr; int n_pages = 0; const int* n_free = nullptr; const int* prefix_len = nullptr;
    int t_max = 0; int* q_start = nullptr; int* pos = nullptr; int* slots = nullptr;
    int* len_out = nullptr; int* n_free_out = nullptr; int* err = nullptr; int* scratch = nullptr;
};
size_t pages_scratch_bytes(int nseq);
hipError_t launch_pages_step(const PagesStep& a, hipStream_t s);

// Penalties, biases and masks on rows of logits (strata_logits_process). keys: logits_key_bytes(n, rows) bytes of scratch
// (when ids is given).
struct LogitsProcess {
    const float* x = nullptr; uint64_t x_stride = 0; float* out = nullptr; uint64_t out_stride = 0; int n = 0, rows = 0;
    int* hist = nullptr; uint64_t hist_stride = 0; int* hist_len = nullptr; const int* hist_from = nullptr; int last = 0;
    const float* pen = nullptr;
    const int* bias_start = nullptr; const int* bias_ids = nullptr; const float* bias_vals = nullptr; int n_bias = 0;
    const uint32_t* mask = nullptr; uint64_t mask_stride = 0;
    int* ids = nullptr; int append = 0; uint64_t* keys = nullptr;
};
size_t logits_key_bytes(int n, int rows);
hipError_t launch_logits_process(const LogitsProcess& a, hipStream_t s);

// Positions of a prefix and a sequence's own keys behind it: the attention numbers both in one int32 list, with up to 63 places
// between them and a tile and a wave's step past its end.
constexpr uint64_t PAGED_ATTN_KEYS = (1ull << 31) - 1024;

// Attention of a ragged batch over pages (strata_attn_paged). ws: paged_attn_ws_bytes() bytes of workspace.
struct PagedAttn {
    const float* q = nullptr; const uint16_t* kc = nullptr; const uint16_t* vc = nullptr; const float* qg = nullptr;
    float* out = nullptr;
    int t = 0, max_q = 0; const int* pos = nullptr; const int* q_start = nullptr; const int* len = nullptr; int nseq = 0;
    const int* tables = nullptr; int max_pages = 0, page_shift = 0, n_pages = 0;
    const int* prefix = nullptr; const int* prefix_len = nullptr; int max_prefix = 0;
    int nh = 0, nkv = 0, hd = 0; float scale = 0; const float* sink = nullptr; int win = 0;
    void* ws = nullptr;
};
size_t paged_attn_ws_bytes(const PagedAttn& a);
hipError_t launch_attn_paged(const PagedAttn& a, hipStream_t s);

}  // namespace strata
