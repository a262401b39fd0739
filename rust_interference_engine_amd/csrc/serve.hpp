// serve.hpp — arguments and launchers of the batched serving operators: rows appended
// to a paged cache, attention over pages and over packed prompts, token log probabilities.
#pragma once

#include "common.hpp"
#include "serve_index.hpp"

namespace rie {

// Keys and values of a launch: pages (table given) or the packed rows of the prompts.
// Strides are in bytes.
struct KvView {
    const uint8_t *k = nullptr, *v = nullptr;
    int64_t k_row = 0, k_head = 0, v_row = 0, v_head = 0;
    int64_t page = 0;              // from one page to the next
    const int *table = nullptr;    // [n_seq][table_stride] page ids
    int64_t table_stride = 0;
    int page_shift = 0, n_pages = 0;
    int cap = 0;                   // positions that a table row (or the packed rows) can address
};

struct BatchView {
    const int *starts = nullptr, *lens = nullptr;  // lens: nullptr where every token is new
    int n_seq = 0, n_rows = 0, max_new = 0, max_len = 0;
};

struct ServeAttnArgs {
    KvView kv;
    BatchView b;
    const uint8_t *q = nullptr;
    uint8_t *out = nullptr;
    int64_t q_row = 0, q_head = 0, o_row = 0, o_head = 0;  // bytes
    int n_head = 0, n_kv = 0, G = 0, hd = 0, ty = 0, window = 0;
    float scale = 1, softcap = 0;
    float *part = nullptr, *ml = nullptr;  // split partials [row][head][S][hd] and [row][head][S][2]
    int C = 0, S = 1;                      // split_plan
    int n_blocks = 0;                      // blocks of query rows (tile kernel)
};
constexpr int SERVE_MAX_SPLIT = 128;
// whether the few-rows kernel takes the launch (else the tile kernel), and its splits
bool serve_attn_few(const ServeAttnArgs &a);
SplitPlan serve_attn_splits(const ServeAttnArgs &a);
// bytes of the partials of a launch (0 without splits)
size_t serve_attn_ws(const ServeAttnArgs &a);
bool serve_attn_head_dim_ok(int hd);
void launch_serve_attn(ServeAttnArgs a, void *ws, hipStream_t st);

struct PagedAppendArgs {
    KvView kv;  // kv.k and kv.v are written
    BatchView b;
    const uint8_t *k = nullptr, *v = nullptr;
    int64_t k_row = 0, k_head = 0, v_row = 0, v_head = 0;  // of the new rows, bytes
    int n_kv = 0, hd = 0, ty = 0, src_ty = 0;
};
void launch_paged_append(const PagedAppendArgs &a, hipStream_t st);

struct LogprobArgs {
    const void *x = nullptr;
    int ty = 0, n = 0, V = 0;
    int64_t ld = 0;  // elements between rows
    const int *targets = nullptr;
    float *logprob = nullptr, *entropy = nullptr;
    int n_top = 0;
    int *top_ids = nullptr;
    float *top_logprobs = nullptr;
};
constexpr int LOGPROB_MAX_TOP = 64;
constexpr int LOGPROB_MAX_V = 1 << 21;
size_t logprobs_ws(int n, int V);
void launch_logprobs(const LogprobArgs &a, void *ws, hipStream_t st);

}  // namespace rie
