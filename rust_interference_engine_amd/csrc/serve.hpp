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

// Pages of 8 bits: a value is its code times the scale of its block of positions and head
struct Scales8 {
    float *k = nullptr, *v = nullptr;
    uint32_t page = 0, block = 0, head = 0;  // strides, values
    int block_shift = 0;
};
constexpr float SCALE8_MIN = 0x1p-60f, SCALE8_MAX = 0x1p50f;  // of blocks that hold anything but zeros
struct ServeAttn8Args {
    ServeAttnArgs a;  // a.ty: type of queries and outputs
    Scales8 s;
};
size_t serve_attn8_ws(const ServeAttnArgs &a);
void launch_serve_attn8(ServeAttn8Args x, void *ws, hipStream_t st);

struct PagedAppendArgs {
    KvView kv;  // kv.k and kv.v are written
    BatchView b;
    const uint8_t *k = nullptr, *v = nullptr;
    int64_t k_row = 0, k_head = 0, v_row = 0, v_head = 0;  // of the new rows, bytes
    int n_kv = 0, hd = 0, ty = 0, src_ty = 0;
};
void launch_paged_append(const PagedAppendArgs &a, hipStream_t st);
struct PagedAppend8Args {
    PagedAppendArgs a;  // a.ty is not looked at
    Scales8 s;
};
void launch_paged_append8(const PagedAppend8Args &x, hipStream_t st);

// Rows of queries and keys turned by their positions: those given, or those of the batch's rows
struct RotaryArgs {
    BatchView b;
    KvView kv;  // kv.table is not read; it says that positions go by lens
    const int *positions = nullptr;
    const double *freqs = nullptr;  // [dims / 2]
    float magnitude = 1;
    int hd = 0, dims = 0, n_q = 0, n_k = 0, src_ty = 0, dst_ty = 0;
    bool interleaved = false, in_place = false, wide = false;  // wide: rows and halves are 16-byte aligned
    const uint8_t *q = nullptr, *k = nullptr;
    uint8_t *q_out = nullptr, *k_out = nullptr;
    int64_t q_row = 0, q_head = 0, k_row = 0, k_head = 0, qo_row = 0, qo_head = 0, ko_row = 0, ko_head = 0;  // bytes
};
constexpr int ROTARY_MAX_HD = 1024;
void launch_rotary(const RotaryArgs &a, hipStream_t st);

// The n_out best (beam, token) candidates of each of n requests of n_beams beams, a row of logits each
struct BeamArgs {
    const void *x = nullptr;
    int ty = 0, n = 0, n_beams = 0, V = 0, n_out = 0, pad = 0;
    int64_t ld = 0;  // elements between rows
    const float *scores = nullptr;
    const int *finished = nullptr;
    float *next = nullptr;
    int *parents = nullptr, *tokens = nullptr;
};
constexpr int BEAM_MAX_BEAMS = 64, BEAM_MAX_OUT = 128, BEAM_MAX_V = 1 << 21;
size_t beam_ws(int n, int n_beams, int V, int n_out);
void launch_beam(const BeamArgs &a, void *ws, hipStream_t st);

// A pool of pages: the table rows of n_seq sequences, how many pages each holds and how many
// positions it has, the rows that hold each page (0: free), and what calls count
struct PoolView {
    int n_seq = 0, n_pages = 0, cols = 0, page_shift = 0;
    int *table = nullptr, *lens = nullptr, *held = nullptr, *refs = nullptr, *counts = nullptr;
    int64_t table_stride = 0;
};
// Memory that is divided into pages as the caches are; all of a page's bytes lie together
struct PageBuf {
    uint8_t *base;
    int64_t stride, bytes;
};
constexpr int POOL_MAX_SEQ = 4096, POOL_MAX_PAGES = 1 << 24, POOL_MAX_COLS = 1 << 20;
size_t page_reserve_ws(const PoolView &p);
size_t page_fork_ws(const PoolView &p);
size_t page_compact_ws(const PoolView &p);
void launch_page_reserve(const PoolView &p, void *ws, hipStream_t st);
void launch_page_fork(const PoolView &p, const int *src, const PageBuf *bufs, int n_bufs, void *ws, hipStream_t st);
void launch_page_free(const PoolView &p, const int *which, hipStream_t st);
void launch_page_compact(const PoolView &p, const PageBuf *bufs, int n_bufs, void *ws, hipStream_t st);
void launch_page_copy(const PageBuf *bufs, int n_bufs, int n_pages, const int *src, const int *dst, int n, hipStream_t st);

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
