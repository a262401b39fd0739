// decoding.cpp — the C ABI of what a batch's decoding needs beside attention (include/rie_hip.h):
// rotary positions, beam selection, a pool of pages.  Checks of what the host can see, and the
// launches on the caller's stream.
#include "serve_check.hpp"

#include <array>
#include <climits>
#include <cmath>
#include <vector>

namespace {

using namespace rie;

bool is_float(int ty) { return ty == T_F32 || is16(ty); }
int bytes_of(int ty) { return ty == T_F32 ? 4 : 2; }

// Rows and heads of values of es bytes: aligned to them, strides within 2^40
void check_loose(const void *p, int64_t row, int64_t head, int es, const char *what) {
    if ((uintptr_t)p % es) throw bad(std::string(what) + " has to be aligned to its type");
    const int64_t most = (int64_t)1 << 40;
    if (row < 0 || row > most || head < 0 || head > most) throw bad(std::string(what) + ": strides have to lie in 0..2^40");
}
bool aligned16(const void *p, int64_t row, int64_t head, int es) { return ((uintptr_t)p | (uint64_t)(row * es) | (uint64_t)(head * es)) % 16 == 0; }

PoolView pool_view(const rie_hip_pool *p) {
    if (!p) throw bad("pool is NULL");
    if (p->n_seq < 1 || p->n_seq > POOL_MAX_SEQ) throw bad("n_seq has to lie in 1.." + std::to_string(POOL_MAX_SEQ));
    if (p->n_pages < 1 || p->n_pages > POOL_MAX_PAGES || p->table_cols < 1 || p->table_cols > POOL_MAX_COLS) throw bad("n_pages has to lie in 1..2^24, table_cols in 1..2^20");
    if (p->page_size < 1 || p->page_size > 4096 || (p->page_size & (p->page_size - 1))) throw Error{E_UNSUPPORTED, "page_size has to be a power of two in 1..4096"};
    if (p->n_seq > 1 && (p->table_stride < p->table_cols || p->table_stride > (int64_t)1 << 40)) throw bad("table_stride has to lie in table_cols..2^40");
    PoolView v;
    v.n_seq = p->n_seq;
    v.n_pages = p->n_pages;
    v.cols = p->table_cols;
    v.page_shift = __builtin_ctz((unsigned)p->page_size);
    v.table = p->table;
    v.table_stride = p->n_seq > 1 ? p->table_stride : 0;
    v.lens = p->lens;
    v.held = p->held;
    v.refs = p->refs;
    v.counts = p->counts;
    return v;
}

void check_pool(const PoolView &p, const OnDevice &dev) {
    dev.check(p.table, "table");
    dev.check(p.lens, "lens");
    dev.check(p.held, "held");
    dev.check(p.refs, "refs");
    dev.check(p.counts, "counts");
}

std::vector<PageBuf> page_bufs(const rie_hip_page_buf *b, int32_t n, int n_pages) {
    if (n < 0 || n > 4096) throw bad("n_bufs has to lie in 0..4096");
    if (n && !b) throw bad("bufs is NULL");
    std::vector<PageBuf> v;
    for (int i = 0; i < n; i++) {
        const int64_t stride = used(n_pages, b[i].page_stride);
        if (b[i].page_bytes < 1 || b[i].page_bytes > (int64_t)1 << 30 || b[i].page_bytes % 4) throw bad("bufs: page_bytes has to be a multiple of 4 in 1..2^30");
        if ((uintptr_t)b[i].base % 4 || stride % 4) throw bad("bufs: base and page_stride have to be multiples of 4");
        if (n_pages > 1 && (stride < b[i].page_bytes || stride > (int64_t)1 << 40)) throw bad("bufs: page_stride has to lie in page_bytes..2^40");
        v.push_back(PageBuf{(uint8_t *)b[i].base, stride, b[i].page_bytes});
    }
    return v;
}

void check_bufs(const std::vector<PageBuf> &v, const OnDevice &dev) {
    for (const PageBuf &b : v) dev.check(b.base, "bufs");
}

void check_ws(const void *ws, size_t bytes, size_t need) {
    if (bytes < need) throw bad("workspace of " + std::to_string(bytes) + " bytes, " + std::to_string(need) + " needed");
    if ((uintptr_t)ws % 16) throw bad("ws has to be 16-byte aligned");
}

void check_beam(int32_t n, int32_t n_beams, int32_t n_vocab, int32_t n_out) {
    if (n < 1 || n > 1 << 22 || n_beams < 1 || n_beams > BEAM_MAX_BEAMS || (int64_t)n * n_beams > 1 << 22) throw bad("n_beams has to lie in 1..64, n*n_beams in 1..2^22");
    if (n_vocab < 1 || n_vocab > BEAM_MAX_V) throw bad("n_vocab has to lie in 1..2^21");
    if (n_out < 1 || n_out > BEAM_MAX_OUT || n_out > (int64_t)n_beams * n_vocab) throw bad("n_out has to lie in 1..128 and not pass n_beams*n_vocab");
    if ((int64_t)n * n_beams * n_vocab > (int64_t)1 << 40) throw bad("n*n_beams*n_vocab has to stay under 2^40");  // 2^32 threads
}

}  // namespace

extern "C" {

int32_t rie_hip_k_rotary(const rie_hip_rotary *x, const rie_hip_seqs *seqs, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (!x) throw bad("rotary is NULL");
        if (!seqs == !x->positions) throw bad("positions or seqs has to be given, not both");
        if (!is_float(x->src_ty) || !is_float(x->dst_ty)) throw Error{E_UNSUPPORTED, "rows have to be f32, f16 or bf16"};
        if (x->head_dim < 2 || x->head_dim > ROTARY_MAX_HD || x->dims < 2 || x->dims > x->head_dim || x->dims % 2) throw Error{E_UNSUPPORTED, "head_dim has to lie in 2..1024, dims be even and not pass it"};
        if (x->n_q < 0 || x->n_k < 0 || x->n_q > 4096 || x->n_k > 4096 || x->n_q + x->n_k < 1) throw bad("n_q and n_k have to lie in 0..4096, one of them above 0");
        if (!std::isfinite(x->magnitude)) throw bad("magnitude has to be finite");
        RotaryArgs a;
        if (seqs) {
            a.b = batch(seqs, true);
            if (a.b.n_rows != x->n_rows) throw bad("n_rows and seqs.n_rows differ");
            a.kv.table = seqs->lens;
            a.kv.cap = INT32_MAX;
        } else {
            if (x->n_rows < 1 || x->n_rows > MOST_ROWS) throw bad("n_rows has to lie in 1..2^26-4");
            a.b.n_rows = x->n_rows;
        }
        a.positions = x->positions;
        a.freqs = x->freqs;
        if ((uintptr_t)a.freqs % 8) throw bad("freqs has to be aligned to its type");
        a.magnitude = x->magnitude;
        a.hd = x->head_dim;
        a.dims = x->dims;
        a.n_q = x->n_q;
        a.n_k = x->n_k;
        a.src_ty = x->src_ty;
        a.dst_ty = x->dst_ty;
        a.interleaved = x->interleaved != 0;
        const int es = bytes_of(a.src_ty), ed = bytes_of(a.dst_ty);
        a.in_place = true;
        a.wide = a.dims % 16 == 0 && a.hd % 8 == 0;
        std::array<RowsAt, 2> in_at{}, out_at{};  // of q, of k
        const auto rows = [&](int heads, const void *in, int64_t row, int64_t head, void *out, int64_t o_row, int64_t o_head, const char *what) {
            row = used(x->n_rows, row);
            head = used(heads, head);
            o_row = used(x->n_rows, o_row);
            o_head = used(heads, o_head);
            check_loose(in, row, head, es, what);
            check_loose(out, o_row, o_head, ed, what);
            check_apart({{x->n_rows, o_row}, {heads, o_head}}, a.hd, what);
            const bool place = in == out;
            if (place && (row != o_row || head != o_head || a.src_ty != a.dst_ty)) throw bad(std::string(what) + ": rows that are turned in place keep their type and strides");
            a.in_place = a.in_place && place;
            const int i = what[0] == 'k';
            in_at[i] = RowsAt{in, x->n_rows, row * es, heads, head * es, (int64_t)a.hd * es};
            out_at[i] = RowsAt{out, x->n_rows, o_row * ed, heads, o_head * ed, (int64_t)a.hd * ed};
            if (!place && rows_overlap(in_at[i], out_at[i])) throw bad(std::string(what) + " and " + what + "_out share memory");
            a.wide = a.wide && aligned16(in, row, head, es) && aligned16(out, o_row, o_head, ed);
            return std::array<int64_t, 4>{row * es, head * es, o_row * ed, o_head * ed};
        };
        if (a.n_q) {
            const auto s = rows(a.n_q, x->q, x->q_row_stride, x->q_head_stride, x->q_out, x->q_out_row_stride, x->q_out_head_stride, "q");
            a.q = (const uint8_t *)x->q;
            a.q_out = (uint8_t *)x->q_out;
            a.q_row = s[0], a.q_head = s[1], a.qo_row = s[2], a.qo_head = s[3];
        }
        if (a.n_k) {
            const auto s = rows(a.n_k, x->k, x->k_row_stride, x->k_head_stride, x->k_out, x->k_out_row_stride, x->k_out_head_stride, "k");
            a.k = (const uint8_t *)x->k;
            a.k_out = (uint8_t *)x->k_out;
            a.k_row = s[0], a.k_head = s[1], a.ko_row = s[2], a.ko_head = s[3];
        }
        if (a.n_q && a.n_k) {
            if (rows_overlap(out_at[0], out_at[1])) throw bad("q_out and k_out share memory");
            if (!a.in_place && rows_overlap(out_at[0], in_at[1])) throw bad("q_out and k share memory");
            if (!a.in_place && rows_overlap(out_at[1], in_at[0])) throw bad("k_out and q share memory");
        }
        const OnDevice dev((hipStream_t)stream);
        dev.check(a.freqs, "freqs");
        if (seqs) {
            dev.check(a.b.starts, "starts");
            dev.check(a.b.lens, "lens");
        } else {
            dev.check(a.positions, "positions");
        }
        if (a.n_q) {
            dev.check(a.q, "q");
            dev.check(a.q_out, "q_out");
        }
        if (a.n_k) {
            dev.check(a.k, "k");
            dev.check(a.k_out, "k_out");
        }
        launch_rotary(a, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

size_t rie_hip_k_beam_select_ws(int32_t n, int32_t n_beams, int32_t n_vocab, int32_t n_out) {
    size_t bytes = 0;
    (void)guarded(nullptr, 0, [&] {
        check_beam(n, n_beams, n_vocab, n_out);
        bytes = beam_ws(n, n_beams, n_vocab, n_out);
    });
    return bytes;
}

int32_t rie_hip_k_beam_select(int32_t ty, const void *logits, int32_t n, int32_t n_beams, int32_t n_vocab, int64_t row_stride,
                              const float *scores, const int32_t *finished, int32_t pad, int32_t n_out, float *next_scores,
                              int32_t *parents, int32_t *tokens, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (!is_float(ty)) throw Error{E_UNSUPPORTED, "logits have to be f32, f16 or bf16"};
        check_beam(n, n_beams, n_vocab, n_out);
        if ((uintptr_t)logits % bytes_of(ty)) throw bad("logits have to be aligned to their type");
        if (row_stride < 0 || row_stride > (int64_t)1 << 40) throw bad("row_stride has to lie in 0..2^40");
        if (finished && (pad < 0 || pad >= n_vocab)) throw bad("pad has to be a token");
        check_ws(ws, ws_bytes, beam_ws(n, n_beams, n_vocab, n_out));
        const OnDevice dev((hipStream_t)stream);
        dev.check(logits, "logits");
        dev.check(scores, "scores");
        if (finished) dev.check(finished, "finished");
        dev.check(next_scores, "next_scores");
        dev.check(parents, "parents");
        dev.check(tokens, "tokens");
        dev.check(ws, "ws");
        BeamArgs a;
        a.x = logits;
        a.ty = ty;
        a.n = n;
        a.n_beams = n_beams;
        a.V = n_vocab;
        a.ld = (int64_t)n * n_beams > 1 ? row_stride : 0;
        a.scores = scores;
        a.finished = finished;
        a.pad = pad;
        a.n_out = n_out;
        a.next = next_scores;
        a.parents = parents;
        a.tokens = tokens;
        launch_beam(a, ws, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

size_t rie_hip_k_page_ws(const rie_hip_pool *pool) {
    size_t bytes = 0;
    (void)guarded(nullptr, 0, [&] {
        const PoolView p = pool_view(pool);
        bytes = std::max({page_reserve_ws(p), page_fork_ws(p), page_compact_ws(p)});
    });
    return bytes;
}

int32_t rie_hip_k_page_reserve(const rie_hip_pool *pool, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const PoolView p = pool_view(pool);
        check_ws(ws, ws_bytes, page_reserve_ws(p));
        const OnDevice dev((hipStream_t)stream);
        check_pool(p, dev);
        dev.check(ws, "ws");
        launch_page_reserve(p, ws, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

int32_t rie_hip_k_page_fork(const rie_hip_pool *pool, const int32_t *src, const rie_hip_page_buf *bufs, int32_t n_bufs, void *ws,
                            size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const PoolView p = pool_view(pool);
        const std::vector<PageBuf> b = page_bufs(bufs, n_bufs, p.n_pages);
        check_ws(ws, ws_bytes, page_fork_ws(p));
        const OnDevice dev((hipStream_t)stream);
        check_pool(p, dev);
        dev.check(src, "src");
        check_bufs(b, dev);
        dev.check(ws, "ws");
        launch_page_fork(p, src, b.data(), n_bufs, ws, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

int32_t rie_hip_k_page_free(const rie_hip_pool *pool, const int32_t *which, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const PoolView p = pool_view(pool);
        const OnDevice dev((hipStream_t)stream);
        check_pool(p, dev);
        dev.check(which, "which");
        launch_page_free(p, which, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

int32_t rie_hip_k_page_compact(const rie_hip_pool *pool, const rie_hip_page_buf *bufs, int32_t n_bufs, void *ws, size_t ws_bytes,
                               void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const PoolView p = pool_view(pool);
        const std::vector<PageBuf> b = page_bufs(bufs, n_bufs, p.n_pages);
        check_ws(ws, ws_bytes, page_compact_ws(p));
        const OnDevice dev((hipStream_t)stream);
        check_pool(p, dev);
        check_bufs(b, dev);
        dev.check(ws, "ws");
        launch_page_compact(p, b.data(), n_bufs, ws, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

int32_t rie_hip_k_page_copy(const rie_hip_page_buf *bufs, int32_t n_bufs, int32_t n_pages, const int32_t *src, const int32_t *dst,
                            int32_t n, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (n_pages < 1 || n_pages > POOL_MAX_PAGES || n < 1 || n > POOL_MAX_PAGES) throw bad("n_pages and n have to lie in 1..2^24");
        const std::vector<PageBuf> b = page_bufs(bufs, n_bufs, n_pages);
        const OnDevice dev((hipStream_t)stream);
        check_bufs(b, dev);
        dev.check(src, "src");
        dev.check(dst, "dst");
        launch_page_copy(b.data(), n_bufs, n_pages, src, dst, n, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

}  // extern "C"
