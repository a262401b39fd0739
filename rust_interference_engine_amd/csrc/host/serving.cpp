// serving.cpp — the C ABI of the batched serving operators (include/rie_hip.h): checks of
// what the host can see, and the launches on the caller's stream.
#include "../../../include/rie_hip.h"

#include "../serve.hpp"
#include "guard.hpp"

#include <algorithm>
#include <cmath>
#include <string>

using rie::Error;
using rie::guarded;

namespace {

Error bad(const std::string &m) { return Error{rie::E_RUNTIME, m}; }

// The stream's device is the current one while this lives.
class OnDevice {
  public:
    explicit OnDevice(hipStream_t st) {
        RIE_HIP_CHECK(hipGetDevice(&was_));
        device = was_;
        if (st) {
            hipDevice_t d;
            RIE_HIP_CHECK(hipStreamGetDevice(st, &d));
            device = (int)d;
        }
        if (device != was_) RIE_HIP_CHECK(hipSetDevice(device));
    }
    ~OnDevice() {
        if (device != was_) (void)hipSetDevice(was_);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

    // p is memory that a kernel on this device may use
    void check(const void *p, const char *what) const {
        if (!p) throw bad(std::string(what) + " is NULL");
        hipPointerAttribute_t a;
        const hipError_t e = hipPointerGetAttributes(&a, p);
        if (e != hipSuccess) (void)hipGetLastError();  // not an error of the launch
        if (e != hipSuccess || (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged))
            throw bad(std::string(what) + " is not device memory");
        if (a.type == hipMemoryTypeDevice && a.device != device)
            throw bad(std::string(what) + " is on device " + std::to_string(a.device) + ", the stream on device " + std::to_string(device));
    }

    int device;

  private:
    int was_;
};

bool is16(int ty) { return ty == rie::T_F16 || ty == rie::T_BF16; }

// A dimension of one entry is at 0, whatever its stride says (that of a tensor's is arbitrary)
int64_t used(int64_t n, int64_t stride) { return n > 1 ? stride : 0; }

// Rows of values of es bytes each start at p + any multiples of the strides: all 16-byte
// aligned, and strides of 2^26 bytes at most, so that 16 rows stay within 31 bits
void check_rows(const void *p, int64_t row, int64_t head, int es, const char *what) {
    const int64_t a = 16 / es, most = ((int64_t)1 << 26) / es;
    if ((uintptr_t)p % 16 || row % a || head % a) throw bad(std::string(what) + ": rows have to be 16-byte aligned");
    if (row < 0 || row > most || head < 0 || head > most) throw bad(std::string(what) + ": strides have to lie in 0.." + std::to_string(most));
}

// Rows that are written, n of each dimension a stride apart: no two of them share a value.  Every
// stride has to cover what the smaller ones span.
struct Dim {
    int64_t n, stride;
};
template <size_t N>
void check_apart(Dim (&&dims)[N], int hd, const char *what) {
    std::sort(dims, dims + N, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
    __int128 span = hd;  // strides of up to 2^40 by counts of up to 2^31
    for (const Dim &d : dims) {
        if (d.n <= 1) continue;
        if (d.stride < span) throw bad(std::string(what) + ": strides below head_dim, or below what the smaller ones span, would make rows overlap");
        span += (__int128)(d.n - 1) * d.stride;
    }
}

constexpr int MOST = 1 << 30;  // positions
constexpr int MOST_ROWS = (1 << 26) - 4;  // 4 to a workgroup of 256: a launch has under 2^32 threads

rie::BatchView batch(const rie_hip_seqs *s, bool lens) {
    if (!s) throw bad("seqs is NULL");
    if (s->n_seq < 1 || s->n_rows < 1 || s->n_seq >= 1 << 24 || s->n_rows > MOST_ROWS) throw bad("n_seq has to lie in 1..2^24-1, n_rows in 1..2^26-4");
    if (s->max_new < 1 || s->max_len < 1 || s->max_new > MOST || s->max_len > MOST) throw bad("max_new and max_len have to lie in 1..2^30");
    rie::BatchView b;
    b.starts = s->starts;
    b.lens = lens ? s->lens : nullptr;
    b.n_seq = s->n_seq;
    b.n_rows = s->n_rows;
    b.max_new = std::min(s->max_new, s->n_rows);
    b.max_len = s->max_len;
    return b;
}

void check_heads(int ty, int hd, int n_kv) {
    if (!is16(ty)) throw Error{rie::E_UNSUPPORTED, "keys and values have to be f16 or bf16"};
    if (!rie::serve_attn_head_dim_ok(hd)) throw Error{rie::E_UNSUPPORTED, "head_dim has to be 32, 64, 96, 128 or 256"};
    if (n_kv < 1 || n_kv > 4096) throw bad("n_kv has to lie in 1..4096");
}

rie::KvView pages_view(const rie_hip_pages *p) {
    if (!p) throw bad("pages is NULL");
    check_heads(p->ty, p->head_dim, p->n_kv);
    if (p->page_size < 16 || p->page_size > 4096 || (p->page_size & (p->page_size - 1)))
        throw Error{rie::E_UNSUPPORTED, "page_size has to be a power of two in 16..4096"};
    if (p->n_pages < 1 || p->table_cols < 1 || p->table_stride < 0) throw bad("n_pages and table_cols have to be positive");
    const int64_t head = used(p->n_kv, p->head_stride), page = used(p->n_pages, p->page_stride);
    check_rows(p->k, p->slot_stride, head, 2, "pages");
    check_rows(p->v, p->slot_stride, head, 2, "pages");
    if (page < 0 || page % 8 || page > ((int64_t)1 << 40)) throw bad("pages: page_stride has to be a multiple of 8 in 0..2^40");
    rie::KvView v;
    v.k = (const uint8_t *)p->k;
    v.v = (const uint8_t *)p->v;
    v.k_row = v.v_row = p->slot_stride * 2;
    v.k_head = v.v_head = head * 2;
    v.page = page * 2;
    v.table = p->table;
    v.table_stride = p->table_stride;
    v.page_shift = __builtin_ctz((unsigned)p->page_size);
    v.n_pages = p->n_pages;
    v.cap = (int)std::min<int64_t>((int64_t)p->table_cols * p->page_size, MOST);
    return v;
}

rie::ServeAttnArgs attention(const rie_hip_seqs *seqs, const rie_hip_attn *at, int ty, int hd, int n_kv, const rie::KvView &kv) {
    if (!at) throw bad("attn is NULL");
    rie::ServeAttnArgs a;
    a.kv = kv;
    a.b = batch(seqs, kv.table != nullptr);
    if (at->n_head < n_kv || at->n_head % n_kv || at->n_head > 4096) throw bad("n_head has to be a multiple of n_kv, at most 4096");
    if (!(at->scale > 0) || !std::isfinite(at->scale)) throw bad("scale has to be positive and finite");
    if (!(at->softcap >= 0) || !std::isfinite(at->softcap)) throw bad("softcap has to be 0 (none) or positive and finite");
    if (at->window < 0) throw bad("window has to be 0 (none) or positive");
    a.q = (const uint8_t *)at->q;
    a.out = (uint8_t *)at->out;
    a.q_row = used(a.b.n_rows, at->q_row_stride) * 2;
    a.q_head = used(at->n_head, at->q_head_stride) * 2;
    a.o_row = used(a.b.n_rows, at->out_row_stride) * 2;
    a.o_head = used(at->n_head, at->out_head_stride) * 2;
    a.n_head = at->n_head;
    a.n_kv = n_kv;
    a.G = at->n_head / n_kv;
    a.hd = hd;
    a.ty = ty;
    a.window = at->window;
    a.scale = at->scale;
    a.softcap = at->softcap;
    if (!kv.table) a.b.max_len = std::min(a.b.max_len, a.b.max_new);
    else a.b.max_len = std::min(a.b.max_len, kv.cap);
    // a launch has under 2^32 threads: 256 to a workgroup, 4 (row, head) pairs to one where the splits are added up
    if ((int64_t)a.b.n_rows * a.n_head > MOST_ROWS || ((int64_t)a.b.n_seq + (int64_t)a.b.n_rows * a.G / 128) * n_kv >= 1 << 24)
        throw bad("n_rows*n_head has to lie in 1..2^26-4, n_seq*n_kv under 2^24");
    return a;
}

void run_attention(const rie::ServeAttnArgs &a, void *ws, size_t ws_bytes, void *stream) {
    check_rows(a.q, a.q_row / 2, a.q_head / 2, 2, "q");
    check_rows(a.out, a.o_row / 2, a.o_head / 2, 2, "out");
    check_apart({{a.b.n_rows, a.o_row / 2}, {a.n_head, a.o_head / 2}}, a.hd, "out");
    const size_t need = rie::serve_attn_ws(a);
    if (ws_bytes < need) throw bad("workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");
    if ((uintptr_t)ws % 16) throw bad("ws has to be 16-byte aligned");
    const OnDevice dev((hipStream_t)stream);
    dev.check(a.q, "q");
    dev.check(a.out, "out");
    dev.check(a.kv.k, "k");
    dev.check(a.kv.v, "v");
    dev.check(a.b.starts, "starts");
    if (a.kv.table) {
        dev.check(a.kv.table, "table");
        dev.check(a.b.lens, "lens");
    }
    if (need) dev.check(ws, "ws");
    rie::launch_serve_attn(a, ws, (hipStream_t)stream);
    RIE_HIP_CHECK(hipGetLastError());
}

rie::KvView packed_view(int ty, int hd, int n_kv, int n_rows, const void *k, const void *v, int64_t kr, int64_t kh, int64_t vr, int64_t vh) {
    check_heads(ty, hd, n_kv);
    kr = used(n_rows, kr);
    vr = used(n_rows, vr);
    kh = used(n_kv, kh);
    vh = used(n_kv, vh);
    check_rows(k, kr, kh, 2, "k");
    check_rows(v, vr, vh, 2, "v");
    rie::KvView x;
    x.k = (const uint8_t *)k;
    x.v = (const uint8_t *)v;
    x.k_row = kr * 2;
    x.k_head = kh * 2;
    x.v_row = vr * 2;
    x.v_head = vh * 2;
    return x;
}

}  // namespace

extern "C" {

int32_t rie_hip_k_paged_append(const rie_hip_pages *pages, const rie_hip_seqs *seqs, int32_t src_ty, const void *k, const void *v,
                               int64_t row_stride, int64_t head_stride, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        rie::PagedAppendArgs a;
        a.kv = pages_view(pages);
        a.b = batch(seqs, true);
        if (src_ty != rie::T_F32 && src_ty != pages->ty) throw Error{rie::E_UNSUPPORTED, "new rows have to be f32 or of the pages' type"};
        const int es = src_ty == rie::T_F32 ? 4 : 2;
        const int64_t row = used(a.b.n_rows, row_stride), head = used(pages->n_kv, head_stride);
        check_rows(k, row, head, es, "k");
        check_rows(v, row, head, es, "v");
        // keys and values too, which may lie between one another
        const int64_t apart = (const uint16_t *)pages->v - (const uint16_t *)pages->k;
        check_apart({{pages->page_size, pages->slot_stride}, {pages->n_kv, pages->head_stride}, {pages->n_pages, pages->page_stride},
                     {2, apart < 0 ? -apart : apart}}, pages->head_dim, "pages");
        a.k = (const uint8_t *)k;
        a.v = (const uint8_t *)v;
        a.k_row = a.v_row = row * es;
        a.k_head = a.v_head = head * es;
        a.n_kv = pages->n_kv;
        a.hd = pages->head_dim;
        a.ty = pages->ty;
        a.src_ty = src_ty;
        const OnDevice dev((hipStream_t)stream);
        dev.check(a.kv.k, "pages");
        dev.check(a.kv.v, "pages");
        dev.check(a.kv.table, "table");
        dev.check(a.b.starts, "starts");
        dev.check(a.b.lens, "lens");
        dev.check(k, "k");
        dev.check(v, "v");
        rie::launch_paged_append(a, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

size_t rie_hip_k_paged_attention_ws(const rie_hip_pages *pages, const rie_hip_seqs *seqs, const rie_hip_attn *attn) {
    size_t n = 0;
    (void)guarded(nullptr, 0, [&] {
        if (!pages) throw bad("pages is NULL");
        n = rie::serve_attn_ws(attention(seqs, attn, pages->ty, pages->head_dim, pages->n_kv, pages_view(pages)));
    });
    return n;
}

int32_t rie_hip_k_paged_attention(const rie_hip_pages *pages, const rie_hip_seqs *seqs, const rie_hip_attn *attn, void *ws,
                                  size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        const rie::KvView kv = pages_view(pages);
        if (!kv.table) throw bad("table is NULL");
        run_attention(attention(seqs, attn, pages->ty, pages->head_dim, pages->n_kv, kv), ws, ws_bytes, stream);
    });
}

size_t rie_hip_k_packed_attention_ws(const rie_hip_seqs *seqs, int32_t ty, int32_t head_dim, int32_t n_kv, const rie_hip_attn *attn) {
    size_t n = 0;
    (void)guarded(nullptr, 0, [&] {
        check_heads(ty, head_dim, n_kv);
        n = rie::serve_attn_ws(attention(seqs, attn, ty, head_dim, n_kv, rie::KvView{}));
    });
    return n;
}

int32_t rie_hip_k_packed_attention(const rie_hip_seqs *seqs, int32_t ty, int32_t head_dim, int32_t n_kv, const void *k, const void *v,
                                   int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                                   const rie_hip_attn *attn, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (!seqs) throw bad("seqs is NULL");
        const rie::KvView kv = packed_view(ty, head_dim, n_kv, seqs->n_rows, k, v, k_row_stride, k_head_stride, v_row_stride, v_head_stride);
        run_attention(attention(seqs, attn, ty, head_dim, n_kv, kv), ws, ws_bytes, stream);
    });
}

size_t rie_hip_k_token_logprobs_ws(int32_t n, int32_t n_vocab) {
    return n < 1 || n_vocab < 1 || n_vocab > rie::LOGPROB_MAX_V ? 0 : rie::logprobs_ws(n, n_vocab);
}

int32_t rie_hip_k_token_logprobs(int32_t ty, const void *logits, int32_t n, int32_t n_vocab, int64_t row_stride,
                                 const int32_t *targets, float *logprob, float *entropy, int32_t n_top, int32_t *top_ids,
                                 float *top_logprobs, void *ws, size_t ws_bytes, void *stream, char *err, size_t err_len) {
    return guarded(err, err_len, [&] {
        if (ty != rie::T_F32 && !is16(ty)) throw Error{rie::E_UNSUPPORTED, "logits have to be f32, f16 or bf16"};
        if (n < 1 || n > 1 << 22 || n_vocab < 1 || n_vocab > rie::LOGPROB_MAX_V) throw bad("n has to lie in 1..2^22, n_vocab in 1..2^21");
        if ((int64_t)n * n_vocab > (int64_t)1 << 40) throw bad("n*n_vocab has to stay under 2^40");  // 2^32 threads
        const int es = ty == rie::T_F32 ? 4 : 2;
        if ((uintptr_t)logits % es) throw bad("logits have to be aligned to their type");
        if (row_stride < 0 || row_stride > (int64_t)1 << 40) throw bad("row_stride has to lie in 0..2^40");
        if (n_top < 0 || n_top > rie::LOGPROB_MAX_TOP || n_top > n_vocab) throw bad("n_top has to lie in 0..64 and not pass n_vocab");
        if (!targets != !logprob) throw bad("targets and logprob have to be given together");
        if (n_top && (!top_ids || !top_logprobs)) throw bad("top_ids or top_logprobs is NULL");
        const size_t need = rie::logprobs_ws(n, n_vocab);
        if (ws_bytes < need) throw bad("workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(need) + " needed");
        if ((uintptr_t)ws % 16) throw bad("ws has to be 16-byte aligned");
        const OnDevice dev((hipStream_t)stream);
        dev.check(logits, "logits");
        dev.check(ws, "ws");
        if (targets) {
            dev.check(targets, "targets");
            dev.check(logprob, "logprob");
        }
        if (entropy) dev.check(entropy, "entropy");
        if (n_top) {
            dev.check(top_ids, "top_ids");
            dev.check(top_logprobs, "top_logprobs");
        }
        rie::LogprobArgs a;
        a.x = logits;
        a.ty = ty;
        a.n = n;
        a.V = n_vocab;
        a.ld = row_stride;
        a.targets = targets;
        a.logprob = logprob;
        a.entropy = entropy;
        a.n_top = n_top;
        a.top_ids = top_ids;
        a.top_logprobs = top_logprobs;
        rie::launch_logprobs(a, ws, (hipStream_t)stream);
        RIE_HIP_CHECK(hipGetLastError());
    });
}

}  // extern "C"
