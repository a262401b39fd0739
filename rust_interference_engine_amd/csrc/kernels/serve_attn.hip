// serve_attn.hip — causal grouped-query attention of a batch of sequences over a cache
// of pages, or over packed prompts whose keys and values lie beside the queries:
//
//   o_t = Σ_j softmax_j(s_tj) v_j,  s_tj = scale · q_t·k_j  (cap · tanh(s / cap) with a softcap)
//
// over the positions j ≤ p_t, and j > p_t − window with a window, of token t at position
// p_t of its sequence.  A token that sees nothing gets zeros.  q, k, v and o are all f16
// or all bf16; scores, the softmax's maximum and sum, and the outputs are f32 sums.
//
// Rounding.  A probability enters the second product in the tensors' own type, rounded to
// nearest; the sum that the output is divided by adds the same rounded values, so that a
// row's weights add up to one.  The error this brings is about that of rounding the output
// once more (2^-9 of a bf16 value, 2^-12 of an f16 one, both root mean square).  The
// maximum that is subtracted is only moved when a score passes it by 2^8, so a probability
// lies in 0..2^8; f16 ones are multiplied by 2^6, since small ones would be subnormal.
//
// Values that are infinite or NaN reach the tokens that see them and no others: a tile that
// some token sees in part is searched for them as it is staged, and if there are any, they
// are added to the outputs one by one and replaced by zeros in the matrix product, where
// they would meet probabilities of zero.
//
// Two kernels.  attn_tile_kernel takes 128 query rows (token · group + head of the group,
// so the heads of a group share their keys) per workgroup and goes through the positions in
// tiles; attn_few_kernel takes a sequence with at most 32 rows, a tile per wave, and is
// bound by the reading of the cache.  Both compute Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ: a query is a
// lane's column in either product, so that its softmax state and probabilities stay in the
// lane; the value tile is read transposed from LDS (ds_read_b64_tr_b16) in the order of
// positions in which the first product leaves the probabilities.
#include "../common.hpp"
#include "../device.hpp"
#include "../serve.hpp"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace rie {

namespace {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 8 values of the tensors' type in a lane's operand registers
template <bool BF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
template <bool BF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}
// two f32 values rounded to nearest, packed
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const f32x2 v = {a, b};
    if constexpr (BF) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2_t));
}
// c + both halves of w
template <bool BF>
__device__ __forceinline__ float add2(uint32_t w, float c) {
    if constexpr (BF) return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), c, false);
    else return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_t, w), __builtin_bit_cast(half2_t, 0x3C003C00u), c, false);
}
template <bool BF>
__device__ __forceinline__ float value16(uint32_t bits) {
    return BF ? __uint_as_float(bits << 16) : h2f(bits);
}
// whether any of 8 values is infinite or NaN: its exponent bits are all ones
template <bool BF>
__device__ __forceinline__ bool nonfinite8(u32x4 v) {
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) any = any || (v[i] & E) == E || (v[i] & (E << 16)) == (E << 16);
    return any;
}
// w with infinite and NaN halves replaced by zeros
template <bool BF>
__device__ __forceinline__ uint32_t finite2(uint32_t w) {
    constexpr uint32_t E = BF ? 0x7F80u : 0x7C00u;
    if ((w & E) == E) w &= 0xFFFF0000u;
    if ((w & (E << 16)) == (E << 16)) w &= 0xFFFFu;
    return w;
}

// 4 values of one column: lane l of a group of 16 lanes names the 8 bytes of row l / 4 that
// hold columns 4·(l % 4) …, and gets rows 0..3 of column l
__device__ __forceinline__ u32x2 read_tr(const uint8_t *p) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(uintptr_t)(uint32_t)(uintptr_t)p));
}

// Probabilities are 2^(s − m + P_SHIFT)
template <bool BF>
constexpr float P_SHIFT = BF ? 0.0f : 6.0f;
constexpr float M_SLACK = 8.0f;  // how far a score may pass the maximum that is subtracted

// The largest i in [0, n) with key(starts[i], i) ≤ x, for keys that rise with i (0 where
// there is none): 64 candidates at a time, one per lane.
template <class F>
__device__ __forceinline__ int wave_find(const int *starts, int n, int x, F key) {
    int lo = 0;
    while (true) {
        const int w = (n + 63) >> 6;
        const int i = (int)(threadIdx.x & 63) * w;
        const bool le = i < n && key(starts[lo + imin(i, n - 1)], lo + i) <= x;
        const int c = imax((int)__popcll(__ballot(le)) - 1, 0);
        lo += c * w;
        n = imin(w, n - c * w);
        if (w == 1) break;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ SeqView view_of(const BatchView &b, const KvView &kv, int i) {
    const int s = b.starts[i], e = b.starts[i + 1];
    // packed rows: as many positions as rows
    SeqView v = seq_view(s, e, b.lens ? b.lens[i] : INT32_MAX, b.n_rows, kv.table ? kv.cap : INT32_MAX);
    if (!kv.table) v.len = v.n_new;
    v.row0 = __builtin_amdgcn_readfirstlane(v.row0);
    v.n_new = __builtin_amdgcn_readfirstlane(v.n_new);
    v.len = __builtin_amdgcn_readfirstlane(v.len);
    return v;
}

// Offset in bytes of position g's row (the same for a group of up to 16 positions that
// starts at a multiple of its size) in keys or values; ok: false for a page id that is
// none.  g < len.
__device__ __forceinline__ bool page_of(const KvView &kv, const int *trow, int g, int &page) {
    page = trow[g >> kv.page_shift];
    const bool ok = (unsigned)page < (unsigned)kv.n_pages;
    page = ok ? page : 0;
    return ok;
}

template <int HD>
constexpr int HDP = HD <= 64 ? 64 : HD <= 128 ? 128 : HD;  // values between rows of a tile in LDS
// 16-byte chunk c of row r goes to chunk c ^ swz(r), so that the lanes of a read, which
// take the same chunk of many rows (keys) or 4 chunks of 4 rows (values), use all banks
template <int HD>
__device__ __forceinline__ int swz_v(int r) { return HDP<HD> >= 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }

// score → exponent in log2 units, where the softcap makes it one already
template <bool CAP>
__device__ __forceinline__ float cap_score(float s, float in, float out) {
    if constexpr (!CAP) return s;
    const float e = exp2_hw(s * in);  // e^(2 s / cap)
    return out * (1.0f - 2.0f / (e + 1.0f));
}

// 16 bytes per lane from global memory (base + off) to LDS: lane l's go to dst + 16·l, with base
// and dst the same for the wave.  Written as the instruction, since the compiler waits for the
// builtin's copies before it reads any LDS, also of the buffers that they do not write; it has
// no result register, and the callers wait (wait_vmem) before the barrier behind which the
// copy is read.  Nothing else here uses m0.  Loads return in order, so waits that count without these wait longer at most.
__device__ __forceinline__ void copy_lds(const uint8_t *base, int off, const uint8_t *dst) {
    const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)dst);
    const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(from) : "memory");
}

constexpr int TILE_M = 128;  // query rows of a workgroup
// A tile in LDS.  A wave copies 1 KB at a time, its lanes' 16-byte chunks side by side, which
// is RPI whole rows in an order of their own choice: keys by chunk, then row, so that the 32
// rows' chunks of a read lie in all banks and a row's chunks at fixed distances; values by 64
// bytes of a row (32 dims), then row, for the same reasons of the transposed read.  Blocks are
// PAD bytes further apart than 1 KB where the next block's rows would meet the same banks.
// Rows shorter than their place (head sizes 32 and 96) leave the chunks behind them unused.
template <int HD>
struct TileLds {
    static constexpr int CPR = HDP<HD> / 8, RPI = 64 / CPR;  // chunks per row, rows per block
    static constexpr int K_BLOCK = 1024 + RPI * 16, V_BLOCK = 1024 + (RPI == 2 ? 128 : 0);
    static __device__ __forceinline__ int key(int r, int chunk) { return r / RPI * K_BLOCK + chunk * (RPI * 16) + r % RPI * 16; }
    static __device__ __forceinline__ int value(int r, int chunk) { return r / RPI * V_BLOCK + chunk / 4 * (RPI * 64) + r % RPI * 64 + chunk % 4 * 16; }
    // row and chunk of a lane's place in a block
    static __device__ __forceinline__ int key_row(int lane) { return lane % RPI; }
    static __device__ __forceinline__ int key_chunk(int lane) { return lane / RPI; }
    static __device__ __forceinline__ int value_row(int lane) { return lane / 4 % RPI; }
    static __device__ __forceinline__ int value_chunk(int lane) { return lane / (4 * RPI) * 4 + lane % 4; }
};

template <int HD>
constexpr int TILE_KT = HD <= 128 ? 64 : 32;  // positions of a tile

// A tile's work is cut into groups of 32 positions (KB to a tile), and the three steps of a
// group run in three places: while the vector units make the probabilities of group h, the
// matrix units form the outputs of h − 1 and the scores of h + 1, so that neither waits for
// the other within a wave.  K and V tiles go from global memory straight to LDS, two buffers
// each, one barrier per tile: at tile t's barrier the loads of K(t + 1) and V(t + KB − 2) are
// complete, K(t) and V(t + KB − 3) have been read, and K(t + 2) and V(t + KB − 1) are
// requested into their places.
template <int HD, bool BF, bool CAP>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_tile_kernel(ServeAttnArgs a) {
    constexpr int KT = TILE_KT<HD>, KB = KT / 32, RW = KT / 4, KS = HD / 16, DB = HD / 32;
    using Lds = TileLds<HD>;
    constexpr int RPI = Lds::RPI, NLD = RW / RPI, KBYTES = KT / RPI * Lds::K_BLOCK, VBYTES = KT / RPI * Lds::V_BLOCK;
    constexpr int NG = KT / 16;                                     // groups of 16 positions, which lie in one page
    __shared__ __align__(16) uint8_t s_k0[KBYTES], s_k1[KBYTES], s_v0[VBYTES], s_v1[VBYTES];
    __shared__ __align__(16) int s_nf[4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int G = a.G, kvh = blockIdx.x % a.n_kv;
    const int blk = a.n_blocks - 1 - (int)(blockIdx.x / a.n_kv);  // a sequence's longest rows first
    const int si = wave_find(a.b.starts, a.b.n_seq, blk, [&](int s, int i) { return block_base(iclamp(s, 0, a.b.n_rows), i, G, TILE_M); });
    const SeqView sv = view_of(a.b, a.kv, si);
    const int lb = blk - block_base(sv.row0, si, G, TILE_M);
    const int n_rows = sv.n_new * G;
    if (lb < 0 || lb >= (n_rows + TILE_M - 1) / TILE_M) return;
    const int r0 = lb * TILE_M, r1 = imin(r0 + TILE_M, n_rows) - 1;
    const int pos0 = sv.len - sv.n_new;  // position of token 0
    const KeyRange kr = key_range(sv, r0 / G, r1 / G, a.window);
    const int nt = tile_count(kr, KT), ns = split_count(nt, a.C, a.S), sp = blockIdx.y;
    if (sp >= ns) return;
    const int t_begin = first_tile(kr, KT) + sp * a.C, t_end = sp == ns - 1 ? first_tile(kr, KT) + nt : t_begin + a.C;

    // this lane's query row, and what the rows of its wave see
    const int row = r0 + w * 32 + (lane & 31);
    const bool live = row < n_rows;
    const int tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
    const int p_q = live ? pos0 + tok : -1;
    const int lo_q = a.window > 0 ? p_q - a.window : -1;  // sees j in (lo_q, p_q]
    const bool wave_live = r0 + w * 32 <= r1;
    const int w_t0 = imin(r0 + w * 32, r1) / G, w_t1 = imin(r0 + w * 32 + 31, r1) / G;
    const int all_hi = pos0 + w_t0, all_lo = a.window > 0 ? pos0 + w_t1 - a.window : -1;  // every row of the wave sees (all_lo, all_hi]
    const int wg_hi = pos0 + r0 / G, wg_lo = a.window > 0 ? pos0 + r1 / G - a.window : -1;  // and of the workgroup
    u32x4 qf[KS];
    {
        const uint8_t *qp = a.q + (int64_t)(sv.row0 + tok) * a.q_row + head * a.q_head + h * 16;
#pragma unroll
        for (int i = 0; i < KS; i++) qf[i] = live ? *(const u32x4 *)(qp + i * 32) : u32x4{0, 0, 0, 0};
    }

    // ---- copies: wave w's are rows w·RW .. of a tile, which lie in one page ----
    const int *trow = a.kv.table ? a.kv.table + (int64_t)si * a.kv.table_stride : nullptr;
    const uint8_t *kbase = a.kv.k + kvh * a.kv.k_head, *vbase = a.kv.v + kvh * a.kv.v_head;
    const int k_r = Lds::key_row(lane), k_c = imin(Lds::key_chunk(lane), HD / 8 - 1) * 16;
    const int v_r = Lds::value_row(lane), v_c = imin(Lds::value_chunk(lane), HD / 8 - 1) * 16;
    // page ids of the groups of a tile, a lane each: requested a tile ahead of their use
    auto request_pages = [&](int t) { return trow && t < t_end ? trow[imin(t * KT + imin(lane, NG - 1) * 16, kr.hi - 1) >> a.kv.page_shift] : 0; };
    struct Tile {
        int page, bad;  // the wave's own page; bit g: the page of group g is none
    };
    auto tile_of = [&](int ids) {
        Tile x{0, 0};
        if (trow) {
            const bool ok = (unsigned)ids < (unsigned)a.kv.n_pages;
            x.bad = (int)(__ballot(!ok) & ((1u << NG) - 1));
            x.page = __builtin_amdgcn_readlane(ok ? ids : 0, w * RW / 16);  // a page that is none: any that exists, whose values nobody sees
        }
        return x;
    };
    auto copy = [&](auto is_v, int t, int page, uint8_t *dst) __attribute__((always_inline)) {
        if (t >= t_end) return;
        constexpr bool V = decltype(is_v)::value;
        const int64_t rs = V ? a.kv.v_row : a.kv.k_row;
        const int g0 = imin(t * KT + w * RW, (kr.hi - 1) & ~(RW - 1)), n = kr.hi - g0;  // rows behind the last one seen: copies of it
        const uint8_t *src = V ? vbase : kbase;
        if (trow) src += page * a.kv.page + (g0 & ((1 << a.kv.page_shift) - 1)) * rs;
        else src += (sv.row0 + g0) * rs;
        const int cr = V ? v_r : k_r, cc = V ? v_c : k_c;
        uint8_t *d = dst + w * NLD * (V ? Lds::V_BLOCK : Lds::K_BLOCK);
#pragma unroll
        for (int i = 0; i < NLD; i++) copy_lds(src, imin(i * RPI + cr, n - 1) * (int)rs + cc, d + i * (V ? Lds::V_BLOCK : Lds::K_BLOCK));
    };
    using K_ = std::false_type;
    using V_ = std::true_type;

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = -FLT_MAX, l = 0;
    // exponent of a score in log2 units is s · c
    const float c = CAP ? 1.0f : a.scale * LOG2E_F, cap_in = CAP ? 2.0f * LOG2E_F * a.scale / a.softcap : 0.0f, cap_out = CAP ? a.softcap * LOG2E_F : 0.0f;
    // the lane's places in a tile: keys row-wise, values transposed
    const int k_at = Lds::key(lane & 31, h), v_at = Lds::value(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (lane & 1) * 8;

    f32x16 s[2];
    u32x4 pf[2][2];
    auto scores = [&](const uint8_t *kt, int kb, f32x16 &d) __attribute__((always_inline)) {
        d = f32x16{};
#pragma unroll
        for (int i = 0; i < KS; i++) d = mfma32<BF>(*(const u32x4 *)(kt + k_at + Lds::key(kb * 32, 2 * i)), qf[i], d);
    };
    auto outputs = [&](const uint8_t *vt, int kb, const u32x4 (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const uint8_t *vp = vt + v_at + Lds::value(kb * 32 + st * 16, 4 * d);
                const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(8, 0));
                o[d] = mfma32<BF>(u32x4{v0[0], v0[1], v1[0], v1[1]}, p[st], o[d]);
            }
    };
    // group (t, kb): probabilities of its scores x → p; outputs of the group before from values
    // (vt, vkb) and probabilities po; scores of the group behind from keys (kt, nkb) → y
    auto group = [&](int key0, int bad2, f32x16 &x, u32x4 (&p)[2], const u32x4 (&po)[2], f32x16 &y, const uint8_t *vt, int vkb, const uint8_t *kt, int nkb) __attribute__((always_inline)) {
        if constexpr (CAP) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = cap_score<CAP>(x[e], cap_in, cap_out);
        }
        // positions of the lane's scores: key0 + 4 h + (8 (e / 4) + e % 4)
        if (key0 + 31 > all_hi) {
            const int d = p_q - key0 - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = 8 * (e / 4) + e % 4 <= d ? x[e] : -INFINITY;
        }
        if (key0 <= all_lo) {
            const int d = lo_q - key0 - 4 * h;
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = 8 * (e / 4) + e % 4 > d ? x[e] : -INFINITY;
        }
        if (bad2) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = bad2 >> (e / 8) & 1 ? -INFINITY : x[e];
        }
        float mx = fmaxf(fmaxf(x[0], x[1]), x[2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) mx = fmaxf(fmaxf(mx, x[e]), x[e + 1]);
        mx = fmaxf(mx, x[15]) * c;
        const bool moved = __any(mx > m + M_SLACK);
        float al = 1;
        if (moved) {
            float a0, a1;
            pair_f<32>(mx, a0, a1);
            const float mn = fmaxf(m, fmaxf(a0, a1));
            al = exp2_hw(m - mn);
            m = mn;
            l *= al;
        }
        // Eight rounds of an output product and a score product, operands read two rounds ahead,
        // with a share of the probabilities after each: the fences keep the order.
        constexpr int NV = 2 * DB, NR = NV > KS ? NV : KS;
        y = f32x16{};
        const float ref = P_SHIFT<BF> - m;
        u32x4 kf[KS], vf[NV];
        auto read_v = [&](int u) {
            const uint8_t *vp = vt + v_at + Lds::value(vkb * 32 + u / DB * 16, u % DB * 4);
            const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(8, 0));
            vf[u] = u32x4{v0[0], v0[1], v1[0], v1[1]};
        };
        auto read_k = [&](int u) { kf[u] = *(const u32x4 *)(kt + k_at + Lds::key(nkb * 32, 2 * u)); };
        float ex[16];
        auto exps = [&](int i) {
            ex[2 * i] = exp2_hw(fmaf(x[2 * i], c, ref));
            ex[2 * i + 1] = exp2_hw(fmaf(x[2 * i + 1], c, ref));
        };
        auto pack = [&](int i) { p[i / 4][i % 4] = pack2<BF>(ex[2 * i], ex[2 * i + 1]); };
        auto add = [&](int i) { l = add2<BF>(p[i / 4][i % 4], l); };
#pragma unroll
        for (int i = 0; i < 2; i++) {
            read_v(i);
            read_k(i);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NR; i++) {
            if (i < NV) o[i % DB] = mfma32<BF>(vf[i], po[i / DB], o[i % DB]);
            if (i + 2 < NV) read_v(i + 2);
#pragma unroll
            for (int u = i * 8 / NR; u < (i + 1) * 8 / NR; u++) exps(u);
            __builtin_amdgcn_sched_barrier(0);
            if (i < KS) y = mfma32<BF>(kf[i], qf[i], y);
            if (i + 2 < KS) read_k(i + 2);
#pragma unroll
            for (int u = i * 8 / NR; u < (i + 1) * 8 / NR; u++) {
                pack(u);
                if (u) add(u - 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        add(7);
        // all three belong into this block: the compiler would move the probabilities to where
        // they are used, and make two copies of the block
        asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(l));
        int after = __builtin_amdgcn_readfirstlane(moved);
        asm volatile("" : "+s"(after));
        if (after) {  // the outputs so far were formed with the maximum before
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= al;
        }
    };
    // Infinite and NaN values of tile t, some of whose positions some row does not see: added
    // to the outputs of the rows that see them, then replaced by zeros.  All waves call this.
    auto apart = [&](int t, int bad, uint8_t *vt) __attribute__((always_inline)) {
        if ((t + 1) * KT - 1 <= wg_hi && t * KT > wg_lo && !bad) return;
        bool nf = false;
#pragma unroll
        for (int i = 0; i < NLD; i++) nf = nf || nonfinite8<BF>(*(const u32x4 *)(vt + (w * NLD + i) * Lds::V_BLOCK + lane * 16));
        const int f = __any(nf);
        if (lane == 0) s_nf[w] = f;
        lds_barrier();
        if (!__builtin_amdgcn_readfirstlane(s_nf[0] | s_nf[1] | s_nf[2] | s_nf[3])) return;
        for (int r = 0; r < KT; r++) {
            const int j = t * KT + r;
            const bool see = j <= p_q && j > lo_q && !(bad >> (r / 16) & 1);
            if (!__any(see)) continue;
            const uint8_t *vp = vt + Lds::value(r, 0) + 8 * h;
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) {  // dim 32 d + 8 (e / 4) + 4 h + e % 4
                    const float v = value16<BF>(*(const uint16_t *)(vp + Lds::value(0, 4 * d + e / 4) + e % 4 * 2));
                    o[d][e] += (see & !(fabsf(v) <= FLT_MAX)) ? v : 0.0f;
                }
        }
        lds_barrier();
#pragma unroll
        for (int i = 0; i < NLD; i++) {
            u32x4 *p = (u32x4 *)(vt + (w * NLD + i) * Lds::V_BLOCK + lane * 16);
            u32x4 v = *p;
            for (int e = 0; e < 4; e++) v[e] = finite2<BF>(v[e]);
            *p = v;
        }
        lds_barrier();
    };

    if (t_begin < t_end) {
        Tile cur = tile_of(request_pages(t_begin)), nxt = tile_of(request_pages(t_begin + 1));
        int ids = request_pages(t_begin + 2);
        int prev_bad = 0;  // KB = 1: of tile t − 1
        copy(K_{}, t_begin, cur.page, s_k0);
        copy(K_{}, t_begin + 1, nxt.page, s_k1);
        if constexpr (KB == 2) copy(V_{}, t_begin, cur.page, s_v0);
        // the first group's outputs before it: zeros
        for (int i = w; i < 32 / RPI; i += 4) *(u32x4 *)(s_v1 + Lds::value((KB - 1) * 32 + i * RPI, 0) + lane * 16) = u32x4{0, 0, 0, 0};
        pf[1][0] = pf[1][1] = u32x4{0, 0, 0, 0};
        wait_vmem();
        lds_barrier();
        if (wave_live) scores(s_k0, 0, s[0]);
        auto tile = [&](int t, uint8_t *k_t, uint8_t *k_n, uint8_t *v_t, uint8_t *v_n, f32x16 &x0, f32x16 &x1, u32x4 (&p0)[2], u32x4 (&p1)[2]) __attribute__((always_inline)) {
            if constexpr (KB == 2)
                if (wave_live) group(t * KT, cur.bad & 3, x0, p0, p1, x1, v_n, 1, k_t, 1);
            wait_vmem();
            lds_barrier();
            const Tile third = tile_of(ids);
            copy(K_{}, t + 2, third.page, k_t);
            if constexpr (KB == 2) copy(V_{}, t + 1, nxt.page, v_n);
            else copy(V_{}, t, cur.page, v_t);
            ids = request_pages(t + 3);
            if constexpr (KB == 2) {
                apart(t, cur.bad, v_t);
                if (wave_live) group(t * KT + 32, cur.bad >> 2, x1, p1, p0, x0, v_t, 0, k_n, 0);
            } else {
                if (t > t_begin) apart(t - 1, prev_bad, v_n);
                if (wave_live) group(t * KT, cur.bad, x0, p0, p1, x1, v_n, 0, k_n, 0);
                prev_bad = cur.bad;
            }
            cur = nxt;
            nxt = third;
        };
        int t = t_begin;
        for (; t < t_end; t += 2) {
            if constexpr (KB == 2) tile(t, s_k0, s_k1, s_v0, s_v1, s[0], s[1], pf[0], pf[1]);
            else tile(t, s_k0, s_k1, s_v0, s_v1, s[0], s[1], pf[0], pf[1]);
            if (t + 1 >= t_end) break;
            if constexpr (KB == 2) tile(t + 1, s_k1, s_k0, s_v1, s_v0, s[0], s[1], pf[0], pf[1]);
            else tile(t + 1, s_k1, s_k0, s_v1, s_v0, s[1], s[0], pf[1], pf[0]);
        }
        // the last group's outputs
        const bool odd = (t_end - t_begin) & 1;
        if constexpr (KB == 1) {
            wait_vmem();
            lds_barrier();
            apart(t_end - 1, prev_bad, odd ? s_v0 : s_v1);
        }
        if (wave_live) {
            if (odd) outputs(s_v0, KB - 1, pf[KB == 2 ? 1 : 0]);
            else outputs(s_v1, KB - 1, pf[1]);
        }
    }

    float l0, l1;
    pair_f<32>(l, l0, l1);
    l = l0 + l1;
    if (!live) return;
    if (ns == 1) {
        const float inv = l > 0 || l != l ? 1.0f / l : 0.0f;
        uint8_t *op = a.out + (int64_t)(sv.row0 + tok) * a.o_row + head * a.o_head + h * 8;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 v = {pack2<BF>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv), pack2<BF>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)};
                *(u32x2 *)(op + d * 64 + e * 16) = v;
            }
    } else {
        const int64_t at = ((int64_t)(sv.row0 + tok) * a.n_head + head) * a.S + sp;
        float *pp = a.part + at * HD + 4 * h;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) *(f32x4 *)(pp + d * 32 + e * 8) = f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
        if (h == 0) *(f32x2 *)(a.ml + at * 2) = f32x2{m, l};
    }
}

// At most 16·NB query rows of a sequence and KV head: each of the workgroup's 4 waves takes
// every fourth tile of 32 positions, and the waves' results are added up at the end.  Keys go
// from global memory straight to operand registers, values through the wave's own LDS; both
// are requested a tile ahead, so no barrier lies between the reading and the arithmetic.
constexpr int FEW_KT = 32, FEW_STEP = 4 * FEW_KT;

template <int HD, bool BF, bool CAP, int NB>
__global__ __launch_bounds__(256) void attn_few_kernel(ServeAttnArgs a) {
    constexpr int KT = FEW_KT, NLD = KT * HD / 8 / 64, ROWB = HDP<HD> * 2, KS = HD / 32, DB = HD / 16;
    constexpr int VB = KT * ROWB, OB = 16 * NB * HD * 4;  // a wave's values, and its outputs at the end
    constexpr int WB = VB > OB ? VB : OB;
    __shared__ __align__(16) uint8_t s_buf[4][WB];
    __shared__ float s_ml[4][16 * NB][2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    const int G = a.G, kvh = blockIdx.x % a.n_kv, si = blockIdx.x / a.n_kv;
    const SeqView sv = view_of(a.b, a.kv, si);
    const int n_rows = imin(sv.n_new * G, 16 * NB);
    if (n_rows == 0) return;
    const int n_tok = (n_rows + G - 1) / G, pos0 = sv.len - sv.n_new;
    const KeyRange kr = key_range(sv, 0, n_tok - 1, a.window);
    const int t0 = first_tile(kr, FEW_STEP), nt = tile_count(kr, FEW_STEP), ns = split_count(nt, a.C, a.S), sp = blockIdx.y;
    if (sp >= ns) return;
    const int begin = (t0 + sp * a.C) * 4 + w, end = imin((sp == ns - 1 ? t0 + nt : t0 + (sp + 1) * a.C) * 4, (kr.hi + KT - 1) / KT);

    int p_q[NB], lo_q[NB];
    u32x4 qf[NB][KS];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int row = b * 16 + col, tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
        const bool live = row < n_rows;
        p_q[b] = live ? pos0 + tok : -1;
        lo_q[b] = a.window > 0 ? p_q[b] - a.window : -1;
        const uint8_t *qp = a.q + (int64_t)(sv.row0 + tok) * a.q_row + head * a.q_head + g * 16;
#pragma unroll
        for (int i = 0; i < KS; i++) qf[b][i] = live ? *(const u32x4 *)(qp + i * 64) : u32x4{0, 0, 0, 0};
    }
    const int all_hi = pos0, all_lo = a.window > 0 ? pos0 + n_tok - 1 - a.window : -1;

    const int *trow = a.kv.table ? a.kv.table + (int64_t)si * a.kv.table_stride : nullptr;
    const uint8_t *kbase = a.kv.k + kvh * a.kv.k_head, *vbase = a.kv.v + kvh * a.kv.v_head;
    uint8_t *sv_t = s_buf[w];
    u32x4 rk[2][KS], rv[NLD];
    int r_bad = 0;  // bit b: the tile's 16 positions b lie in a page that is none
    auto load = [&](int t) {
        r_bad = 0;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int g0 = t * KT + b * 16;
            const uint8_t *kp = kbase, *vp = vbase;
            bool ok = true;
            if (g0 < kr.hi) {
                int page;
                ok = page_of(a.kv, trow, g0, page);
                const int slot = g0 & ((1 << a.kv.page_shift) - 1);
                kp += page * a.kv.page + slot * a.kv.k_row;
                vp += page * a.kv.page + slot * a.kv.v_row;
            }
            if (!ok) r_bad |= 1 << b;
            const int n = ok ? kr.hi - g0 : 0;
#pragma unroll
            for (int i = 0; i < KS; i++) {
                rk[b][i] = u32x4{0, 0, 0, 0};
                if (col < n) rk[b][i] = *(const u32x4 *)(kp + col * (int)a.kv.k_row + i * 64 + g * 16);
            }
#pragma unroll
            for (int i = 0; i < NLD / 2; i++) {
                const int r = (i * 64 + lane) / (HD / 8), ch = (i * 64 + lane) % (HD / 8);
                rv[b * (NLD / 2) + i] = u32x4{0, 0, 0, 0};
                if (r < n) rv[b * (NLD / 2) + i] = *(const u32x4 *)(vp + r * (int)a.kv.v_row + ch * 16);
            }
        }
    };

    f32x4 o[NB][DB];
    float m[NB], l[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        m[b] = -FLT_MAX;
        l[b] = 0;
#pragma unroll
        for (int d = 0; d < DB; d++) o[b][d] = f32x4{};
    }
    const float c = CAP ? 1.0f : a.scale * LOG2E_F, cap_in = CAP ? 2.0f * LOG2E_F * a.scale / a.softcap : 0.0f, cap_out = CAP ? a.softcap * LOG2E_F : 0.0f;
    const int vr = 4 * g + (col >> 2);
    const int va = vr * ROWB + (lane & 1) * 8, vx = ((lane & 3) >> 1) ^ swz_v<HD>(vr);

    if (begin < end) load(begin);
    for (int t = begin; t < end; t += 4) {
        const int key0 = t * KT, bad = r_bad;
        const bool part = key0 + KT - 1 > all_hi || key0 <= all_lo || bad;  // some row does not see all of the tile
        f32x4 s[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                s[b][kb] = f32x4{};
#pragma unroll
                for (int i = 0; i < KS; i++) s[b][kb] = mfma16<BF>(rk[kb][i], qf[b][i], s[b][kb]);
            }
        bool nf = false;
#pragma unroll
        for (int i = 0; i < NLD; i++) {
            const int r = i / (NLD / 2) * 16 + (i % (NLD / 2) * 64 + lane) / (HD / 8), ch = (i % (NLD / 2) * 64 + lane) % (HD / 8);
            *(u32x4 *)(sv_t + r * ROWB + ((ch ^ swz_v<HD>(r)) << 4)) = rv[i];
            if (part) nf = nf || nonfinite8<BF>(rv[i]);
        }
        wave_sync();
        if (t + 4 < end) load(t + 4);
        if (part && __any(nf)) {  // rare
            for (int r = 0; r < KT; r++) {
                const int j = key0 + r;
                const uint8_t *vp = sv_t + r * ROWB;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const bool see = j <= p_q[b] && j > lo_q[b] && !(bad >> (r / 16) & 1);
                    if (!__any(see)) continue;
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int dim = d * 16 + 4 * g + e;
                            const float x = value16<BF>(*(const uint16_t *)(vp + (((dim >> 3) ^ swz_v<HD>(r)) << 4) + (dim & 7) * 2));
                            if (see && !(fabsf(x) <= FLT_MAX)) o[b][d][e] += x;
                        }
                }
            }
            wave_sync();
#pragma unroll
            for (int i = 0; i < NLD; i++) {
                const int r = i / (NLD / 2) * 16 + (i % (NLD / 2) * 64 + lane) / (HD / 8), ch = (i % (NLD / 2) * 64 + lane) % (HD / 8);
                u32x4 *p = (u32x4 *)(sv_t + r * ROWB + ((ch ^ swz_v<HD>(r)) << 4));
                u32x4 x = *p;
                for (int e = 0; e < 4; e++) x[e] = finite2<BF>(x[e]);
                *p = x;
            }
            wave_sync();
        }
        u32x4 pf[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (CAP) s[b][kb][e] = cap_score<CAP>(s[b][kb][e], cap_in, cap_out);
                    if (part) {
                        const int j = key0 + kb * 16 + 4 * g + e;
                        if (j > p_q[b] || j <= lo_q[b] || (bad >> kb & 1)) s[b][kb][e] = -INFINITY;
                    }
                    mx = fmaxf(mx, s[b][kb][e]);
                }
            mx *= c;
            if (__any(mx > m[b] + M_SLACK)) {
                float x0, x1, y0, y1;
                pair_f<16>(mx, x0, x1);
                pair_f<32>(fmaxf(x0, x1), y0, y1);
                const float mn = fmaxf(m[b], fmaxf(y0, y1)), al = exp2_hw(m[b] - mn);
                m[b] = mn;
                l[b] *= al;
#pragma unroll
                for (int d = 0; d < DB; d++) o[b][d] *= al;
            }
            const float ref = P_SHIFT<BF> - m[b];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                pf[b][e] = pack2<BF>(exp2_hw(fmaf(s[b][e / 2][2 * (e & 1)], c, ref)), exp2_hw(fmaf(s[b][e / 2][2 * (e & 1) + 1], c, ref)));
                l[b] = add2<BF>(pf[b][e], l[b]);
            }
        }
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const uint8_t *vp = sv_t + va + ((vx ^ (2 * d)) << 4);
            const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + 16 * ROWB);
#pragma unroll
            for (int b = 0; b < NB; b++) o[b][d] = mfma16<BF>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pf[b], o[b][d]);
        }
        wave_sync();
    }

    // the four waves' results
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float x0, x1, y0, y1;
        pair_f<16>(l[b], x0, x1);
        pair_f<32>(x0 + x1, y0, y1);
        float *po = (float *)sv_t + (b * 16 + col) * HD + 4 * g;
#pragma unroll
        for (int d = 0; d < DB; d++) *(f32x4 *)(po + d * 16) = o[b][d];
        if (g == 0) {
            s_ml[w][b * 16 + col][0] = m[b];
            s_ml[w][b * 16 + col][1] = y0 + y1;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n_rows * (HD / 4); i += 256) {
        const int r = i / (HD / 4), d4 = i % (HD / 4), tok = r / G, head = kvh * G + r - tok * G;
        float mm = s_ml[0][r][0];
#pragma unroll
        for (int k = 1; k < 4; k++) mm = fmaxf(mm, s_ml[k][r][0]);
        f32x4 acc = f32x4{};
        float L = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = exp2_hw(s_ml[k][r][0] - mm);
            L = fmaf(f, s_ml[k][r][1], L);
            const f32x4 x = *(const f32x4 *)((const float *)s_buf[k] + r * HD + d4 * 4);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = fmaf(f, x[e], acc[e]);
        }
        if (ns == 1) {
            const float inv = L > 0 || L != L ? 1.0f / L : 0.0f;
            uint8_t *op = a.out + (int64_t)(sv.row0 + tok) * a.o_row + head * a.o_head + d4 * 8;
            *(u32x2 *)op = u32x2{pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
        } else {
            const int64_t at = ((int64_t)(sv.row0 + tok) * a.n_head + head) * a.S + sp;
            *(f32x4 *)(a.part + at * HD + d4 * 4) = acc;
            if (d4 == 0) *(f32x2 *)(a.ml + at * 2) = f32x2{mm, L};
        }
    }
}

// The splits of each (row, head), added up: a wave takes one, lane l the values l·HD/64 …
// M rows per block and KT positions per tile are those of the kernel that made the partials.
template <bool BF>
__global__ __launch_bounds__(256) void serve_combine_kernel(ServeAttnArgs a, int M, int KT) {
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = id / a.n_head, head = id - row * a.n_head, G = a.G;
    if (row >= a.b.n_rows) return;
    const int si = wave_find(a.b.starts, a.b.n_seq, row, [&](int s, int) { return iclamp(s, 0, a.b.n_rows); });
    const SeqView sv = view_of(a.b, a.kv, si);
    if (row < sv.row0 || row >= sv.row0 + sv.n_new) return;
    const int r = (row - sv.row0) * G + head % G, n_rows = sv.n_new * G, r0 = r / M * M, r1 = imin(r0 + M, n_rows) - 1;
    const int ns = split_count(tile_count(key_range(sv, r0 / G, r1 / G, a.window), KT), a.C, a.S);
    if (ns == 1) return;
    const int64_t at = ((int64_t)row * a.n_head + head) * a.S;
    const f32x2 ml = lane < ns ? *(const f32x2 *)(a.ml + (at + lane) * 2) : f32x2{-FLT_MAX, 0};
    const float mm = xmax_f<64>(ml[0]), f = exp2_hw(ml[0] - mm);
    const float L = xsum_f<64>(lane < ns ? f * ml[1] : 0.0f);
    const float inv = L > 0 || L != L ? 1.0f / L : 0.0f;
    uint8_t *op = a.out + (int64_t)row * a.o_row + head * a.o_head;
    for (int d = lane * 2; d < a.hd; d += 128) {
        f32x2 acc = f32x2{};
        for (int s = 0; s < ns; s++) {
            const f32x2 x = *(const f32x2 *)(a.part + (at + s) * a.hd + d);
            const float fs = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s));
            acc[0] = fmaf(fs, x[0], acc[0]);
            acc[1] = fmaf(fs, x[1], acc[1]);
        }
        *(uint32_t *)(op + d * 2) = pack2<BF>(acc[0] * inv, acc[1] * inv);
    }
}

// New rows into their pages: a wave per token row, 8 values of K or V per lane and step.
template <int SRC, bool BF>  // SRC: bytes of a source value
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= a.b.n_rows) return;
    const int si = wave_find(a.b.starts, a.b.n_seq, row, [&](int s, int) { return iclamp(s, 0, a.b.n_rows); });
    const SeqView sv = view_of(a.b, a.kv, si);
    if (row < sv.row0 || row >= sv.row0 + sv.n_new) return;
    const int pos = sv.len - sv.n_new + row - sv.row0;
    int page;
    if (pos < 0 || !page_of(a.kv, a.kv.table + (int64_t)si * a.kv.table_stride, pos, page)) return;
    const int64_t slot = pos & ((1 << a.kv.page_shift) - 1);
    const int per = a.hd / 8, n = a.n_kv * per;
    for (int i = lane; i < 2 * n; i += 64) {
        const bool is_v = i >= n;
        const int x = is_v ? i - n : i, h = x / per, ch = x - h * per;
        const uint8_t *src = is_v ? a.v + row * a.v_row + h * a.v_head : a.k + row * a.k_row + h * a.k_head;
        uint8_t *dst = const_cast<uint8_t *>(is_v ? a.kv.v + h * a.kv.v_head + slot * a.kv.v_row : a.kv.k + h * a.kv.k_head + slot * a.kv.k_row) + page * a.kv.page;
        u32x4 y;
        if constexpr (SRC == 4) {
            const f32x4 u = *(const f32x4 *)(src + ch * 32), v = *(const f32x4 *)(src + ch * 32 + 16);
            y = u32x4{pack2<BF>(u[0], u[1]), pack2<BF>(u[2], u[3]), pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3])};
        } else {
            y = *(const u32x4 *)(src + ch * 16);
        }
        *(u32x4 *)(dst + ch * 16) = y;
    }
}

template <int HD, bool BF>
void launch_hd(const ServeAttnArgs &a, hipStream_t st) {
    const bool cap = a.softcap > 0;
    if (serve_attn_few(a)) {
        const dim3 grid(a.b.n_seq * a.n_kv, a.S);
        if (a.b.max_new * a.G <= 16) {
            if (cap) attn_few_kernel<HD, BF, true, 1><<<grid, 256, 0, st>>>(a);
            else attn_few_kernel<HD, BF, false, 1><<<grid, 256, 0, st>>>(a);
        } else {
            if (cap) attn_few_kernel<HD, BF, true, 2><<<grid, 256, 0, st>>>(a);
            else attn_few_kernel<HD, BF, false, 2><<<grid, 256, 0, st>>>(a);
        }
    } else {
        const dim3 grid(a.n_blocks * a.n_kv, a.S);
        if (cap) attn_tile_kernel<HD, BF, true><<<grid, 256, 0, st>>>(a);
        else attn_tile_kernel<HD, BF, false><<<grid, 256, 0, st>>>(a);
    }
}

template <bool BF>
void launch_ty(const ServeAttnArgs &a, hipStream_t st) {
    switch (a.hd) {
    case 32: launch_hd<32, BF>(a, st); break;
    case 64: launch_hd<64, BF>(a, st); break;
    case 96: launch_hd<96, BF>(a, st); break;
    case 128: launch_hd<128, BF>(a, st); break;
    default: launch_hd<256, BF>(a, st); break;
    }
}

int tile_kt(int hd) { return hd <= 128 ? TILE_KT<128> : TILE_KT<256>; }

}  // namespace

bool serve_attn_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

bool serve_attn_few(const ServeAttnArgs &a) { return a.kv.table && (int64_t)a.b.max_new * a.G <= 32; }

SplitPlan serve_attn_splits(const ServeAttnArgs &a) {
    const bool few = serve_attn_few(a);
    const int KT = few ? FEW_STEP : tile_kt(a.hd);
    const int64_t blocks = few ? a.b.n_seq : block_count(a.b.n_rows, a.b.n_seq, a.G, TILE_M);
    // positions that a block's rows see, at most
    int64_t span = a.b.max_len;
    if (a.window > 0) span = std::min<int64_t>(span, (int64_t)a.window + std::min<int64_t>(a.b.max_new, few ? 32 : TILE_M / a.G + 1) + KT);
    const int tiles = (int)((span + KT - 1) / KT);
    return few ? split_plan(blocks * a.n_kv, tiles, 1024, 1, SERVE_MAX_SPLIT) : split_plan(blocks * a.n_kv, tiles, 512, 4, SERVE_MAX_SPLIT);
}

size_t serve_attn_ws(const ServeAttnArgs &a) {
    const SplitPlan p = serve_attn_splits(a);
    return p.S == 1 ? 0 : (size_t)a.b.n_rows * a.n_head * p.S * (a.hd + 2) * sizeof(float);
}

void launch_serve_attn(ServeAttnArgs a, void *ws, hipStream_t st) {
    const SplitPlan p = serve_attn_splits(a);
    const bool few = serve_attn_few(a);
    a.C = p.C;
    a.S = p.S;
    a.part = (float *)ws;
    a.ml = a.part + (size_t)a.b.n_rows * a.n_head * p.S * a.hd;
    a.n_blocks = (int)block_count(a.b.n_rows, a.b.n_seq, a.G, TILE_M);
    const bool bf = a.ty == T_BF16;
    if (bf) launch_ty<true>(a, st);
    else launch_ty<false>(a, st);
    if (p.S > 1) {
        const int M = few ? 32 : TILE_M, KT = few ? FEW_STEP : tile_kt(a.hd), grid = (int)(((int64_t)a.b.n_rows * a.n_head + 3) / 4);
        if (bf) serve_combine_kernel<true><<<grid, 256, 0, st>>>(a, M, KT);
        else serve_combine_kernel<false><<<grid, 256, 0, st>>>(a, M, KT);
    }
}

void launch_paged_append(const PagedAppendArgs &a, hipStream_t st) {
    const int grid = (a.b.n_rows + 3) / 4;
    if (a.src_ty == T_F32) {
        if (a.ty == T_BF16) paged_append_kernel<4, true><<<grid, 256, 0, st>>>(a);
        else paged_append_kernel<4, false><<<grid, 256, 0, st>>>(a);
    } else {
        paged_append_kernel<2, false><<<grid, 256, 0, st>>>(a);
    }
}

}  // namespace rie
