// serve_attn.hip — causal grouped-query attention of a batch of sequences over a cache
// of pages, or over packed prompts whose keys and values lie beside the queries:
//
//   o_t = Σ_j softmax_j(s_tj) v_j,  s_tj = scale · q_t·k_j  (cap · tanh(s / cap) with a softcap)
//
// over the positions j ≤ p_t, and j > p_t − window with a window, of token t at position
// p_t of its sequence.  A token that sees nothing, or nothing above −inf, gets zeros.  q, k, v and o are all f16
// or all bf16; scores, the softmax's maximum and sum, and the outputs are f32 sums.
//
// Rounding.  In the tile kernel a probability enters the second product in the tensors' own
// type, rounded to nearest; the sum that the output is divided by adds the same rounded values,
// so that a row's weights add up to one.  The error this brings is about that of rounding the
// output once more (2-norm against float64, bf16: 2.1e-3, the output's own rounding 1.6e-3).
// The few-rows kernel takes what that rounding leaves as a second product, its matrix units
// being idle (1.6e-3 and 1.6e-3).  The maximum that is subtracted is only moved when a score
// passes it by 2^8, so a probability lies in 0..2^8; f16 ones are multiplied by 2^6, since
// small ones would be subnormal, bf16 ones by 2^-32 (P_SHIFT).
//
// Values that are infinite or NaN reach the tokens that see them and no others: a tile that
// some token sees in part is searched for them, and if there are any, they are added to the
// outputs one by one and replaced by zeros in the matrix product, where they would meet
// probabilities of zero.  Outputs that are NaN all the same are formed from the infinite and NaN
// values alone at the end (NonFinite).
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

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
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

// Addresses in LDS as numbers: sums with constants become the instructions' offsets, where
// generic pointers take a register for every one, 50 to 70 of them in the tile kernel, which
// then holds all 256 (and one more is a spill whose reload waits for the copies: 219 to 272 us
// for chunks in a batch of 13; 202 without a spill, 219 here with 209 vector registers; scalars,
// 45 to 62 of them from head size 96 on, are kept in lanes of vector registers; four prompts
// of 64-wide heads, 3 waves on a SIMD instead of 2: 187, with pointers 201).
__device__ __forceinline__ uint32_t lds_at(const void *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t *)p; }
__device__ __forceinline__ u32x4 lds_16(uint32_t at) { return *(__attribute__((address_space(3))) const u32x4 *)(uintptr_t)at; }
// 4 values of one column: lane l of a group of 16 lanes names the 8 bytes of row l / 4 that
// hold columns 4·(l % 4) …, and gets rows 0..3 of column l
__device__ __forceinline__ u32x2 read_tr(uint32_t at) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(uintptr_t)at));
}
// Probabilities are 2^(s − m + P_SHIFT).  bf16 ones are made so small that no sum over 2^24 positions
// passes the largest value, which may be the largest of f32; they have its exponents.  What that
// takes at the other end: terms under 2^-126, which are values under 2^-94, may count as zeros.
template <bool BF>
constexpr float P_SHIFT = BF ? -32.0f : 6.0f;
constexpr float M_SLACK = 8.0f;  // how far a score may pass the maximum that is subtracted

__device__ __forceinline__ SeqView uniform(const SeqView &v) {
    return SeqView{__builtin_amdgcn_readfirstlane(v.row0), __builtin_amdgcn_readfirstlane(v.n_new), __builtin_amdgcn_readfirstlane(v.len),
                   __builtin_amdgcn_readfirstlane(v.over)};
}
// x, the same for the whole wave, where the compiler cannot see it (behind divisions, say):
// kept in a scalar register, with branches on it that are no masks
__device__ __forceinline__ int same(int x) { return __builtin_amdgcn_readfirstlane(x); }
// positions that a sequence can have (packed rows: as many as it has rows)
__device__ __forceinline__ SeqView view_at(const BatchView &b, const KvView &kv, int start, int end, int len) {
    SeqView v = seq_view(start, end, len, b.n_rows, kv.table ? kv.cap : INT32_MAX);
    if (!kv.table) v.len = v.n_new;
    return uniform(v);
}
__device__ __forceinline__ SeqView view_of(const BatchView &b, const KvView &kv, int i) {
    return view_at(b, kv, b.starts[i], b.starts[i + 1], b.lens ? b.lens[i] : 0);
}
// The sequence with the largest number i that has key(starts[i], i) ≤ x, for keys that rise
// with i (0 where there is none): 63 candidates at a time, one per lane, whose starts, ends
// and lengths are there at once when so few are left.
template <class F>
__device__ __forceinline__ SeqView find_seq(const BatchView &b, const KvView &kv, int x, int &si, F key) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = b.n_seq;
    while (n > 63) {
        const int w = (n + 62) / 63, i = lane * w;
        const bool le = lane < 63 && i < n && key(b.starts[lo + imin(i, n - 1)], lo + imin(i, n - 1)) <= x;
        const int c = imax((int)__popcll(__ballot(le)) - 1, 0);
        lo += c * w;
        n = imin(w, n - c * w);
    }
    const int i = lo + imin(lane, n), start = b.starts[i], len = b.lens ? b.lens[imin(i, b.n_seq - 1)] : 0;
    const int c = __builtin_amdgcn_readfirstlane(imax((int)__popcll(__ballot(lane < n && key(start, i) <= x)) - 1, 0));
    si = lo + c;
    return view_at(b, kv, __builtin_amdgcn_readlane(start, c), __builtin_amdgcn_readlane(start, c + 1), __builtin_amdgcn_readlane(len, c));
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
// Outputs that came out as NaN, of rows whose probabilities' sum is a number: an infinite value
// has met a probability that was rounded to zero, or a rounding's remainder of either sign, or
// there is a NaN.  The true one is the sum of the infinite and NaN values at the positions that
// its token sees (NaN itself where there are none).  A wave searches them once for all of its
// rows: the positions that every row sees 16 bytes to a lane, into sums that the rows share; of
// those at either end that only some see, 31 at most (a wave's rows are of 32 tokens at most),
// which ones hold such a value.  A prompt of 3000 tokens, 32 heads on 8 of 128: 107 us, with a
// NaN row at its start 412, with nothing but NaN 589; 4 tokens over 40000 positions 40, 129, 152.
// The kernels' arguments are read here again (late_args): kept for this from the start they would
// be spilled, and read back in the loops.
typedef const __attribute__((address_space(4))) ServeAttnArgs *LateArgs;
__device__ __forceinline__ LateArgs late_args() {
    auto *a = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}
template <int HD, bool BF>
struct NonFinite {
    float sum[8];   // over positions [s0, s1), of the 8 dims of chunk (lane % CPR)
    uint64_t some;  // bit b: position(b) holds an infinite or NaN value
    int u0, s0, s1;

    __device__ __forceinline__ int position(int b) const { return b < s0 - u0 ? u0 + b : s1 + b - (s0 - u0); }
    // sequence si's values of KV head kvh at position j, or nullptr; row0: its first row, in packed prompts
    static __device__ __forceinline__ const uint8_t *row(LateArgs a, int si, int row0, int kvh, int j) {
        const uint8_t *v = a->kv.v + kvh * a->kv.v_head;
        if (!a->kv.table) return v + (int64_t)(row0 + j) * a->kv.v_row;
        const int page = a->kv.table[(int64_t)si * a->kv.table_stride + (j >> a->kv.page_shift)];
        if ((unsigned)page >= (unsigned)a->kv.n_pages) return nullptr;
        return v + page * a->kv.page + (j & ((1 << a->kv.page_shift) - 1)) * a->kv.v_row;
    }
    static __device__ __forceinline__ float kept(uint32_t bits) {
        const float x = value16<BF>(bits);
        return fabsf(x) <= FLT_MAX ? 0.0f : x;
    }
    // Some row sees [from, to), all rows [all_from, all_to); the positions of the launch's split are
    // [lo, hi).  The same for the wave, and all of its lanes call this.
    __device__ __forceinline__ void search(LateArgs a, int si, int row0, int kvh, int from, int to, int all_from, int all_to, int lo, int hi) {
        constexpr int CPR = HDP<HD> / 8, RPI = 64 / CPR, AT_ONCE = 4;
        const int lane = threadIdx.x & 63, c = imin(lane % CPR, HD / 8 - 1) * 16, r = lane / CPR;
        u0 = imax(from, lo);
        const int u1 = imax(imin(to, hi), u0);
        s0 = iclamp(all_from, u0, u1);
        s1 = iclamp(all_to, s0, u1);
#pragma unroll
        for (int e = 0; e < 8; e++) sum[e] = 0;
        for (int j0 = s0; j0 < s1; j0 += AT_ONCE * RPI) {
            u32x4 x[AT_ONCE];
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++) {
                const int j = j0 + i * RPI + r;
                const uint8_t *p = j < s1 ? row(a, si, row0, kvh, j) : nullptr;
                x[i] = p ? *(const u32x4 *)(p + c) : u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < AT_ONCE; i++)
                if (nonfinite8<BF>(x[i]))
#pragma unroll
                    for (int e = 0; e < 8; e++) sum[e] += kept(x[i][e / 2] >> (e & 1) * 16 & 0xFFFF);
        }
#pragma unroll
        for (int o = CPR; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] += __shfl_xor(sum[e], o);
        const int j = position(lane);
        const uint8_t *p = j < (lane < s0 - u0 ? s0 : u1) ? row(a, si, row0, kvh, j) : nullptr;
        bool any = false;
        if (p)
            for (int i = 0; i < HD / 8; i++) any = any || nonfinite8<BF>(*(const u32x4 *)(p + i * 16));
        some = __ballot(any);
    }
    // of dims 8 c + 4 half …, for a row that sees positions (lo, hi]; all lanes call this
    __device__ __forceinline__ f32x4 of(LateArgs a, int si, int row0, int kvh, int c, int half, int lo, int hi) const {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float s_lo = __shfl(sum[e], c), s_hi = __shfl(sum[4 + e], c);
            x[e] = half ? s_hi : s_lo;
        }
        for (uint64_t m = some; m; m &= m - 1) {
            const int j = position(__builtin_ctzll(m));
            if (j <= lo || j > hi) continue;
            const u32x2 y = *(const u32x2 *)(row(a, si, row0, kvh, j) + c * 16 + half * 8);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] += kept(y[e / 2] >> (e & 1) * 16 & 0xFFFF);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = x[e] == 0 ? NAN : x[e];
        return x;
    }
};

// score → exponent in log2 units where there is a softcap (the same score where there is none).
// With x = score / cap, cap · tanh(x) is score · (1 − x²/3 + 2x⁴/15 − 17x⁶/315) for |x| under 0.2
// (the next term is 2^-24), and cap · (1 − 2 / (e^2x + 1)) beyond, whose difference keeps 2^-22 of
// the cap: of a score that is a small part of a large cap it would keep nothing.  A scale by cap
// beyond the range of f32 is cut there, so that a score of 0 stays 0.
struct SoftCap {
    float in, lin, out;
};
__device__ __forceinline__ SoftCap soft_cap(const ServeAttnArgs &a) {
    return SoftCap{fminf(a.scale / a.softcap, FLT_MAX), a.scale * LOG2E_F, fminf(a.softcap * LOG2E_F, FLT_MAX)};
}
template <bool CAP>
__device__ __forceinline__ float cap_score(float s, const SoftCap &k) {
    if constexpr (!CAP) return s;
    const float x = s * k.in, t = x * x, e = exp2_hw(x * (2.0f * LOG2E_F));
    const float near = s * k.lin * fmaf(fmaf(fmaf(-17.0f / 315.0f, t, 2.0f / 15.0f), t, -1.0f / 3.0f), t, 1.0f);
    const float far = k.out * fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return fabsf(x) < 0.2f ? near : far;
}

// 16 bytes per lane from global memory (base + off) to LDS: lane l's go to dst + 16·l, with base
// and dst the same for the wave.  Written as the instruction, since the compiler waits for the
// builtin's copies before it reads any LDS, also of the buffers that they do not write; it has
// no result register, and the callers wait (wait_vmem) before the barrier behind which the
// copy is read.  Loads return in order, so waits that count without these wait longer at most.
__device__ __forceinline__ void copy_lds(const uint8_t *base, int off, const uint8_t *dst) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(lds_at(dst));
    const uint64_t from = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32)) << 32 |
                          (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(at), "v"(off), "s"(from) : "m0", "memory");
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
//
// Four packed prompts of up to 5000 tokens, 32 heads on 8 of 128, bf16: 428 us, 890 TFLOP/s
// (381 GFLOP), three quarters of what a library product of 8192 reaches on the card; 486 us
// with tiles staged through registers and the steps one behind the other.  Counters: matrix
// units busy 39 % of the cycles, vector units about as much, LDS 21 %, a quarter of the waves'
// time in waits.  Four buffers of 32 positions instead of two of 64 (loads three tiles ahead, a
// barrier every 32 positions): 429 us, and 248 for 208 us on chunks over pages; products in
// turns instead of scores first: 430; the next products' operands read 5 ahead: 427.
template <int HD, bool BF, bool CAP>
__global__ __launch_bounds__(256, HD <= 128 ? 2 : 1) void attn_tile_kernel(ServeAttnArgs a) {
    constexpr int KT = TILE_KT<HD>, KB = KT / 32, RW = KT / 4, KS = HD / 16, DB = HD / 32;
    using Lds = TileLds<HD>;
    constexpr int RPI = Lds::RPI, NLD = RW / RPI, KBYTES = KT / RPI * Lds::K_BLOCK, VBYTES = KT / RPI * Lds::V_BLOCK;
    constexpr int NG = KT / 16;  // groups of 16 positions, which lie in one page
    __shared__ __align__(16) uint8_t s_k0[KBYTES], s_k1[KBYTES], s_v0[VBYTES], s_v1[VBYTES];
    __shared__ __align__(16) int s_nf[4];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    // the splits of a block side by side, and a KV head's workgroups on one XCD where there are 8 of them
    const int G = a.G, kvh = blockIdx.x % a.n_kv, sp = blockIdx.x / a.n_kv % a.S, blk = blockIdx.x / a.n_kv / a.S;
    int si;
    const SeqView sv = find_seq(a.b, a.kv, blk, si, [&](int s, int i) { return block_base(iclamp(s, 0, a.b.n_rows), i, G, TILE_M); });
    const int n_rows = sv.n_new * G;
    const int lb = (n_rows + TILE_M - 1) / TILE_M - 1 - (blk - block_base(sv.row0, si, G, TILE_M));  // a sequence's longest rows first
    if (lb < 0 || lb >= (n_rows + TILE_M - 1) / TILE_M) return;
    const int r0 = same(lb * TILE_M), r1 = same(imin(r0 + TILE_M, n_rows) - 1), tok0 = same(r0 / G), tok1 = same(r1 / G);
    const int pos0 = sv.pos0();  // position of token 0
    const KeyRange kr = key_range(sv, tok0, tok1, a.window);
    const int hi = same(kr.hi), nt = same(tile_count(kr, KT)), ns = same(split_count(nt, a.C, a.S));
    if (sp >= ns) return;
    const int t_first = same(first_tile(kr, KT)), t_begin = t_first + sp * a.C, t_end = sp == ns - 1 ? t_first + nt : t_begin + a.C;

    // this lane's query row, and what the rows of its wave see
    const int row = r0 + w * 32 + (lane & 31);
    const bool live = row < n_rows;
    const int tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
    const int p_q = live ? imin(pos0 + tok, sv.len - 1) : -1;
    const int lo_q = before_window(pos0 + tok, a.window);  // sees j in (lo_q, p_q]
    const bool wave_live = r0 + w * 32 <= r1;
    const int w_t0 = same(imin(r0 + w * 32, r1) / G), w_t1 = same(imin(r0 + w * 32 + 31, r1) / G);
    const int all_hi = imin(pos0 + w_t0, sv.len - 1), all_lo = before_window(pos0 + w_t1, a.window);  // every row of the wave sees (all_lo, all_hi]
    const int wg_hi = imin(pos0 + tok0, sv.len - 1), wg_lo = before_window(pos0 + tok1, a.window);    // and of the workgroup
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
    const int k_row = (int)a.kv.k_row, v_row = (int)a.kv.v_row, k_off = k_r * k_row + k_c, v_off = v_r * v_row + v_c;
    // Page ids of a tile's groups of 16 positions, a lane each, requested a tile ahead of their
    // use (ids that stay in a register for several tiles, 64 pages at once, made the compiler
    // wait for all copies where their loads join the loop: 424 to 461 us for four packed prompts).
    const int page_mask = (1 << a.kv.page_shift) - 1;
    auto request_pages = [&](int t) __attribute__((always_inline)) {
        return trow && t < t_end ? trow[imin(t * KT + imin(lane, NG - 1) * 16, hi - 1) >> a.kv.page_shift] : 0;
    };
    // a tile's place in memory for this wave's rows, and (bit g) which of its groups of 16
    // positions lie in a page that is none (one that exists is read, and nobody sees its values)
    struct Tile {
        int64_t k, v;
        int rows, bad;  // rows: how many of the wave's are seen by some token
    };
    auto tile_of = [&](int t, int ids) __attribute__((always_inline)) {
        const int g0 = imin(t * KT + w * RW, (hi - 1) & ~(RW - 1));  // rows behind the last one seen: copies of it
        Tile x;
        x.rows = hi - g0;
        x.bad = 0;
        if (trow) {
            const bool ok = (unsigned)ids < (unsigned)a.kv.n_pages;
            x.bad = same((int)(__ballot(!ok) & ((1u << NG) - 1)));
            const int64_t page = __builtin_amdgcn_readlane(ok ? ids : 0, w * RW / 16), slot = g0 & page_mask;
            x.k = page * a.kv.page + slot * a.kv.k_row;
            x.v = page * a.kv.page + slot * a.kv.v_row;
        } else {
            x.k = (int64_t)(sv.row0 + g0) * a.kv.k_row;
            x.v = (int64_t)(sv.row0 + g0) * a.kv.v_row;
        }
        return x;
    };
    auto copy = [&](auto is_v, const uint8_t *src, int rows, uint8_t *dst) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
        constexpr int BLOCK = V ? Lds::V_BLOCK : Lds::K_BLOCK;
        const int rs = V ? v_row : k_row;
        uint8_t *d = dst + w * NLD * BLOCK;
        if (rows >= RW) {
#pragma unroll
            for (int i = 0; i < NLD; i++) copy_lds(src + i * RPI * rs, V ? v_off : k_off, d + i * BLOCK);
        } else {
#pragma unroll
            for (int i = 0; i < NLD; i++) copy_lds(src, imin(i * RPI + (V ? v_r : k_r), rows - 1) * rs + (V ? v_c : k_c), d + i * BLOCK);
        }
    };
    using K_ = std::false_type;
    using V_ = std::true_type;

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = -FLT_MAX, l = 0, ym = 0;  // ym: largest score of the group whose turn is next
    // exponent of a score in log2 units is s · c
    const float c = CAP ? 1.0f : a.scale * LOG2E_F;
    const SoftCap cap = CAP ? soft_cap(a) : SoftCap{};
    // the lane's places in a tile: keys row-wise, values transposed
    const int k_at = Lds::key(lane & 31, h), v_at = Lds::value(4 * h + ((lane & 15) >> 2), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) + (lane & 1) * 8;

    f32x16 s[2];
    u32x4 pf[2][2];
    auto scores = [&](uint32_t kt, int kb, f32x16 &d) __attribute__((always_inline)) {
        d = f32x16{};
#pragma unroll
        for (int i = 0; i < KS; i++) d = mfma32<BF>(lds_16(kt + k_at + Lds::key(kb * 32, 2 * i)), qf[i], d);
    };
    auto max16 = [&](const f32x16 &x) __attribute__((always_inline)) {
        float v = fmaxf(fmaxf(x[0], x[1]), x[2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) v = fmaxf(fmaxf(v, x[e]), x[e + 1]);
        return fmaxf(v, x[15]);
    };
    auto outputs = [&](uint32_t vt, int kb, const u32x4 (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const uint32_t vp = vt + v_at + Lds::value(kb * 32 + st * 16, 4 * d);
                const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(8, 0));
                o[d] = mfma32<BF>(u32x4{v0[0], v0[1], v1[0], v1[1]}, p[st], o[d]);
            }
    };
    // group (t, kb): probabilities of its scores x → p; outputs of the group before from values
    // (vt, vkb) and probabilities po; scores of the group behind from keys (kt, nkb) → y
    auto group = [&](int key0, int bad2, f32x16 &x, u32x4 (&p)[2], const u32x4 (&po)[2], f32x16 &y, uint32_t vt, int vkb, uint32_t kt, int nkb) __attribute__((always_inline)) {
        // positions of the lane's scores: key0 + 4 h + (8 (e / 4) + e % 4)
        float mx = ym;
        const bool late = key0 + 31 > all_hi, early = key0 <= all_lo;
        if (CAP || late || early || bad2) {
            if constexpr (CAP) {
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = cap_score<CAP>(x[e], cap);
            }
            if (late) {
                const int d = p_q - key0 - 4 * h;
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = 8 * (e / 4) + e % 4 <= d ? x[e] : -INFINITY;
            }
            if (early) {
                const int d = lo_q - key0 - 4 * h;
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = 8 * (e / 4) + e % 4 > d ? x[e] : -INFINITY;
            }
            if (bad2) {
#pragma unroll
                for (int e = 0; e < 16; e++) x[e] = bad2 >> (e / 8) & 1 ? -INFINITY : x[e];
            }
            mx = max16(x);
        }
        mx *= c;
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
        // Eight rounds of matrix products, first the scores', then the outputs', operands read three
        // products ahead, with a share of the probabilities after each; the next group's maximum
        // at the end, so that its own round begins with it.  The fences keep the order.
        constexpr int NV = 2 * DB, NM = KS + NV;
        y = f32x16{};
        const float ref = P_SHIFT<BF> - m;
        u32x4 fr[NM];
        auto read = [&](int u) __attribute__((always_inline)) {
            if (u >= NM) return;
            if (u < KS) {
                fr[u] = lds_16(kt + k_at + Lds::key(nkb * 32, 2 * u));
            } else {
                const uint32_t vp = vt + v_at + Lds::value(vkb * 32 + (u - KS) / DB * 16, (u - KS) % DB * 4);
                const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(8, 0));
                fr[u] = u32x4{v0[0], v0[1], v1[0], v1[1]};
            }
        };
        float ex[16];
        auto exps = [&](int i) __attribute__((always_inline)) {
            ex[2 * i] = exp2_hw(fmaf(x[2 * i], c, ref));
            ex[2 * i + 1] = exp2_hw(fmaf(x[2 * i + 1], c, ref));
        };
        auto pack = [&](int i) __attribute__((always_inline)) { p[i / 4][i % 4] = pack2<BF>(ex[2 * i], ex[2 * i + 1]); };
        auto add = [&](int i) __attribute__((always_inline)) { l = add2<BF>(p[i / 4][i % 4], l); };
        auto product = [&](int u) __attribute__((always_inline)) {
            if (u < KS) y = mfma32<BF>(fr[u], qf[u], y);
            else o[(u - KS) % DB] = mfma32<BF>(fr[u], po[(u - KS) / DB], o[(u - KS) % DB]);
        };
        constexpr int AHEAD = 3;
#pragma unroll
        for (int u = 0; u < AHEAD; u++) read(u);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int u0 = i * NM / 8, u1 = (i + 1) * NM / 8;
            if (u0 < u1) {
                product(u0);
                read(u0 + AHEAD);
            }
            exps(i);
            if (u0 < u1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = u0 + 1; u < u1; u++) {
                product(u);
                read(u + AHEAD);
                if (u < u1 - 1) __builtin_amdgcn_sched_barrier(0);
            }
            pack(i);
            if (i) add(i - 1);
            if (u0 + 1 < u1) __builtin_amdgcn_sched_barrier(0);
            if (i == 6) {
                ym = fmaxf(fmaxf(y[0], y[1]), y[2]);
#pragma unroll
                for (int e = 3; e < 9; e += 2) ym = fmaxf(fmaxf(ym, y[e]), y[e + 1]);
            }
            if (i == 7) {
#pragma unroll
                for (int e = 9; e < 15; e += 2) ym = fmaxf(fmaxf(ym, y[e]), y[e + 1]);
                ym = fmaxf(ym, y[15]);
            }
        }
        add(7);
        // all three belong into this block: the compiler would move the probabilities to where
        // they are used, and make two copies of the block
        asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(l), "+v"(ym));
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
                    if (e % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few values in registers at a time
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
        const int ids0 = request_pages(t_begin), ids1 = request_pages(t_begin + 1);
        int ids = request_pages(t_begin + 2);
        Tile cur = tile_of(t_begin, ids0), nxt = tile_of(t_begin + 1, ids1);
        int bad_before = 0;  // KB = 1: of tile t − 1
        copy(K_{}, kbase + cur.k, cur.rows, s_k0);
        if (t_begin + 1 < t_end) copy(K_{}, kbase + nxt.k, nxt.rows, s_k1);
        if constexpr (KB == 2) copy(V_{}, vbase + cur.v, cur.rows, s_v0);
        // the first group's outputs before it: zeros
        for (int i = w; i < 32 / RPI; i += 4) *(u32x4 *)(s_v1 + Lds::value((KB - 1) * 32 + i * RPI, 0) + lane * 16) = u32x4{0, 0, 0, 0};
        pf[1][0] = pf[1][1] = u32x4{0, 0, 0, 0};
        wait_vmem();
        lds_barrier();
        if (wave_live) {
            scores(lds_at(s_k0), 0, s[0]);
            ym = max16(s[0]);
        }
        auto tile = [&](int t, uint8_t *k_t, uint8_t *k_n, uint8_t *v_t, uint8_t *v_n, f32x16 &x0, f32x16 &x1, u32x4 (&p0)[2], u32x4 (&p1)[2]) __attribute__((always_inline)) {
            if constexpr (KB == 2)
                if (wave_live) group(t * KT, cur.bad & 3, x0, p0, p1, x1, lds_at(v_n), 1, lds_at(k_t), 1);
            wait_vmem();
            lds_barrier();
            Tile third{};
            if (t + 2 < t_end) {
                third = tile_of(t + 2, ids);
                copy(K_{}, kbase + third.k, third.rows, k_t);
            }
            ids = request_pages(t + 3);
            if constexpr (KB == 2) {
                if (t + 1 < t_end) copy(V_{}, vbase + nxt.v, nxt.rows, v_n);
                apart(t, cur.bad, v_t);
                if (wave_live) group(t * KT + 32, cur.bad >> 2, x1, p1, p0, x0, lds_at(v_t), 0, lds_at(k_n), 0);
            } else {
                copy(V_{}, vbase + cur.v, cur.rows, v_t);
                if (t > t_begin) apart(t - 1, bad_before, v_n);
                if (wave_live) group(t * KT, cur.bad, x0, p0, p1, x1, lds_at(v_n), 0, lds_at(k_n), 0);
                bad_before = cur.bad;
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
            apart(t_end - 1, bad_before, odd ? s_v0 : s_v1);
        }
        if (wave_live) {
            if (odd) outputs(lds_at(s_v0), KB - 1, pf[KB == 2 ? 1 : 0]);
            else outputs(lds_at(s_v1), KB - 1, pf[1]);
        }
    }

    float l0, l1;
    pair_f<32>(l, l0, l1);
    l = l0 + l1;
    const LateArgs late = late_args();  // also what the stores need
    bool nan = false;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) nan |= o[d][e] != o[d][e];
    const float inv = ns > 1 ? 1.0f : l > 0 || l != l ? 1.0f / l : 0.0f;
    uint8_t *op = late->out + (int64_t)(sv.row0 + tok) * late->o_row + head * late->o_head + h * 8;
    const int64_t at = ((int64_t)(sv.row0 + tok) * late->n_head + head) * late->S + sp;
    float *pp = late->part + at * HD + 4 * h;
    if (!live) {
        // nothing to store; the search below is the whole wave's
    } else if (ns == 1) {
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const u32x2 v = {pack2<BF>(o[d][4 * e] * inv, o[d][4 * e + 1] * inv), pack2<BF>(o[d][4 * e + 2] * inv, o[d][4 * e + 3] * inv)};
                *(u32x2 *)(op + d * 64 + e * 16) = v;
            }
    } else {
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) *(f32x4 *)(pp + d * 32 + e * 8) = f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
        if (h == 0) *(f32x2 *)(late->ml + at * 2) = f32x2{m, l};
    }
    const bool again = live && nan && l == l;
    if (!__any(again)) return;
    NonFinite<HD, BF> nf;
    nf.search(late, si, sv.row0, kvh, imax(before_window(pos0 + w_t0, late->window) + 1, 0), imin(pos0 + w_t1, sv.len - 1) + 1, all_lo + 1, all_hi + 1,
              t_begin * KT, t_end * KT);
    for (int k = 0; k < HD / 8; k++) {  // the lane's dims: 8 k + 4 h …
        const f32x4 x = nf.of(late, si, sv.row0, kvh, k, h, lo_q, p_q);
        if (!again) continue;
        for (int e = 0; e < 4; e++) {
            if (ns == 1) {
                uint16_t *y = (uint16_t *)(op + k * 16) + e;
                if (value16<BF>(*y) != value16<BF>(*y)) *y = (uint16_t)pack2<BF>(x[e], x[e]);
            } else if (pp[k * 8 + e] != pp[k * 8 + e]) {
                pp[k * 8 + e] = x[e];
            }
        }
    }
}

// At most 16·NB query rows of a sequence and KV head: each of the workgroup's 4 waves takes
// every fourth tile of 32 positions, and the waves' results are added up at the end.  Keys go
// from global memory straight to operand registers, values to the wave's own part of LDS, so no
// barrier lies between the reading and the arithmetic; each is requested as soon as its place
// is free, and the other waves of the CU (16 at head size 128) keep the memory busy meanwhile.
// The matrix units being idle, a probability is two values of the tensors' type (value and
// remainder), and the outputs are as exact as their own rounding.
//
// Bound: HBM.  One token over 100003 positions (4 KV heads of 128, bf16, 205 MB): 40 us, 5.1
// TB/s, what a copy reaches, and 5.7 for the join of 112 splits; of 48 sequences (8 KV heads,
// f16, up to 4000 positions, 298 MB): 67 us, 4.4 TB/s, and 6.8, the sequences' different lengths
// being the difference.  Values through registers, 8 waves on a CU: 74 us.
constexpr int FEW_KT = 32, FEW_STEP = 4 * FEW_KT;
template <int HD, int NB>
constexpr int FEW_WAVES = NB == 1 ? (HD <= 128 ? 4 : 2) : (HD <= 64 ? 3 : HD <= 128 ? 2 : 1);  // of a SIMD, as registers allow

// the 16-bit value nearest to a, as f32
template <bool BF>
__device__ __forceinline__ float low16(uint32_t w) { return BF ? __uint_as_float(w << 16) : h2f(w & 0xFFFF); }
template <bool BF>
__device__ __forceinline__ float high16(uint32_t w) { return BF ? __uint_as_float(w & 0xFFFF0000u) : h2f(w >> 16); }

template <int HD, bool BF, bool CAP, int NB>
__global__ __launch_bounds__(256, (FEW_WAVES<HD, NB>)) void attn_few_kernel(ServeAttnArgs a) {
    using Lds = TileLds<HD>;
    constexpr int KT = FEW_KT, RPI = Lds::RPI, NLD = KT / RPI, KS = HD / 32, DB = HD / 16;
    constexpr int VB = NLD * Lds::V_BLOCK, OB = 16 * NB * HD * 4;  // a wave's values, and its outputs at the end
    constexpr int WB = VB > OB ? VB : OB;
    __shared__ __align__(16) uint8_t s_buf[4][WB];
    __shared__ float s_ml[4][16 * NB][2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
    const int G = a.G, kvh = blockIdx.x % a.n_kv, si = blockIdx.x / a.n_kv;
    const SeqView sv = view_of(a.b, a.kv, si);
    const int n_rows = imin(sv.n_new * G, 16 * NB);
    if (n_rows == 0) return;
    const int n_tok = same((n_rows + G - 1) / G), pos0 = sv.pos0();
    const KeyRange kr = key_range(sv, 0, n_tok - 1, a.window);
    const int hi = same(kr.hi), t0 = same(first_tile(kr, FEW_STEP)), nt = same(tile_count(kr, FEW_STEP)), ns = same(split_count(nt, a.C, a.S)), sp = blockIdx.y;
    if (sp >= ns) return;
    const int begin = (t0 + sp * a.C) * 4 + w, end = imin((sp == ns - 1 ? t0 + nt : t0 + (sp + 1) * a.C) * 4, (hi + KT - 1) / KT);

    int p_q[NB], lo_q[NB];
    u32x4 qf[NB][KS];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int row = b * 16 + col, tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
        const bool live = row < n_rows;
        p_q[b] = live ? imin(pos0 + tok, sv.len - 1) : -1;
        lo_q[b] = before_window(pos0 + tok, a.window);
        const uint8_t *qp = a.q + (int64_t)(sv.row0 + tok) * a.q_row + head * a.q_head + g * 16;
#pragma unroll
        for (int i = 0; i < KS; i++) qf[b][i] = live ? *(const u32x4 *)(qp + i * 64) : u32x4{0, 0, 0, 0};
    }
    const int all_hi = imin(pos0, sv.len - 1), all_lo = before_window(pos0 + n_tok - 1, a.window);

    const int *trow = a.kv.table + (int64_t)si * a.kv.table_stride;
    const uint8_t *kbase = a.kv.k + kvh * a.kv.k_head, *vbase = a.kv.v + kvh * a.kv.v_head;
    uint8_t *vt = s_buf[w];
    const int k_row = (int)a.kv.k_row, v_row = (int)a.kv.v_row;
    const int v_r = Lds::value_row(lane), v_c = imin(Lds::value_chunk(lane), HD / 8 - 1) * 16;
    // Page ids of a tile's two groups of 16 positions (lanes 0 and 1), requested a tile ahead.
    // Positions behind the last one seen are read as copies of it.
    auto first_of = [&](int t, int b) { return imin(t * KT + b * 16, (hi - 1) & ~15); };
    // The lane's number is taken anew each time: what it adds, kept, was a register too many at
    // 128-wide heads with a softcap, whose reload waits for the copies (64 tokens over 2000
    // positions, 8 KV heads: 122.4 us, now 117.5).
    auto request_pages = [&](int t) {
        int id = threadIdx.x;
        asm volatile("" : "+v"(id));
        return t < end ? trow[first_of(t, id & 1) >> a.kv.page_shift] : 0;
    };
    struct Pages {
        int id[2], bad;  // bad bit b: the page of group b is none (any that exists is read, and nobody sees it)
    };
    auto pages_of = [&](int ids) {
        const bool ok = (unsigned)ids < (unsigned)a.kv.n_pages;
        const int id = ok ? ids : 0;
        Pages x;
        x.bad = (int)(__ballot(!ok) & 3);
        x.id[0] = __builtin_amdgcn_readlane(id, 0);
        x.id[1] = __builtin_amdgcn_readlane(id, 1);
        return x;
    };
    u32x4 rk[2][KS];
    auto load_keys = [&](int t, const Pages &pg) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int g0 = first_of(t, b), slot = g0 & ((1 << a.kv.page_shift) - 1);
            const uint8_t *kp = kbase + pg.id[b] * a.kv.page + slot * a.kv.k_row;
            const int off = imin(col, hi - 1 - g0) * k_row + g * 16;
#pragma unroll
            for (int i = 0; i < KS; i++) rk[b][i] = *(const u32x4 *)(kp + off + i * 64);
        }
    };
    auto copy_values = [&](int t, const Pages &pg) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const int g0 = first_of(t, b), slot = g0 & ((1 << a.kv.page_shift) - 1), last = hi - 1 - g0;
            const uint8_t *vp = vbase + pg.id[b] * a.kv.page + slot * a.kv.v_row;
#pragma unroll
            for (int i = 0; i < NLD / 2; i++) copy_lds(vp, imin(i * RPI + v_r, last) * v_row + v_c, vt + (b * (NLD / 2) + i) * Lds::V_BLOCK);
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
    const float c = CAP ? 1.0f : a.scale * LOG2E_F;
    const SoftCap cap = CAP ? soft_cap(a) : SoftCap{};
    const int v_at = Lds::value(4 * g + (col >> 2), (lane & 3) >> 1) + (lane & 1) * 8;

    Pages pg{};
    int ids = 0;
    if (begin < end) {
        pg = pages_of(request_pages(begin));
        load_keys(begin, pg);
        copy_values(begin, pg);
        ids = request_pages(begin + 4);
    }
    for (int t = begin; t < end; t += 4) {
        const int key0 = t * KT, bad = pg.bad;
        const bool part = key0 + KT - 1 > all_hi || key0 <= all_lo || bad;  // some row does not see all of the tile
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        f32x4 s[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                s[b][kb] = f32x4{};
#pragma unroll
                for (int i = 0; i < KS; i++) s[b][kb] = mfma16<BF>(rk[kb][i], qf[b][i], s[b][kb]);
            }
        if (t + 4 < end) {
            pg = pages_of(ids);
            load_keys(t + 4, pg);
            ids = request_pages(t + 8);
        }
        if (part) {
            bool nf = false;
#pragma unroll
            for (int i = 0; i < NLD; i++) nf = nf || nonfinite8<BF>(*(const u32x4 *)(vt + i * Lds::V_BLOCK + lane * 16));
            if (__any(nf)) {  // rare: added one by one for the rows that see them, then zeros
                for (int r = 0; r < KT; r++) {
                    const int j = key0 + r;
                    const uint8_t *vp = vt + Lds::value(r, 0) + 8 * (g & 1);
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const bool see = j <= p_q[b] && j > lo_q[b] && !(bad >> (r / 16) & 1);
                        if (!__any(see)) continue;
#pragma unroll
                        for (int d = 0; d < DB; d++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {  // dim 16 d + 4 g + e
                                const float x = value16<BF>(*(const uint16_t *)(vp + Lds::value(0, 2 * d) + (g >> 1) * 16 + e * 2));
                                o[b][d][e] += (see & !(fabsf(x) <= FLT_MAX)) ? x : 0.0f;
                            }
                    }
                }
                wave_sync();
#pragma unroll
                for (int i = 0; i < NLD; i++) {
                    u32x4 *p = (u32x4 *)(vt + i * Lds::V_BLOCK + lane * 16);
                    u32x4 x = *p;
                    for (int e = 0; e < 4; e++) x[e] = finite2<BF>(x[e]);
                    *p = x;
                }
                wave_sync();
            }
        }
        u32x4 pf[NB][2];  // probabilities, and what their rounding left
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if constexpr (CAP) s[b][kb][e] = cap_score<CAP>(s[b][kb][e], cap);
                    if (part) {
                        const int j = key0 + kb * 16 + 4 * g + e;
                        s[b][kb][e] = (j > p_q[b]) | (j <= lo_q[b]) | (bad >> kb & 1) ? -INFINITY : s[b][kb][e];
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
                const float p0 = exp2_hw(fmaf(s[b][e / 2][2 * (e & 1)], c, ref)), p1 = exp2_hw(fmaf(s[b][e / 2][2 * (e & 1) + 1], c, ref));
                const uint32_t near = pack2<BF>(p0, p1);
                pf[b][0][e] = near;
                pf[b][1][e] = pack2<BF>(p0 - low16<BF>(near), p1 - high16<BF>(near));
                l[b] += p0 + p1;
            }
        }
#pragma unroll
        for (int d = 0; d < DB; d++) {
            const uint32_t vp = lds_at(vt) + v_at + Lds::value(0, 2 * d);
            const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(16, 0));
            const u32x4 vf = {v0[0], v0[1], v1[0], v1[1]};
#pragma unroll
            for (int b = 0; b < NB; b++) {
                o[b][d] = mfma16<BF>(vf, pf[b][1], o[b][d]);
                o[b][d] = mfma16<BF>(vf, pf[b][0], o[b][d]);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the values have been read: their place is free
        if (t + 4 < end) copy_values(t + 4, pg);
    }

    // the four waves' results
    wave_sync();
#pragma unroll
    for (int b = 0; b < NB; b++) {
        float x0, x1, y0, y1;
        pair_f<16>(l[b], x0, x1);
        pair_f<32>(x0 + x1, y0, y1);
        float *po = (float *)vt + (b * 16 + col) * HD + 4 * g;
#pragma unroll
        for (int d = 0; d < DB; d++) *(f32x4 *)(po + d * 16) = o[b][d];
        if (g == 0) {
            s_ml[w][b * 16 + col][0] = m[b];
            s_ml[w][b * 16 + col][1] = y0 + y1;
        }
    }
    __syncthreads();
    const LateArgs late = late_args();
    NonFinite<HD, BF> nf;
    bool searched = false;
    for (int i0 = w * 64; i0 < n_rows * (HD / 4); i0 += 256) {
        const bool live = i0 + lane < n_rows * (HD / 4);
        const int i = live ? i0 + lane : i0, r = i / (HD / 4), d4 = i % (HD / 4), tok = r / G, head = kvh * G + r - tok * G;
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
        if (__any(L == L && (acc[0] != acc[0] || acc[1] != acc[1] || acc[2] != acc[2] || acc[3] != acc[3]))) {  // rare
            if (!searched)
                nf.search(late, si, 0, kvh, imax(before_window(pos0, late->window) + 1, 0), imin(pos0 + n_tok - 1, sv.len - 1) + 1, all_lo + 1, all_hi + 1,
                          (t0 + sp * late->C) * FEW_STEP, (sp == ns - 1 ? t0 + nt : t0 + (sp + 1) * late->C) * FEW_STEP);
            searched = true;
            const f32x4 x = nf.of(late, si, 0, kvh, d4 / 2, d4 & 1, before_window(pos0 + tok, late->window), imin(pos0 + tok, sv.len - 1));
            for (int e = 0; e < 4; e++)
                if (L == L && acc[e] != acc[e]) acc[e] = x[e];
        }
        if (!live) break;
        if (ns == 1) {
            const float inv = L > 0 || L != L ? 1.0f / L : 0.0f;
            uint8_t *op = late->out + (int64_t)(sv.row0 + tok) * late->o_row + head * late->o_head + d4 * 8;
            *(u32x2 *)op = u32x2{pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
        } else {
            const int64_t at = ((int64_t)(sv.row0 + tok) * late->n_head + head) * late->S + sp;
            *(f32x4 *)(late->part + at * HD + d4 * 4) = acc;
            if (d4 == 0) *(f32x2 *)(late->ml + at * 2) = f32x2{mm, L};
        }
    }
}

// The splits of each (row, head), added up by W waves: HD / 4 lanes hold a split's values, and
// the groups of so many lanes take the splits in turn.  W = 4 where there are few rows, whose
// time is that of the loads behind one another, W = 1 (4 rows to a workgroup) where there are
// many: one token over 100003 positions (32 heads, 61 splits) 19.9 us with a wave that read its
// splits one by one.  M rows per block and KT positions per tile are those of the kernel that
// made the partials.
template <bool BF, int W>
__global__ __launch_bounds__(256) void serve_combine_kernel(ServeAttnArgs a, int M, int KT) {
    __shared__ float s_f[4][SERVE_MAX_SPLIT];
    __shared__ f32x4 s_o[W == 1 ? 1 : 256];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), id = W == 1 ? blockIdx.x * 4 + w : blockIdx.x;
    const int row = id / a.n_head, head = id - row * a.n_head, G = a.G;
    if (row >= a.b.n_rows) return;
    int si;
    const SeqView sv = find_seq(a.b, a.kv, row, si, [&](int s, int) { return iclamp(s, 0, a.b.n_rows); });
    if (row < sv.row0 || row >= sv.row0 + sv.n_new) return;
    const int r = (row - sv.row0) * G + head % G, n_rows = sv.n_new * G, r0 = r / M * M, r1 = imin(r0 + M, n_rows) - 1;
    const int ns = split_count(tile_count(key_range(sv, r0 / G, r1 / G, a.window), KT), a.C, a.S);
    if (ns == 1) return;
    const int64_t at = ((int64_t)row * a.n_head + head) * a.S;
    const int lpr = a.hd / 4, per = 64 / lpr, g = lane / lpr, d = lane - g * lpr;  // lanes of a split, splits of a wave
    // the first splits' values are requested before the maxima that weigh them are known
    constexpr int FIRST = W == 1 ? 2 : 8;
    const float *p = a.part + at * a.hd + d * 4;
    const int s0 = g < per ? w % W * per + g : ns;
    f32x4 x[FIRST];
#pragma unroll
    for (int k = 0; k < FIRST; k++) x[k] = s0 + k * W * per < ns ? *(const f32x4 *)(p + (int64_t)(s0 + k * W * per) * a.hd) : f32x4{};
    float m0 = -FLT_MAX, l0 = 0, m1 = -FLT_MAX, l1 = 0;
    if (lane < ns) {
        m0 = a.ml[(at + lane) * 2];
        l0 = a.ml[(at + lane) * 2 + 1];
    }
    if (lane + 64 < ns) {
        m1 = a.ml[(at + lane + 64) * 2];
        l1 = a.ml[(at + lane + 64) * 2 + 1];
    }
    const float mm = xmax_f<64>(fmaxf(m0, m1)), f0 = exp2_hw(m0 - mm), f1 = exp2_hw(m1 - mm);
    const float L = xsum_f<64>(f0 * l0 + f1 * l1);
    const float inv = L > 0 || L != L ? 1.0f / L : 0.0f;
    s_f[w][lane] = f0 * inv;
    s_f[w][lane + 64] = f1 * inv;
    wave_sync();
    f32x4 acc = f32x4{};
#pragma unroll
    for (int k = 0; k < FIRST; k++)
        if (s0 + k * W * per < ns) {
            const float f = s_f[w][s0 + k * W * per];
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = fmaf(f, x[k][e], acc[e]);
        }
#pragma unroll 4
    for (int s = s0 + FIRST * W * per; s < ns; s += W * per) {
        const f32x4 y = *(const f32x4 *)(p + (int64_t)s * a.hd);
        const float f = s_f[w][s];
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = fmaf(f, y[e], acc[e]);
    }
    if constexpr (W > 1) {
        s_o[threadIdx.x] = acc;
        __syncthreads();
        if (w) return;
        acc = f32x4{};
        if (g == 0)
            for (int i = 0; i < W; i++)
                for (int k = 0; k < per; k++) acc += s_o[i * 64 + k * lpr + d];
    } else {
        f32x4 sum = acc;
        for (int k = 1; k < per; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] += __shfl(acc[e], lane + k * lpr);
        acc = sum;
    }
    if (g == 0) {
        if (L == L)  // rare: a split's infinity has met a weight of zero
            for (int e = 0; e < 4; e++)
                if (acc[e] != acc[e]) {
                    float sum = 0;
                    for (int s = 0; s < ns; s++) {
                        const float y = p[(int64_t)s * a.hd + e];
                        if (!(fabsf(y) <= FLT_MAX)) sum += y;
                    }
                    acc[e] = sum;
                }
        uint8_t *op = a.out + (int64_t)row * a.o_row + head * a.o_head;
        *(u32x2 *)(op + d * 8) = u32x2{pack2<BF>(acc[0], acc[1]), pack2<BF>(acc[2], acc[3])};
    }
}

// New rows into their pages: a wave per token row, 8 values of K or V per lane and step.
// Bound: HBM, 2854 rows of 2 x 8 heads of 128, f32 to bf16 (35 MB) 7.1 us, 4.9 TB/s; a step of
// 61 rows 3 us, which is a launch.
template <int SRC, bool BF>  // SRC: bytes of a source value
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= a.b.n_rows) return;
    int si;
    const SeqView sv = find_seq(a.b, a.kv, row, si, [&](int s, int) { return iclamp(s, 0, a.b.n_rows); });
    if (row < sv.row0 || row >= sv.row0 + sv.n_new) return;
    const int pos = sv.pos0() + row - sv.row0;
    int page;
    if (pos < 0 || pos >= sv.len || !page_of(a.kv, a.kv.table + (int64_t)si * a.kv.table_stride, pos, page)) return;
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
        if (few_row_blocks(true, a.b.max_new, a.G) == 1) {
            if (cap) attn_few_kernel<HD, BF, true, 1><<<grid, 256, 0, st>>>(a);
            else attn_few_kernel<HD, BF, false, 1><<<grid, 256, 0, st>>>(a);
        } else {
            if (cap) attn_few_kernel<HD, BF, true, 2><<<grid, 256, 0, st>>>(a);
            else attn_few_kernel<HD, BF, false, 2><<<grid, 256, 0, st>>>(a);
        }
    } else {
        const int grid = a.n_blocks * a.n_kv * a.S;
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

// (row, head) pairs up to which the splits are added up by four waves each
constexpr int COMBINE_FEW = 2048;

}  // namespace

bool serve_attn_head_dim_ok(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

bool serve_attn_few(const ServeAttnArgs &a) { return few_row_blocks(a.kv.table, a.b.max_new, a.G) > 0; }

SplitPlan serve_attn_splits(const ServeAttnArgs &a) {
    const bool few = serve_attn_few(a);
    const int KT = few ? FEW_STEP : tile_kt(a.hd);
    const int64_t blocks = few ? a.b.n_seq : block_count(a.b.n_rows, a.b.n_seq, a.G, TILE_M);
    // positions that a block's rows see, at most
    int64_t span = a.b.max_len;
    if (a.window > 0) span = std::min<int64_t>(span, (int64_t)a.window + std::min<int64_t>(a.b.max_new, few ? FEW_ROWS : TILE_M / a.G + 1) + KT);
    const int tiles = (int)((span + KT - 1) / KT);
    // Few rows: 4096 workgroups where there is so much, since sequences differ in length, and at
    // least 256 positions each (48 tokens over up to 4000 positions, 8 KV heads: 85.9 us at 1024
    // workgroups, 75.0 at 2048, 73.2 at 4096, 74.3 at 8192); a cache of under 512 positions is
    // not split, a second launch being longer than its loads.
    if (few) return split_plan(blocks * a.n_kv, tiles, 4096, 2, SERVE_MAX_SPLIT);
    // Tiles: 2 us each with every slot taken (64 positions of 128 values, plain bf16: f16 takes 0 to 5 % more
    // and a softcap 1.4 to 1.6 times it, which would split a little more), partials at 4.5 TB/s.
    // Chunks in a batch of 13 (488 workgroups): 208 us in one, 202 to 248 in 2 to 5 splits;
    // window prompts with 256-wide heads (123) 31.5 in one, 47.7 in 4; one long prompt is split.
    const double part_us = (double)a.b.n_rows * a.n_head * a.hd * 8 / 4.5e6;
    return tile_plan(blocks * a.n_kv, a.hd <= 128 ? 512 : 256, tiles, 2.0 * KT * a.hd / (64 * 128), part_us, SERVE_MAX_SPLIT);
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
        const int M = few ? FEW_ROWS : TILE_M, KT = few ? FEW_STEP : tile_kt(a.hd);
        const int64_t n = (int64_t)a.b.n_rows * a.n_head;
        if (n <= COMBINE_FEW) {
            if (bf) serve_combine_kernel<true, 4><<<n, 256, 0, st>>>(a, M, KT);
            else serve_combine_kernel<false, 4><<<n, 256, 0, st>>>(a, M, KT);
        } else {
            if (bf) serve_combine_kernel<true, 1><<<(n + 3) / 4, 256, 0, st>>>(a, M, KT);
            else serve_combine_kernel<false, 1><<<(n + 3) / 4, 256, 0, st>>>(a, M, KT);
        }
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
