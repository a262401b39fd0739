// serve_attn8.hip — the paged cache in 8 bits, and attention over it.  A value is a code of
// −127..127 times a scale, which the values of one head at a block of 16, 32, … positions of a
// page share:
//
//   append:     s' = max(s, max |x| / 127) over the block's new values x (s: 0 where the block
//               holds no earlier position),  c = round(x / s'),  earlier codes c' = round(c · s / s')
//   attention:  o_t = Σ_j softmax_j(s_tj) v_j  with  s_tj = scale · q_t·k_j  as over 16-bit pages
//
// Rounding.  Codes are small whole numbers, exact in any of the matrix units' types, and a scale
// is the same for all values of a product's row, so it is applied to f32 sums: scores are
// (q · codes) · s_k, and a value's scale goes into the exponent of its probability,
// p · s_v = 2^(score + log2 s_v − m).  m is the maximum of these exponents, so that what is
// multiplied with the codes stays in f16's range whatever the scales are; the sum of the
// probabilities alone is formed in f32 as Σ (p · s_v) / s_v.  In the few-rows kernel queries are
// three 8-bit parts of a whole number (23 bits, relative to a row's largest value), and p · s_v
// two f16 parts; in the tile kernel queries are f16 as they are (bf16 ones with a row's power of
// two taken out, exact but for values 2^28 times smaller than the row's largest), p · s_v one f16,
// rounded to nearest.
//
// Infinite and NaN values cannot be codes: a block that was given one has a NaN scale, and the
// tokens that see any of its positions get NaN.  Those that see none of it are unaffected: codes
// are finite, and exponents are masked after the scales are in.
#include "../common.hpp"
#include "../serve_device.hpp"

#include <algorithm>
#include <cfloat>
#include <type_traits>

namespace rie {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A scale as the kernels use it: NaN where it is negative or too large, as append takes it.  That of a
// block of zeros, whose codes are zeros, is any number.
__device__ __forceinline__ float usable(float s) { return s >= 0 && s <= SCALE8_MAX ? fmaxf(s, SCALE8_MIN) : NAN; }

// 4 codes in f16.  1024 + (code + 128) is f16's 0x6400 with the code, its sign bit turned over, as
// the low byte; the difference is exact.
__device__ __forceinline__ void halves4(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = codes ^ 0x80808080u;
    const half2_t bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
}

// 8 bytes of one column: lanes 2r and 2r + 1 of a group of 16 name the 16 bytes of row r, and
// lane l gets rows 0..7 of column l
__device__ __forceinline__ u32x2 read_tr8(uint32_t at) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(uintptr_t)at));
}

constexpr float P_SHIFT8 = 6.0f;  // p · s_v is 2^(exponent − m + P_SHIFT8): at most 2^14, and small ones are normal f16 numbers

// ---- a sequence with at most 16·NB query rows: a tile of 32 positions per wave ----
//
// As over 16-bit pages (attn_few_kernel): each of the workgroup's 4 waves takes every fourth tile,
// keys go from global memory to operand registers, values to the wave's own part of LDS, and the
// waves' results are added up at the end.  Keys meet the query's 8-bit parts on integer matrix
// instructions as they are; values are read transposed, 8 positions of a dim to a lane, and made
// f16 there, 10 vector instructions for 8 values.
//
// Bound: HBM while all workgroups stream, and their beginning: starts, page ids, scales and the
// first tile lie behind one another.  48 tokens over up to 4000 positions, 32/8 heads of 128
// (149 MB) 34 us (4.4 TB/s, where a copy reaches 5.2) and 6 for the join, 1 over 100003 positions,
// 32/4 of 128 (103 MB) 21.5 (4.8 TB/s) and 5.  With two blocks of 16 rows (5 tokens of 16 sequences
// over 4000 positions, 32/8 of 128) 47 for the call, where 1 token takes 31: twice the products, at
// half as many waves.
constexpr int FEW8_KT = 32, FEW8_STEP = 4 * FEW8_KT;          // positions of a wave's tile and of a step
constexpr int FEW8_LEAST = 2, FEW8_BEGIN = 1, FEW8_SEQS = 64;  // steps that a piece is worth, those that a sequence's beginning takes; sequences that are cut in pieces
// of a SIMD: with splits as many as registers allow, with pieces two, which have all that they need
constexpr int few8_waves(int hd, int nb, bool pieces) {
    return nb == 1 ? (hd <= 128 && !pieces ? 4 : 2) : hd <= 64 && !pieces ? 3 : hd <= 128 ? 2 : 1;
}

// How the positions are divided.  Pieces (S = 0): the steps of all sequences in a row are cut into
// P equal pieces, two workgroups to a CU (per KV head), wherever the cuts fall.  A workgroup goes
// through the sequences of its piece; one that it has all of goes to the outputs, and at most two
// (its first, its last) to partial results, which few8_join_kernel adds up.  Everyone finds the
// cuts from the lengths, a lane for each sequence.  Splits: S for each sequence, of C steps, the
// last of all that are left; P = S times the sequences, split by split.
//
// Pieces are for lengths that differ, of few sequences: 48 tokens over up to 4000 positions, 32/8
// heads of 128, 43 us (splits 50.7), 32 over up to 8000, 32/4 heads, 31.3 (39).  One sequence is
// faster in splits (100003 positions 27.8, in pieces 29.7), which take nothing to find, and so are
// sequences that pieces hold several of, whose beginnings then lie behind one another (500 of up
// to 1500, 32/4 heads of 128, 168 us; whole 87).  Pieces for one workgroup to a CU: 53 for 43; for
// four, which spill registers, 52.  The limit of 64 is that of a wave's lanes.  At it, pieces, splits
// of twelve steps and of two: 64 of up to 4000, 32/8 of 128, 57.6, 68.4 and 60.5 us, 64 of up to 1500
// 33.0, 28.3 and 33.4.  Behind it, splits of twelve and of two: 65 of up to 4000 64.0 and 50.8, 100 of
// them 98.6 and 94.9, 100 of up to 1500 37.4 and 44.5, 300 of them 103.6 and 119, 200 of up to 3000,
// 15/5 of 64, 48.0 and 46.9.
struct Few8Cut {
    int P, S, C;
};
__device__ __forceinline__ SeqView few8_view(const ServeAttnArgs &a, int i) {
    return i < a.b.n_seq ? seq_view(a.b.starts[i], a.b.starts[i + 1], a.b.lens[i], a.b.n_rows, a.kv.cap) : SeqView{0, 0, 0};
}
// Rows of a sequence, at most
template <int M>
__device__ __forceinline__ int few8_rows(const ServeAttnArgs &a) { return imin(imin(a.b.max_new, M) * a.G, M); }
__device__ __forceinline__ int few8_steps(const ServeAttnArgs &a, const SeqView &v, int R) {
    if (v.n_new == 0) return 0;
    return imax(tile_count(key_range(v, 0, imin(v.n_new, (R + a.G - 1) / a.G) - 1, a.window), FEW8_STEP), 1);
}
// A lane's sequence among those of pieces: its steps and its beginning
__device__ __forceinline__ int few8_units(const ServeAttnArgs &a, const SeqView &v, int R) {
    const int n = few8_steps(a, v, R);
    return n ? n + FEW8_BEGIN : 0;
}
// Units of a piece.  A sequence has at most 2^23 and a few, and pieces hold FEW8_SEQS sequences at most: sums fit 31 bits
__device__ __forceinline__ int few8_per(int total, int P) { return imax((total + P - 1) / P, FEW8_LEAST); }
// begins: of a piece, whether it has the sequence's first step
template <int HD>
__device__ __forceinline__ int64_t few8_part(const Few8Cut &cut, int kvh, int piece, bool begins, int R) {
    return (((int64_t)kvh * cut.P + piece) * (cut.S ? 1 : 2) + (cut.S ? 0 : begins)) * part_floats(R, HD);
}

// A wave's values in LDS: it copies 1 KB at a time, RPI whole rows, by 16-byte chunk, then row
template <int HD>
struct Value8Lds {
    static constexpr int HDP = HD <= 32 ? 32 : HD <= 64 ? 64 : HD <= 128 ? 128 : 256;
    static constexpr int CPR = HDP / 16, RPI = 64 / CPR;
    // a read takes 128 bytes of rows 0..7, say, and of rows 16..23: those lie in other banks
    static constexpr int BLOCK = 1024 + (RPI == 8 ? 64 : RPI == 16 ? 128 : 0);
    static __device__ __forceinline__ int at(int r, int chunk) { return r / RPI * BLOCK + chunk * (RPI * 16) + r % RPI * 16; }
    static __device__ __forceinline__ int row(int lane) { return lane % RPI; }
    static __device__ __forceinline__ int chunk(int lane) { return lane / RPI; }
};

template <int HD, bool BF, bool CAP, int NB, bool PIECES>
__global__ __launch_bounds__(256, few8_waves(HD, NB, PIECES)) void attn8_few_kernel(ServeAttn8Args x, Few8Cut cut, float *parts) {
    using Lds = Value8Lds<HD>;
    const ServeAttnArgs &a = x.a;
    constexpr int KT = FEW8_KT, RPI = Lds::RPI, NLD = KT / RPI, DB = HD / 16;
    // a sum (of 96 dims) formed by products of 64 and of 32 dims in turn had other bits from call to call
    constexpr int K64 = HD % 64 ? 0 : HD / 64, K32 = HD % 64 ? HD / 32 : 0, KS = K64 + K32;  // products of 64 or of 32 dims
    constexpr int VB = NLD * Lds::BLOCK, OB = 16 * NB * HD * 4;  // a wave's values, and its outputs at the end
    constexpr int WB = VB > OB ? VB : OB;
    __shared__ __align__(16) uint8_t s_buf[4][WB];
    __shared__ float s_ml[4][16 * NB][2];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), G = a.G, R = few8_rows<16 * NB>(a), kvh = blockIdx.x % a.n_kv, piece = blockIdx.x / a.n_kv;

    // what a piece of `per` steps has of the n of sequence si, the first of which is the piece's number base
    auto sequence = [&](int si, const SeqView &sv, int per, int base, int n) __attribute__((always_inline)) {
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));  // nothing of it is kept in registers from one sequence to the next
        const int g = lane >> 4, col = lane & 15;
        const int n_rows = imin(imin(sv.n_new, 16 * NB) * G, R);
        const int n_tok = same((n_rows + G - 1) / G), pos0 = sv.pos0();
        const KeyRange kr = key_range(sv, 0, n_tok - 1, a.window);
        const int hi = same(kr.hi), t0 = same(first_tile(kr, FEW8_STEP)), nt = same(tile_count(kr, FEW8_STEP));
        const int s0 = imax(-base, 0), s1 = imin(per - base, nt);
        const bool whole = base >= 0 && per - base >= n;
        const int begin = (t0 + s0) * 4 + w, end = imin((t0 + s1) * 4, (hi + KT - 1) / KT);

        int p_q[NB], lo_q[NB];
        const int all_hi = imin(pos0, sv.len - 1), all_lo = before_window(pos0 + n_tok - 1, a.window);

        const int *trow = a.kv.table + (int64_t)si * a.kv.table_stride;
        const uint8_t *kbase = a.kv.k + kvh * a.kv.k_head, *vbase = a.kv.v + kvh * a.kv.v_head;
        uint8_t *vt = s_buf[w];
        const int k_row = (int)a.kv.k_row, v_row = (int)a.kv.v_row, page_mask = (1 << a.kv.page_shift) - 1;
        const int v_r = Lds::row(lane), v_c = imin(Lds::chunk(lane), HD / 16 - 1) * 16;
        // Page ids of a tile's two groups of 16 positions (even and odd lanes), requested a tile ahead.
        // Positions behind the last one seen are read as copies of it.
        auto first_of = [&](int t, int b) { return imin(t * KT + b * 16, (hi - 1) & ~15); };
        auto request_pages = [&](int t) { return t < end ? trow[first_of(t, lane & 1) >> a.kv.page_shift] : 0; };
        struct Pages {
            int id, id0, id1, bad;  // the lane's; bad bit b: the page of group b is none (any that exists is read, and nobody sees it)
        };
        auto pages_of = [&](int ids) {
            const bool ok = (unsigned)ids < (unsigned)a.kv.n_pages;
            Pages p;
            p.id = ok ? ids : 0;
            p.bad = (int)(__ballot(!ok) & 3);
            p.id0 = __builtin_amdgcn_readlane(p.id, 0);
            p.id1 = __builtin_amdgcn_readlane(p.id, 1);
            return p;
        };
        // lanes 0 and 1: the scales of the groups' keys; 2 and 3: of their values
        const float *sbase = ((lane & 2) ? x.s.v : x.s.k) + (int64_t)kvh * x.s.head;
        auto request_scales = [&](int t, const Pages &pg) {
            const int slot = first_of(t, lane & 1) & page_mask;
            return sbase[(uint64_t)(uint32_t)pg.id * x.s.page + (uint64_t)(uint32_t)(slot >> x.s.block_shift) * x.s.block];
        };
        u32x4 rk[2][KS];
        auto load_keys = [&](int t, const Pages &pg) __attribute__((always_inline)) {
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const int g0 = first_of(t, b), slot = g0 & page_mask;
                const uint8_t *kp = kbase + (b ? pg.id1 : pg.id0) * a.kv.page + slot * a.kv.k_row;
                const int off = imin(col, hi - 1 - g0) * k_row;
#pragma unroll
                for (int i = 0; i < K64; i++) rk[b][i] = *(const u32x4 *)(kp + off + i * 64 + g * 16);
#pragma unroll
                for (int i = 0; i < K32; i++) {
                    const u32x2 y = *(const u32x2 *)(kp + off + i * 32 + g * 8);
                    rk[b][i] = u32x4{y[0], y[1], 0, 0};
                }
            }
        };
        auto copy_values = [&](int t, const Pages &pg) __attribute__((always_inline)) {
            if constexpr (RPI <= 16) {
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const int g0 = first_of(t, b), slot = g0 & page_mask, last = hi - 1 - g0;
                    const uint8_t *vp = vbase + (b ? pg.id1 : pg.id0) * a.kv.page + slot * a.kv.v_row;
#pragma unroll
                    for (int i = 0; i < NLD / 2; i++) copy_lds(vp, imin(i * RPI + v_r, last) * v_row + v_c, vt + (b * (NLD / 2) + i) * Lds::BLOCK);
                }
            } else {  // both groups in one copy: their distance may pass 32 bits, so by way of registers
                const int b = v_r >> 4, g0 = first_of(t, b), slot = g0 & page_mask;
                const uint8_t *vp = vbase + (b ? pg.id1 : pg.id0) * a.kv.page + slot * a.kv.v_row + imin(v_r & 15, hi - 1 - g0) * v_row + v_c;
                *(u32x4 *)(vt + lane * 16) = *(const u32x4 *)vp;
            }
        };

        // the first tile is on its way before the queries are made ready
        int ids = request_pages(begin);
        u32x4 raw[NB][KS][2];
        bool live[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int row = b * 16 + col, tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
            live[b] = row < n_rows;
            p_q[b] = live[b] ? imin(pos0 + tok, sv.len - 1) : -1;
            lo_q[b] = before_window(pos0 + tok, a.window);
            const uint8_t *qp = a.q + (int64_t)(sv.row0 + tok) * a.q_row + head * a.q_head;
#pragma unroll
            for (int i = 0; i < KS; i++)
#pragma unroll
                for (int u = 0; u < (K64 ? 2 : 1); u++) raw[b][i][u] = *(const u32x4 *)(qp + (K64 ? i * 64 + g * 16 : i * 32 + g * 8) * 2 + u * 16);
        }
        Pages pg{};
        float sc = 1;
        if (begin < end) {
            pg = pages_of(ids);
            sc = request_scales(begin, pg);
            load_keys(begin, pg);
            copy_values(begin, pg);
            ids = request_pages(begin + 4);
        }

        // Queries: a row's values are whole numbers of at most 2^22 times 2^(e − 22), in three 8-bit parts
        u32x4 qf[NB][KS][3];
        float qs[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            float most = 0;
            bool finite = true;
#pragma unroll
            for (int i = 0; i < KS; i++) {
#pragma unroll
                for (int u = 0; u < (K64 ? 2 : 1); u++) {
                    if (!live[b]) raw[b][i][u] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float f = fabsf(value16<BF>(raw[b][i][u][e / 2] >> (e & 1) * 16 & 0xFFFF));
                        finite = finite && f <= FLT_MAX;
                        most = fmaxf(most, f);
                    }
                }
            }
            float a0, a1, b0, b1;
            pair_f<16>(finite ? most : INFINITY, a0, a1);
            pair_f<32>(fmaxf(a0, a1), b0, b1);
            most = fmaxf(b0, b1);
            const int ex = 22 - __builtin_amdgcn_frexp_expf(most);  // most < 2^(22 − ex)
            qs[b] = most <= FLT_MAX ? __builtin_amdgcn_ldexpf(1.0f, -ex) : NAN;
#pragma unroll
            for (int i = 0; i < KS; i++) {
                u32x4 part[3] = {};
#pragma unroll
                for (int u = 0; u < (K64 ? 2 : 1); u++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float f = value16<BF>(raw[b][i][u][e / 2] >> (e & 1) * 16 & 0xFFFF);
                        const int n = __float2int_rn(__builtin_amdgcn_ldexpf(f, ex));
                        const int lo = (int)(int8_t)n, n1 = (n - lo) >> 8, mid = (int)(int8_t)n1, top = (n1 - mid) >> 8;
                        const int at = (u * 8 + e) / 4, sh = e % 4 * 8;
                        part[0][at] |= (uint32_t)(lo & 255) << sh;
                        part[1][at] |= (uint32_t)(mid & 255) << sh;
                        part[2][at] |= (uint32_t)(top & 255) << sh;
                    }
#pragma unroll
                for (int k = 0; k < 3; k++) qf[b][i][k] = part[k];
            }
        }
        f32x4 o[NB][DB];
        float m[NB], l[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            m[b] = -FLT_MAX;
            l[b] = 0;
#pragma unroll
            for (int d = 0; d < DB; d++) o[b][d] = f32x4{};
        }
        const SoftCap cap = CAP ? soft_cap(a) : SoftCap{};
        // where the lane reads values: positions 4 g … of both groups, 16 dims of a chunk
        const int r8 = col >> 1, v_at = Lds::at((r8 & 3) + 4 * g + (r8 >> 2) * 16, 0) + (lane & 1) * 8;

        for (int t = begin; t < end; t += 4) {
            const int key0 = t * KT, bad = pg.bad;
            const bool part = key0 + KT - 1 > all_hi || key0 <= all_lo || bad;  // some row does not see all of the tile
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const float us = usable(sc), lg = __builtin_amdgcn_logf(us), rc = us == us ? 1.0f / us : 1.0f;
            float ks[2], lv[2], iv[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                ks[b] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(us), b));
                lv[b] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(lg), 2 + b));
                iv[b] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(rc), 2 + b));
            }
            f32x4 s[NB][2];
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int kb = 0; kb < 2; kb++) {
                    i32x4 n[3] = {};
#pragma unroll
                    for (int k = 0; k < 3; k++)
#pragma unroll
                        for (int i = 0; i < KS; i++) {
                            if constexpr (K64 > 0) {
                                n[k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, rk[kb][i]), __builtin_bit_cast(i32x4, qf[b][i][k]), n[k], 0, 0, 0);
                            } else {
                                const long kk = (long)((uint64_t)rk[kb][i][1] << 32 | rk[kb][i][0]), qq = (long)((uint64_t)qf[b][i][k][1] << 32 | qf[b][i][k][0]);
                                n[k] = __builtin_amdgcn_mfma_i32_16x16x32_i8(kk, qq, n[k], 0, 0, 0);
                            }
                        }
                    // |mid · 256 + lo| is under 2^31 for 256 dims
#pragma unroll
                    for (int e = 0; e < 4; e++) s[b][kb][e] = fmaf((float)n[2][e], 65536.0f, (float)(n[1][e] * 256 + n[0][e]));
                }
            if (t + 4 < end) {
                pg = pages_of(ids);
                sc = request_scales(t + 4, pg);
                load_keys(t + 4, pg);
                ids = request_pages(t + 8);
            }
            u32x4 pf[NB][2];  // probabilities times the values' scales, and what their rounding left
#pragma unroll
            for (int b = 0; b < NB; b++) {
                float mx = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 2; kb++) {
                    const float c = ks[kb] * (CAP ? 1.0f : a.scale * LOG2E_F) * qs[b];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float y = CAP ? cap_score<CAP>(s[b][kb][e] * c, cap) + lv[kb] : fmaf(s[b][kb][e], c, lv[kb]);
                        if (part) {
                            const int j = key0 + kb * 16 + 4 * g + e;
                            y = (j > p_q[b]) | (j <= lo_q[b]) | (bad >> kb & 1) ? -INFINITY : y;
                        }
                        s[b][kb][e] = y;
                        mx = fmaxf(mx, y);
                    }
                }
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
                const float ref = P_SHIFT8 - m[b];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p0 = exp2_hw(s[b][e / 2][2 * (e & 1)] + ref), p1 = exp2_hw(s[b][e / 2][2 * (e & 1) + 1] + ref);
                    const uint32_t near = pack2<false>(p0, p1);
                    pf[b][0][e] = near;
                    pf[b][1][e] = pack2<false>(p0 - h2f(near & 0xFFFF), p1 - h2f(near >> 16));
                    l[b] = fmaf(p0 + p1, iv[e / 2], l[b]);
                }
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const u32x2 c = read_tr8(lds_at(vt) + v_at + Lds::at(0, d));
                u32x4 vf;
                uint32_t h0, h1;
                halves4(c[0], h0, h1);
                vf[0] = h0;
                vf[1] = h1;
                halves4(c[1], h0, h1);
                vf[2] = h0;
                vf[3] = h1;
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    o[b][d] = mfma16<false>(vf, pf[b][1], o[b][d]);
                    o[b][d] = mfma16<false>(vf, pf[b][0], o[b][d]);
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
                const f32x4 y = *(const f32x4 *)((const float *)s_buf[k] + r * HD + d4 * 4);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[e] = fmaf(f, y[e], acc[e]);
            }
            if (whole) {
                const float inv = L > 0 || L != L ? 1.0f / L : 0.0f;
                uint8_t *op = a.out + (int64_t)(sv.row0 + tok) * a.o_row + head * a.o_head + d4 * 8;
                *(u32x2 *)op = u32x2{pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
            } else {
                float *pp = parts + few8_part<HD>(cut, kvh, piece, base >= 0, R);
                *(f32x4 *)(pp + r * HD + d4 * 4) = acc;
                if (d4 == 0) *(f32x2 *)(pp + R * HD + r * 2) = f32x2{mm, L};
            }
        }
    };

    if constexpr (PIECES) {
        __shared__ int s_seq[4][6][64];
        const int lane = threadIdx.x & 63;
        const SeqView view = few8_view(a, lane);
        const int n = few8_units(a, view, R);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        const int per = same(few8_per(__builtin_amdgcn_readlane(upto, 63), cut.P));
        const int base = (int)(upto - n + FEW8_BEGIN - min((int64_t)piece * per, (int64_t)1 << 30));
        const int mine_of[6] = {base, n - FEW8_BEGIN, view.row0, view.n_new, view.len, view.over};
#pragma unroll
        for (int i = 0; i < 6; i++) s_seq[w][i][lane] = mine_of[i];
        bool again = false;
        for (uint64_t mine = __ballot(n > 0 && base < per && base - FEW8_BEGIN + n > 0); mine; mine &= mine - 1) {
            const int j = __builtin_ctzll(mine);
            if (again) __syncthreads();  // the one before has been read
            again = true;
            auto of = [&](int i) { return same(s_seq[w][i][j]); };
            sequence(j, SeqView{of(2), of(3), of(4), of(5)}, per, of(0), of(1));
        }
    } else {
        const int split = piece / a.b.n_seq, si = piece - split * a.b.n_seq;
        const SeqView sv = view_of(a.b, a.kv, si);
        const int n = same(few8_steps(a, sv, R));
        if (n > split * cut.C) sequence(si, sv, split == cut.S - 1 ? 1 << 30 : cut.C, -split * cut.C, n);
    }
}

// Sequences that several pieces or splits have a part of: a workgroup for each row
template <int HD, bool BF, int M>
__global__ __launch_bounds__(256) void few8_join_kernel(ServeAttnArgs a, Few8Cut cut, const float *parts) {
    __shared__ f32x4 s_o[256];
    const int lane = threadIdx.x & 63, kvh = blockIdx.x % a.n_kv, si = blockIdx.x / a.n_kv, r = blockIdx.y, R = few8_rows<M>(a);
    const SeqView sv = view_of(a.b, a.kv, si);
    const int n = same(few8_steps(a, sv, R));
    if (r >= imin(imin(sv.n_new, M) * a.G, R)) return;
    int j0 = 0, ns;
    if (cut.S) {
        ns = split_count(n, cut.C, cut.S);
    } else {
        const int units = few8_units(a, few8_view(a, lane), R);
        const int per = same(few8_per(xsum_i<64>(units), cut.P)), base = same(xsum_i<64>(lane < si ? units : 0)) + FEW8_BEGIN;
        j0 = base / per;
        ns = (base - j0 * per + n - 1) / per + 1;
    }
    if (ns == 1) return;
    constexpr int LPR = HD / 4, AT_ONCE = 256 / LPR;  // lanes of a part's row, parts at a time
    auto part = [&](int s) { return parts + few8_part<HD>(cut, kvh, cut.S ? s * a.b.n_seq + si : j0 + s, s == 0, R); };
    const int g = threadIdx.x / LPR, d = threadIdx.x % LPR;
    const bool in = g < AT_ONCE;
    constexpr int FIRST = 16;  // requested before their weights are known
    f32x4 y[FIRST];
    float my[FIRST];
#pragma unroll
    for (int k = 0; k < FIRST; k++) {
        if (k * AT_ONCE >= ns) break;
        const float *p = part(imin(g + k * AT_ONCE, ns - 1));
        y[k] = *(const f32x4 *)(p + r * HD + d * 4);
        my[k] = p[R * HD + r * 2];
    }
    float m = -FLT_MAX, l = 0;
#pragma unroll 2
    for (int s = lane; s < ns; s += 64) {
        const f32x2 ml = *(const f32x2 *)(part(s) + R * HD + r * 2);
        const float mn = fmaxf(m, ml[0]);
        l = fmaf(l, exp2_hw(m - mn), ml[1] * exp2_hw(ml[0] - mn));
        m = mn;
    }
    const float mm = xmax_f<64>(m), L = xsum_f<64>(l * exp2_hw(m - mm)), inv = L > 0 || L != L ? 1.0f / L : 0.0f;
    f32x4 acc = f32x4{};
    auto add = [&](float ms, const f32x4 &v) {
        const float f = exp2_hw(ms - mm);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[e] = fmaf(f, v[e], acc[e]);
    };
#pragma unroll
    for (int k = 0; k < FIRST; k++) {
        if (k * AT_ONCE >= ns) break;
        if (in && g + k * AT_ONCE < ns) add(my[k], y[k]);
    }
#pragma unroll 4
    for (int s = in ? g + FIRST * AT_ONCE : ns; s < ns; s += AT_ONCE) add(part(s)[R * HD + r * 2], *(const f32x4 *)(part(s) + r * HD + d * 4));
    s_o[threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.x >= LPR) return;
    const int used = imin(AT_ONCE, ns);
    for (int k = 1; k < used; k++) acc += s_o[k * LPR + d];
    const int tok = r / a.G, head = kvh * a.G + r - tok * a.G;
    *(u32x2 *)(a.out + (int64_t)(sv.row0 + tok) * a.o_row + head * a.o_head + d * 8) = u32x2{pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
}

// ---- 32·NW query rows of a sequence and KV head, tiles of 64 (256-wide heads: 32) positions ----
//
// The schedule is that of the 16-bit tile kernel: a tile's work is cut into groups of 32
// positions, and the probabilities of group h are made while the matrix units form the outputs of
// h − 1 and the scores of h + 1.  A tile lies in LDS in f16, which its waves share: codes come
// to registers a tile ahead, each wave's 16 (8) rows, and are made f16 on their way to LDS (5
// vector instructions for 4 values), in the place of a tile that has been read by then.
//
// Bound: a SIMD's matrix and vector instructions, which hardly overlap, and a fifth of the time neither:
// of a wave's tile of 64 positions, head size 128, 1024 cycles are matrix products, and 316 vector
// instructions take about 1400 (exponentials alone 512, codes 160).  Counters, 13 sequences as below:
// the matrix units are busy for 32 % of the SIMDs' cycles, vector instructions issue in 48 %; both waves
// of a SIMD come to the same phase behind each barrier.  Eight waves to a tile (256 rows) where there
// are so many, since then each makes half as many codes: 13 sequences as below, both under a profiler,
// 215 us with four and 200 with eight.
template <int HD>
constexpr int TILE8_KT = HD <= 128 ? 64 : 32;

template <int HD>
constexpr int TILE8_KBYTES = TILE8_KT<HD> / TileLds<HD>::RPI * TileLds<HD>::K_BLOCK;
template <int HD>
constexpr int TILE8_VBYTES = TILE8_KT<HD> / TileLds<HD>::RPI * TileLds<HD>::V_BLOCK;

// Tiles [from, to) of block lb of sequence si: to the outputs, or (part given) unnormalised to part,
// as they lie in the waves' registers, with the rows' maxima and sums behind
template <int HD, bool BF, bool CAP, int NW>
__device__ __forceinline__ void tile8_piece(const ServeAttn8Args &xa, uint8_t *s_tiles, int kvh, int si, const SeqView &sv, int lb, int from, int to, float *part) {
    const ServeAttnArgs &a = xa.a;
    constexpr int TILE_M = 32 * NW;
    constexpr int KT = TILE8_KT<HD>, KB = KT / 32, RW = KT / NW, KS = HD / 16, DB = HD / 32;
    using Lds = TileLds<HD>;
    constexpr int RPI = Lds::RPI, KBYTES = TILE8_KBYTES<HD>, VBYTES = TILE8_VBYTES<HD>;
    constexpr int NG = KT / 16;                                         // groups of 16 positions, which lie in one page and block
    constexpr int CH = RW * (HD / 16), NCH = (CH + 63) / 64;            // 16-byte chunks of a wave's rows, and of a lane
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
    const int G = a.G, n_rows = sv.n_new * G;
    const int r0 = same(lb * TILE_M), r1 = same(imin(r0 + TILE_M, n_rows) - 1), tok0 = same(r0 / G), tok1 = same(r1 / G);
    const int pos0 = sv.pos0();  // position of token 0
    const KeyRange kr = key_range(sv, tok0, tok1, a.window);
    const int hi = same(kr.hi), t_first = same(first_tile(kr, KT)), nt = same(tile_count(kr, KT)), t_begin = same(t_first + imin(from, nt)), t_end = same(t_first + imin(to, nt));

    // this lane's query row, and what the rows of its wave see
    const int row = r0 + w * 32 + (lane & 31);
    const bool live = row < n_rows;
    const int tok = imin(row, n_rows - 1) / G, head = kvh * G + imin(row, n_rows - 1) - tok * G;
    const int p_q = live ? imin(pos0 + tok, sv.len - 1) : -1;
    const int lo_q = before_window(pos0 + tok, a.window);  // sees j in (lo_q, p_q]
    const bool wave_live = r0 + w * 32 <= r1;
    const int w_t0 = same(imin(r0 + w * 32, r1) / G), w_t1 = same(imin(r0 + w * 32 + 31, r1) / G);
    const int all_hi = imin(pos0 + w_t0, sv.len - 1), all_lo = before_window(pos0 + w_t1, a.window);  // every row of the wave sees (all_lo, all_hi]
    u32x4 qf[KS];
    float qs = 1, cq = 0;  // a row's power of two, and a score's factor but for its keys' scale

    // ---- codes: wave w's are rows w·RW .. of a tile, which lie in one page ----
    const int *trow = a.kv.table + (int64_t)si * a.kv.table_stride;
    const uint8_t *kbase = a.kv.k + kvh * a.kv.k_head, *vbase = a.kv.v + kvh * a.kv.v_head;
    const int k_row = (int)a.kv.k_row, v_row = (int)a.kv.v_row, page_mask = (1 << a.kv.page_shift) - 1;
    // Of a tile: page ids of its groups of 16 positions, a lane each, and (lanes 0.. and 4..) their
    // keys' and values' scales.  A page id that is none: any page that exists is read, and nobody
    // sees its values.
    const float *sbase = ((lane & 4) ? xa.s.v : xa.s.k) + (int64_t)kvh * xa.s.head;
    auto group_at = [&](int t) { return imin(t * KT + (lane & (NG - 1)) * 16, (hi - 1) & ~15); };
    auto request_pages = [&](int t) __attribute__((always_inline)) { return trow[group_at(t) >> a.kv.page_shift]; };
    auto known = [&](int id) { return (unsigned)id < (unsigned)a.kv.n_pages ? id : 0; };
    auto bad_of = [&](int ids) __attribute__((always_inline)) { return same((int)(__ballot((unsigned)ids >= (unsigned)a.kv.n_pages) & ((1u << NG) - 1))); };
    auto request_scales = [&](int t, int ids) __attribute__((always_inline)) {
        const int slot = group_at(t) & page_mask;
        return sbase[(uint64_t)(uint32_t)known(ids) * xa.s.page + (uint64_t)(uint32_t)(slot >> xa.s.block_shift) * xa.s.block];
    };
    // Which of its wave's rows and codes' chunks a lane takes, so that 8 lanes' places in LDS lie in
    // other banks: of keys, a column of rows; of values, two chunks of a row, which follow each other
    // there, the pairs of every other two rows the other way round (chunks of 13 sequences up to 8200:
    // 281 us with columns of values, 264 without the turn).
    auto place = [&](auto is_v, int i, int &r, int &c) __attribute__((always_inline)) {
        const int u = CH % 64 ? imin(i * 64 + lane, CH - 1) : i * 64 + lane;
        if constexpr (decltype(is_v)::value) {
            r = u / 2 % RW;
            c = u / (2 * RW) * 2 + u % 2;
        } else {
            r = u % RW;
            c = u / RW;
        }
    };
    int k_off[NCH], v_off[NCH];
#pragma unroll
    for (int i = 0; i < NCH; i++) {
        int r, c;
        place(std::false_type{}, i, r, c);
        k_off[i] = r * k_row + c * 16;
        place(std::true_type{}, i, r, c);
        v_off[i] = r * v_row + c * 16;
    }
    auto load = [&](auto is_v, int t, int ids, u32x4 (&raw)[NCH]) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
        const int rs = V ? v_row : k_row;
        const int g0 = imin(t * KT + w * RW, (hi - 1) & ~(RW - 1));  // rows behind the last one seen: copies of it
        const int64_t page = __builtin_amdgcn_readlane(known(ids), w * RW / 16);
        const uint8_t *src = (V ? vbase : kbase) + page * a.kv.page + (int64_t)(g0 & page_mask) * rs;
        const int last = hi - 1 - g0;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            int off = V ? v_off[i] : k_off[i];
            if (last < RW - 1) {
                int r, c;
                place(is_v, i, r, c);
                off = imin(r, last) * rs + c * 16;
            }
            raw[i] = *(const u32x4 *)(src + off);
        }
    };
    auto store = [&](auto is_v, const u32x4 (&raw)[NCH], uint32_t dst) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
#pragma unroll
        for (int i = 0; i < NCH; i++) {
            if (CH % 64 && i * 64 + lane >= CH) continue;
            int r, c;
            place(is_v, i, r, c);
            r += w * RW;
            u32x4 y[2];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t lo, hi2;
                halves4(raw[i][k], lo, hi2);
                y[k / 2][k % 2 * 2] = lo;
                y[k / 2][k % 2 * 2 + 1] = hi2;
            }
#pragma unroll
            for (int k = 0; k < 2; k++) *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(dst + (V ? Lds::value(r, (2 * c + k) ^ ((r >> 1) & 1)) : Lds::key(r, 2 * c + k))) = y[k];
        }
    };
    using K_ = std::false_type;
    using V_ = std::true_type;

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] = f32x16{};
    float m = -FLT_MAX, l = 0, ym0 = 0, ym1 = 0;  // ym: largest scores of either half of the group whose turn is next
    const SoftCap cap = CAP ? soft_cap(a) : SoftCap{};
    // the lane's places in a tile: keys row-wise, values transposed
    const int k_at = Lds::key(lane & 31, h), v_at = Lds::value(4 * h + ((lane & 15) >> 2), (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ ((lane >> 3) & 1)) + (lane & 1) * 8;

    f32x16 s[2];
    u32x4 pf[2][2];
    struct GroupScales {  // of a group's halves: a score's factor, log2 of the values' scale and its inverse
        float c[2], lv[2], iv[2];
    };
    struct TileScales {  // by lane: a scale, its log2, its inverse
        float s, lg, inv;
    };
    auto tile_scales = [&](float sc) __attribute__((always_inline)) {
        const float us = usable(sc);
        return TileScales{us, __builtin_amdgcn_logf(us), us == us ? __builtin_amdgcn_rcpf(us) : 1.0f};
    };
    auto scales_of = [&](const TileScales &t, int kb) __attribute__((always_inline)) {
        auto lane_of = [](float v, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), i)); };
        GroupScales x;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            x.c[b] = lane_of(t.s, kb * 2 + b) * cq;
            x.lv[b] = lane_of(t.lg, 4 + kb * 2 + b);
            x.iv[b] = lane_of(t.inv, 4 + kb * 2 + b);
        }
        return x;
    };
    auto max8 = [&](const f32x16 &x, int at) __attribute__((always_inline)) {
        float v = fmaxf(fmaxf(x[at], x[at + 1]), x[at + 2]);
        v = fmaxf(fmaxf(v, x[at + 3]), x[at + 4]);
        return fmaxf(fmaxf(fmaxf(v, x[at + 5]), x[at + 6]), x[at + 7]);
    };
    auto scores = [&](uint32_t kt, int kb, f32x16 &d) __attribute__((always_inline)) {
        d = f32x16{};
#pragma unroll
        for (int i = 0; i < KS; i++) d = mfma32<false>(lds_16(kt + k_at + Lds::key(kb * 32, 2 * i)), qf[i], d);
    };
    auto outputs = [&](uint32_t vt, int kb, const u32x4 (&p)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int st = 0; st < 2; st++)
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const uint32_t vp = vt + v_at + Lds::value(kb * 32 + st * 16, 4 * d);
                const u32x2 v0 = read_tr(vp), v1 = read_tr(vp + Lds::value(8, 0));
                o[d] = mfma32<false>(u32x4{v0[0], v0[1], v1[0], v1[1]}, p[st], o[d]);
            }
    };
    // group (t, kb): probabilities of its scores x → p; outputs of the group before from values
    // (vt, vkb) and probabilities po; scores of the group behind from keys (kt, nkb) → y
    auto group = [&](int key0, int bad2, const GroupScales &gs, f32x16 &x, u32x4 (&p)[2], const u32x4 (&po)[2], f32x16 &y, uint32_t vt, int vkb, uint32_t kt, int nkb) __attribute__((always_inline)) {
        // positions of the lane's scores: key0 + 4 h + (8 (e / 4) + e % 4)
        float c[2] = {gs.c[0], gs.c[1]}, lv[2] = {gs.lv[0], gs.lv[1]};
        float mx = fmaxf(fmaf(ym0, c[0], lv[0]), fmaf(ym1, c[1], lv[1]));
        const bool late = key0 + 31 > all_hi, early = key0 <= all_lo;
        if (CAP || late || early || bad2) {
#pragma unroll
            for (int e = 0; e < 16; e++) x[e] = CAP ? cap_score<CAP>(x[e] * c[e / 8], cap) + lv[e / 8] : fmaf(x[e], c[e / 8], lv[e / 8]);
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
            c[0] = c[1] = 1;
            lv[0] = lv[1] = 0;
            mx = fmaxf(max8(x, 0), max8(x, 8));
        }
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
        const float ref[2] = {P_SHIFT8 - m + lv[0], P_SHIFT8 - m + lv[1]};
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
        float ex[16], sum[2] = {0, 0};
        auto exps = [&](int i) __attribute__((always_inline)) {
            ex[2 * i] = exp2_hw(fmaf(x[2 * i], c[i / 4], ref[i / 4]));
            ex[2 * i + 1] = exp2_hw(fmaf(x[2 * i + 1], c[i / 4], ref[i / 4]));
        };
        auto pack = [&](int i) __attribute__((always_inline)) {
            p[i / 4][i % 4] = pack2<false>(ex[2 * i], ex[2 * i + 1]);
            sum[i / 4] += ex[2 * i] + ex[2 * i + 1];
        };
        auto product = [&](int u) __attribute__((always_inline)) {
            if (u < KS) y = mfma32<false>(fr[u], qf[u], y);
            else o[(u - KS) % DB] = mfma32<false>(fr[u], po[(u - KS) / DB], o[(u - KS) % DB]);
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
            if (u0 + 1 < u1) __builtin_amdgcn_sched_barrier(0);
            if (i == 6) ym0 = max8(y, 0);
            if (i == 7) ym1 = max8(y, 8);
        }
        l = fmaf(sum[1], gs.iv[1], fmaf(sum[0], gs.iv[0], l));
        // all three belong into this block: the compiler would move the probabilities to where
        // they are used, and make two copies of the block
        asm volatile("" : "+v"(p[0]), "+v"(p[1]), "+v"(l), "+v"(ym0), "+v"(ym1));
        int after = __builtin_amdgcn_readfirstlane(moved);
        asm volatile("" : "+s"(after));
        if (after) {  // the outputs so far were formed with the maximum before
#pragma unroll
            for (int d = 0; d < DB; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) o[d][e] *= al;
        }
    };

    if (t_begin < t_end) {
        // What is on its way, of a tile t: page ids of t + 3, scales of t + 1, codes of keys t + 2 and of
        // values t + KB − 1, requested in this order at t − 1, so that the codes' arrival is all that is
        // waited for.  All of it is requested whatever t, behind the last tile for its rows again: where
        // a register may or may not have been loaded, the compiler copies it, and waits for all loads
        // to do so.
        int id1, id2, ids, bad0;
        float sc0, sc;
        u32x4 rk[NCH], rv[NCH];
        const uint32_t s_k0 = lds_at(s_tiles), s_k1 = s_k0 + KBYTES, s_v0 = s_k1 + KBYTES, s_v1 = s_v0 + VBYTES;
        {
            const int id0 = request_pages(t_begin);
            id1 = request_pages(t_begin + 1);
            id2 = request_pages(t_begin + 2);
            ids = request_pages(t_begin + 3);
            sc0 = request_scales(t_begin, id0);
            sc = request_scales(t_begin + 1, id1);
            {
                const uint8_t *qp = a.q + (int64_t)(sv.row0 + tok) * a.q_row + head * a.q_head + h * 16;
#pragma unroll
                for (int i = 0; i < KS; i++) qf[i] = live ? *(const u32x4 *)(qp + i * 32) : u32x4{0, 0, 0, 0};
            }
            bad0 = bad_of(id0);
            u32x4 k0[NCH], k1[NCH], v0[NCH];  // the first tiles, all requested at once, and the queries before them
            load(K_{}, t_begin, id0, k0);
            load(K_{}, t_begin + 1, id1, k1);
            load(V_{}, t_begin, id0, KB == 2 ? v0 : rv);
            if constexpr (KB == 2) load(V_{}, t_begin + 1, id1, rv);
            load(K_{}, t_begin + 2, id2, rk);
            if constexpr (BF) {
                float most = 0;
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(value16<true>(qf[i][e / 2] >> (e & 1) * 16 & 0xFFFF)));
                float a0, a1;
                pair_f<32>(most, a0, a1);
                const int ex = 14 - __builtin_amdgcn_frexp_expf(fminf(fmaxf(a0, a1), FLT_MAX));  // infinities stay what they are
                qs = __builtin_amdgcn_ldexpf(1.0f, -ex);
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        qf[i][e] = pack2<false>(__builtin_amdgcn_ldexpf(value16<true>(qf[i][e] & 0xFFFF), ex), __builtin_amdgcn_ldexpf(value16<true>(qf[i][e] >> 16), ex));
            }
            cq = CAP ? qs : a.scale * LOG2E_F * qs;
            store(K_{}, k0, s_k0);
            store(K_{}, k1, s_k1);
            if constexpr (KB == 2) store(V_{}, v0, s_v0);
        }
        // the first group's outputs before it: zeros
        for (int i = w; i < 32 / RPI; i += NW) *(__attribute__((address_space(3))) u32x4 *)(uintptr_t)(s_v1 + Lds::value((KB - 1) * 32 + i * RPI, 0) + lane * 16) = u32x4{0, 0, 0, 0};
        pf[1][0] = pf[1][1] = u32x4{0, 0, 0, 0};
        lds_barrier();
        if (wave_live) {
            scores(s_k0, 0, s[0]);
            ym0 = max8(s[0], 0);
            ym1 = max8(s[0], 8);
        }
        TileScales ts = tile_scales(sc0);
        auto tile = [&](int t, uint32_t k_t, uint32_t k_n, uint32_t v_t, uint32_t v_n, f32x16 &x0, f32x16 &x1, u32x4 (&p0)[2], u32x4 (&p1)[2]) __attribute__((always_inline)) {
            const int bad = bad0;
            if constexpr (KB == 2)
                if (wave_live) group(t * KT, bad & 3, scales_of(ts, 0), x0, p0, p1, x1, v_n, 1, k_t, 1);
            lds_barrier();
            store(K_{}, rk, k_t);
            store(V_{}, rv, KB == 2 ? v_n : v_t);
            const GroupScales gs = scales_of(ts, KB - 1);
            ts = tile_scales(sc);
            bad0 = bad_of(id1);
            const int id3 = ids;
            ids = request_pages(t + 4);
            sc = request_scales(t + 2, id2);
            load(V_{}, t + KB, KB == 2 ? id2 : id1, rv);
            load(K_{}, t + 3, id3, rk);
            id1 = id2;
            id2 = id3;
            if (wave_live) {
                if constexpr (KB == 2) group(t * KT + 32, bad >> 2, gs, x1, p1, p0, x0, v_t, 0, k_n, 0);
                else group(t * KT, bad, gs, x0, p0, p1, x1, v_n, 0, k_n, 0);
            }
        };
        if constexpr (KB == 2) {
            // one tile to a turn, so that the registers that are on their way are the same in every turn
            uint32_t kt = s_k0, kn = s_k1, vt = s_v0, vn = s_v1;
            for (int t = t_begin; t < t_end; t++) {
                tile(t, kt, kn, vt, vn, s[0], s[1], pf[0], pf[1]);
                const uint32_t k = kt, v = vt;
                kt = kn;
                kn = k;
                vt = vn;
                vn = v;
            }
        } else {
            for (int t = t_begin; t < t_end; t += 2) {
                tile(t, s_k0, s_k1, s_v0, s_v1, s[0], s[1], pf[0], pf[1]);
                if (t + 1 >= t_end) break;
                tile(t + 1, s_k1, s_k0, s_v1, s_v0, s[1], s[0], pf[1], pf[0]);
            }
        }
        // the last group's outputs
        const bool odd = (t_end - t_begin) & 1;
        if constexpr (KB == 1) lds_barrier();
        if (wave_live) {
            if (odd) outputs(s_v0, KB - 1, pf[KB == 2 ? 1 : 0]);
            else outputs(s_v1, KB - 1, pf[1]);
        }
    }
    if (!live) return;
    float l0, l1;
    pair_f<32>(l, l0, l1);
    l = l0 + l1;
    if (!part) {
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
        float *pp = part + w * (32 * HD) + lane * 4;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int e = 0; e < 4; e++) *(f32x4 *)(pp + (d * 4 + e) * 256) = f32x4{o[d][4 * e], o[d][4 * e + 1], o[d][4 * e + 2], o[d][4 * e + 3]};
        if (h == 0) *(f32x2 *)(part + TILE_M * HD + (w * 32 + (lane & 31)) * 2) = f32x2{m, l};
    }
}

// The work of a launch, divided evenly: the blocks of all sequences in a row, each as long as its
// tiles take, are cut into as many pieces as workgroups run at a time (per KV head), wherever the
// cuts fall.  A workgroup goes through the blocks of its piece; one that it has all of goes to the
// outputs, and at most two (its first, its last) to partial results, which tile8_join_kernel adds
// up.  With a workgroup for each block, the longest sequence's ran on while the others' were done:
// chunks of 13 sequences up to 8200 258 us; in pieces 183 (kernels alone, under a profiler: 183 the
// tiles, at a lower clock, 6.5 the plan and 11.4 the join).
struct Tile8Plan {
    int64_t total;  // what the tiles of all blocks take
    int n, pad;     // blocks
};
struct Tile8Item {
    int64_t before;  // what the blocks ahead take
    int si, lb;      // sequence, and block of its rows
    int row0, n_new, len, over;
};
constexpr int TILE8_FULL = 16, TILE8_BEGIN = 72, TILE8_LEAST = 10;  // a full tile's time, that until a block's first tile; tiles that a piece is worth
struct Tile8Share {
    int64_t total;
    int P;
    __device__ __forceinline__ int64_t begin(int j) const { return (total * j + P - 1) / P; }  // of piece j
    __device__ __forceinline__ int owner(int64_t x) const { return (int)(x * P / total); }
};
__device__ __forceinline__ Tile8Share tile8_share(int64_t total, int P) {
    return Tile8Share{total, (int)imax(1, (int)min((int64_t)P, total / (TILE8_LEAST * TILE8_FULL)))};
}
struct Tile8Block {
    int rows, nt, cost;  // rows, tiles, and what one takes: waves without rows help to make it
    __device__ __forceinline__ int units() const { return TILE8_BEGIN + imax(nt, 1) * cost; }
    // tiles that begin in the block's first x units
    __device__ __forceinline__ int upto(int64_t x) const { return (int)min((int64_t)imax(nt, 1), (max(x - TILE8_BEGIN, (int64_t)0) + cost - 1) / cost); }
};
template <int M>
__device__ __forceinline__ Tile8Block tile8_block(const ServeAttnArgs &a, const SeqView &sv, int lb, int KT) {
    const int n_rows = sv.n_new * a.G, r0 = lb * M, r1 = imin(r0 + M, n_rows) - 1;
    return Tile8Block{r1 - r0 + 1, tile_count(key_range(sv, r0 / a.G, r1 / a.G, a.window), KT), 11 + 5 * ((r1 - r0) / 32 + 1) * 32 / M};
}
__device__ __forceinline__ SeqView tile8_seq(const Tile8Item &it) { return uniform(SeqView{it.row0, it.n_new, it.len, it.over}); }

// items, and (first) the item with which each piece begins
template <int M>
__global__ __launch_bounds__(1024) void tile8_plan_kernel(ServeAttnArgs a, int KT, Tile8Plan *plan, Tile8Item *items, int *first, int P) {
    __shared__ int64_t s_sum[16];
    __shared__ int s_n[16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int64_t before = 0;
    int n = 0;
    for (int b0 = 0; b0 < a.n_blocks; b0 += 1024) {
        const int id = b0 + tid;
        int64_t units = 0;
        Tile8Item it{};
        if (id < a.n_blocks) {
            int lo = 0, hi = a.b.n_seq;  // the last sequence whose first id is at or before this one
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2;
                if (block_base(iclamp(a.b.starts[mid], 0, a.b.n_rows), mid, a.G, M) <= id) lo = mid;
                else hi = mid;
            }
            const SeqView sv = seq_view(a.b.starts[lo], a.b.starts[lo + 1], a.b.lens[lo], a.b.n_rows, a.kv.cap);
            it = Tile8Item{0, lo, id - block_base(sv.row0, lo, a.G, M), sv.row0, sv.n_new, sv.len, sv.over};
            // blocks whose rows see nothing, too: their zeros are written
            if (it.lb >= 0 && it.lb < (sv.n_new * a.G + M - 1) / M) units = tile8_block<M>(a, sv, it.lb, KT).units();
        }
        int64_t x = units;
        int c = units > 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t y = __shfl_up(x, o);
            const int d = __shfl_up(c, o);
            if (lane >= o) {
                x += y;
                c += d;
            }
        }
        __syncthreads();
        if (lane == 63) {
            s_sum[w] = x;
            s_n[w] = c;
        }
        __syncthreads();
        it.before = before + x - units;
        int place = n + c - (units > 0);
        for (int i = 0; i < 16; i++) {
            if (i < w) {
                it.before += s_sum[i];
                place += s_n[i];
            }
            before += s_sum[i];
            n += s_n[i];
        }
        if (units) items[place] = it;
    }
    if (tid == 0) *plan = Tile8Plan{before, n, 0};
    __syncthreads();
    const Tile8Share share = tile8_share(before, P);
    for (int j = tid; j < share.P && n; j += 1024) {
        const int64_t begin = share.begin(j);
        int lo = 0, hi = n;  // the last block that begins at or before it
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (items[mid].before <= begin) lo = mid;
            else hi = mid;
        }
        first[j] = lo;
    }
}

template <int HD, bool BF, bool CAP, int NW>
__global__ __launch_bounds__(64 * NW, HD <= 128 ? 2 : NW / 4) void attn8_tile_kernel(ServeAttn8Args x, const Tile8Plan *plan, const Tile8Item *items, const int *first, int P, float *parts) {
    constexpr int M = 32 * NW, KT = TILE8_KT<HD>;
    __shared__ __align__(16) uint8_t s_tiles[2 * TILE8_KBYTES<HD> + 2 * TILE8_VBYTES<HD>];
    const ServeAttnArgs &a = x.a;
    // a KV head's workgroups on one XCD where there are 8 of them
    const int kvh = blockIdx.x % a.n_kv, j = blockIdx.x / a.n_kv;
    int i = 0, n = 1;
    int64_t begin = 0, end = 0;
    Tile8Item it{};
    if (plan) {
        i = first[j];  // there for every j
        n = same(plan->n);
        if (n == 0) return;
        const Tile8Share share = tile8_share(plan->total, P);
        if (j >= share.P) return;
        i = same(i);
        it = items[i];
        begin = share.begin(j);
        end = share.begin(j + 1);
    } else {  // a workgroup for each block
        const SeqView sv = find_seq(a.b, a.kv, j, it.si, [&](int s, int q) { return block_base(iclamp(s, 0, a.b.n_rows), q, a.G, M); });
        const int blocks = (sv.n_new * a.G + M - 1) / M;
        it.lb = blocks - 1 - (j - block_base(sv.row0, it.si, a.G, M));  // a sequence's longest rows first
        if (it.lb < 0 || it.lb >= blocks) return;
        it.row0 = sv.row0;
        it.n_new = sv.n_new;
        it.len = sv.len;
        it.over = sv.over;
    }
    for (;;) {
        const SeqView sv = tile8_seq(it);
        const int si = same(it.si), lb = same(it.lb);
        int from = 0, to = INT32_MAX;
        float *part = nullptr;
        bool more = false;
        if (plan) {
            const int64_t before = it.before;
            const Tile8Block k = tile8_block<M>(a, sv, lb, KT);
            from = k.upto(begin - before);
            to = k.upto(end - before);
            if (from > 0 || to < imax(k.nt, 1)) part = parts + (((int64_t)kvh * P + j) * 2 + (begin >= before ? 0 : 1)) * (M * (HD + 2));
            more = ++i < n && before + k.units() < end;
            if (more) it = items[i];
            lds_barrier();  // the tiles of the piece before have been read
        }
        if (from < to) tile8_piece<HD, BF, CAP, NW>(x, s_tiles, kvh, si, sv, lb, from, to, part);
        if (!more) break;
    }
}

// Blocks whose tiles several workgroups took, a workgroup for each of their waves' parts
template <int HD, bool BF, int M>
__global__ __launch_bounds__(256) void tile8_join_kernel(ServeAttnArgs a, int KT, const Tile8Plan *plan, const Tile8Item *items, int P, const float *parts) {
    const int kvh = blockIdx.x % a.n_kv, i = blockIdx.x / a.n_kv, w = blockIdx.y;
    if (i >= plan->n) return;
    const Tile8Share share = tile8_share(plan->total, P);
    const Tile8Item it = items[i];
    const SeqView sv = tile8_seq(it);
    const Tile8Block k = tile8_block<M>(a, sv, it.lb, KT);
    if (w * 32 >= k.rows) return;
    const int j0 = share.owner(it.before + TILE8_BEGIN), j1 = share.owner(it.before + TILE8_BEGIN + (int64_t)(imax(k.nt, 1) - 1) * k.cost);
    if (j0 == j1) return;
    const int lane = threadIdx.x & 63, r = w * 32 + (lane & 31);
    if (r >= k.rows) return;
    constexpr int N = HD / 32;  // 16-byte pieces of a lane: (d, e) = threadIdx.x / 64 + 4 u
    float m = -FLT_MAX, l = 0;
    f32x4 o[N];
#pragma unroll
    for (int u = 0; u < N; u++) o[u] = f32x4{0, 0, 0, 0};
    for (int j = j0; j <= j1; j++) {
        const float *p = parts + (((int64_t)kvh * P + j) * 2 + (share.begin(j) >= it.before ? 0 : 1)) * (M * (HD + 2));
        const f32x2 ml = *(const f32x2 *)(p + M * HD + r * 2);
        f32x4 y[N];
#pragma unroll
        for (int u = 0; u < N; u++) y[u] = *(const f32x4 *)(p + w * (32 * HD) + (threadIdx.x / 64 + 4 * u) * 256 + lane * 4);
        const float mn = fmaxf(m, ml[0]), f = exp2_hw(m - mn), e = exp2_hw(ml[0] - mn);
        m = mn;
        l = fmaf(l, f, ml[1] * e);
#pragma unroll
        for (int u = 0; u < N; u++)
#pragma unroll
            for (int q = 0; q < 4; q++) o[u][q] = fmaf(o[u][q], f, y[u][q] * e);
    }
    const float inv = l > 0 || l != l ? 1.0f / l : 0.0f;
    const int row = it.lb * M + r, tok = row / a.G, head = kvh * a.G + row - tok * a.G;
    uint8_t *op = a.out + (int64_t)(sv.row0 + tok) * a.o_row + head * a.o_head + (lane >> 5) * 8;
#pragma unroll
    for (int u = 0; u < N; u++) *(u32x2 *)(op + (threadIdx.x / 64 + 4 * u) * 16) = u32x2{pack2<BF>(o[u][0] * inv, o[u][1] * inv), pack2<BF>(o[u][2] * inv, o[u][3] * inv)};
}

// ---- new rows into their pages ----
//
// A wave takes what a call brings to one block of positions, of one head's keys or values: the
// rows' largest value, the block's new scale, the codes of earlier positions where it has grown,
// and the new ones.  Codes are those of the formula, ties to even (codes8).
// Blocks are numbered without a list: sequence i owns ids from ⌊start / block⌋ + 2 i on, which
// are enough, since n new tokens touch at most ⌊n / block⌋ + 2 blocks.
//
// Bound: loads behind one another (the sequence, the rows, the page and scale meanwhile), and for
// long prompts the second reading of blocks over 16 positions, from L2.  61 tokens for 4 heads of
// 128 4.3 us; 2854 rows for 8 heads, f32, blocks of 32 (29 MB) 11.0 us.  32 rows kept in registers
// 0.8 more and 0.9 less: steps of single tokens are what a server makes most of.
template <int SRC>  // ggml type
__device__ __forceinline__ void load8(const uint8_t *p, float (&v)[8]) {
    if constexpr (SRC == T_F32) {
        const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    } else {
        const u32x4 a = *(const u32x4 *)p;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = value16<SRC == T_BF16>(a[e / 2] >> (e & 1) * 16 & 0xFFFF);
    }
}

// 8 codes x / s, to the nearest whole number, ties to even.  In f32, by the hardware's inverse, a quotient
// is off by under 2^-15 (of numbers up to 127.5: two roundings and one unit of the inverse, 2^-22 in
// all), so what is 2^-14 or more away from half way between two numbers goes the right way.  The
// others are formed in f64 (prompts 12.2 us with all of them so): x and s have at most 32 bits, so a
// quotient that is not half way itself is 2^-34 of its size away, and x · (1 / s), good to 2^-52, goes
// the right way.  One that is may go either way; what is left then is s / 2 exactly, in the fma as
// in truth.
template <class F>
__device__ __forceinline__ u32x2 codes8(F x, float s) {
    const float inv_f = __builtin_amdgcn_rcpf(s);
    int c[8];
    bool near = false;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float t = (float)x(e) * inv_f, q = rintf(t);
        near = near || fabsf(t - q) > 0.5f - 0x1p-14f;
        c[e] = (int)q;
    }
    if (near) {
        const double inv = 1.0 / (double)s;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double y = x(e), q = rint(y * inv), left = fma(-q, (double)s, y);
            c[e] = (int)q;
            if (fabs(left) == 0.5 * s && (c[e] & 1)) c[e] += left > 0 ? 1 : -1;
        }
    }
    u32x2 y = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e++) y[e / 4] |= ((uint32_t)c[e] & 255) << e % 4 * 8;
    return y;
}

template <int HD, int SRC>
__global__ __launch_bounds__(256) void paged_append8_kernel(PagedAppend8Args x) {
    const PagedAppendArgs &a = x.a;
    constexpr int CPR = HD / 8, RP = 64 / CPR, ROWS = 16, NP = (ROWS + RP - 1) / RP;  // lanes of a row, rows of a pass, rows and passes at a time
    constexpr int ES = SRC == T_F32 ? 4 : 2;
    const int lane = threadIdx.x & 63, u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = u / (2 * a.n_kv), h = u / 2 % a.n_kv;
    const bool is_v = u & 1;
    const int bs = x.s.block_shift, B = 1 << bs;
    if (id >= append8_id(a.b.n_rows, a.b.n_seq, bs)) return;
    int si;
    const SeqView sv = find_seq(a.b, a.kv, id, si, [&](int s, int i) { return append8_id(iclamp(s, 0, a.b.n_rows), i, bs); });
    const int pos0 = sv.pos0(), from = imax(pos0, 0), to = imin(pos0 + sv.n_new, sv.len);  // positions that are written
    const int b0 = same(((from >> bs) + id - append8_id(sv.row0, si, bs)) << bs);          // the block's first position
    if (b0 >= to) return;
    const int first = imax(b0, from), n = imin(b0 + B, to) - first, slot0 = b0 & ((1 << a.kv.page_shift) - 1);
    if (n <= 0) return;
    const uint8_t *src = (is_v ? a.v + h * a.v_head : a.k + h * a.k_head) + (int64_t)(sv.row0 + first - pos0) * (is_v ? a.v_row : a.k_row);
    const int64_t src_row = is_v ? a.v_row : a.k_row, row = is_v ? a.kv.v_row : a.kv.k_row;
    const int r = lane / CPR, ch = lane % CPR;
    const bool on = r < RP;

    float v[NP][8];  // 16 rows at a time; those of a block of 16 stay
    auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int q = r0 + i * RP + r;
            if (on && i * RP + r < ROWS && q < n) load8<SRC>(src + q * src_row + ch * (8 * ES), v[i]);
            else
#pragma unroll
                for (int e = 0; e < 8; e++) v[i][e] = 0;
        }
    };
    load(0);
    int page;
    if (!page_of(a.kv, a.kv.table + (int64_t)si * a.kv.table_stride, b0, page)) return;
    page = same(page);
    float *sp = (is_v ? x.s.v : x.s.k) + (int64_t)page * x.s.page + (int64_t)(slot0 >> bs) * x.s.block + (int64_t)h * x.s.head;
    float was = first > b0 ? *sp : 0.0f;
    uint8_t *dst = const_cast<uint8_t *>(is_v ? a.kv.v + h * a.kv.v_head : a.kv.k + h * a.kv.k_head) + page * a.kv.page + slot0 * row;
    float most = 0;
    bool fine = true;
    for (int r0 = 0; r0 < n; r0 += ROWS) {
        if (r0) load(r0);
#pragma unroll
        for (int i = 0; i < NP; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                fine = fine && fabsf(v[i][e]) <= FLT_MAX;
                most = fmaxf(most, fabsf(v[i][e]));
            }
    }
    was = was != 0 ? usable(was) : 0.0f;
    most = xmax_f<64>(most);
    float now = (float)((double)most / 127.0);
    if (now < SCALE8_MIN) now = 0;
    if (__any(!fine) || now > SCALE8_MAX || was != was) now = NAN;
    else now = fmaxf(now, was);
    if (lane == 0) *sp = now;
    if (first > b0 && now > was) {  // codes of earlier positions
        for (int q = r; q < first - b0; q += RP) {
            if (!on) break;
            u32x2 *p = (u32x2 *)(dst + q * row + ch * 8);
            const u32x2 y = *p;
            *p = codes8([&](int e) { return (double)(int8_t)(y[e / 4] >> e % 4 * 8) * (double)was; }, now);
        }
    }
    for (int r0 = 0; r0 < n; r0 += ROWS) {
        if (n > ROWS) load(r0);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int q = r0 + i * RP + r;
            if (!(on && i * RP + r < ROWS && q < n)) continue;
            *(u32x2 *)(dst + (first - b0 + q) * row + ch * 8) = now > 0 ? codes8([&](int e) { return v[i][e]; }, now) : u32x2{0, 0};
        }
    }
}

int tile8_waves(const ServeAttnArgs &a) { return tile8_wave_count(a.b.n_rows, a.b.n_seq, a.b.max_new, a.G, a.n_kv, a.hd); }
int tile8_m(const ServeAttnArgs &a) { return 32 * tile8_waves(a); }
int tile8_kt(int hd) { return hd <= 128 ? TILE8_KT<128> : TILE8_KT<256>; }

// positions that a block's rows see, at most
int64_t span8(const ServeAttnArgs &a, int tokens, int KT) {
    return a.window > 0 ? std::min<int64_t>(a.b.max_len, (int64_t)a.window + std::min(a.b.max_new, tokens) + KT) : a.b.max_len;
}

bool few8(const ServeAttnArgs &a) { return few_row_blocks(true, a.b.max_new, a.G) > 0; }

int few8_rows_most(const ServeAttnArgs &a) { return (int)std::min<int64_t>((int64_t)a.b.max_new * a.G, 16 * few_row_blocks(true, a.b.max_new, a.G)); }
Few8Cut few8_cut(const ServeAttnArgs &a) {
    const int steps = (int)((span8(a, FEW_ROWS, FEW8_STEP) + FEW8_STEP - 1) / FEW8_STEP), slots = 256 * few8_waves(a.hd, few_row_blocks(true, a.b.max_new, a.G), true);
    const int64_t wgs = (int64_t)a.b.n_seq * a.n_kv;
    if (steps >= 2 * FEW8_LEAST && a.b.n_seq > 1 && a.b.n_seq <= FEW8_SEQS && wgs <= slots)
        return Few8Cut{(int)std::min<int64_t>((int64_t)a.b.n_seq * steps / FEW8_LEAST, slots / a.n_kv), 0, 0};
    // splits of two steps where workgroups are few; where they fill the card, of twelve (500 sequences
    // of up to 1500, 32/4 heads of 128, 111 us with two, 87 whole; 128 of up to 8000, 202 and 242)
    const SplitPlan p = split_plan(wgs, steps, 4096, wgs < 512 ? FEW8_LEAST : 12, SERVE_MAX_SPLIT);
    return Few8Cut{a.b.n_seq * p.S, p.S, p.C};
}

// Pieces per KV head that a launch of the tile kernel is divided into, or 0: a workgroup for each
// block, where the longest is too short to be cut.
int tile8_pieces(const ServeAttnArgs &a) {
    const int KT = tile8_kt(a.hd), M = tile8_m(a);
    const int64_t tiles = (span8(a, M / a.G + 1, KT) + KT - 1) / KT, blocks = block_count(a.b.n_rows, a.b.n_seq, a.G, M);
    if (tiles < 2 * TILE8_LEAST) return 0;
    const int slots = (a.hd <= 32 ? 3 : a.hd <= 128 ? 2 : 1) * 1024 / tile8_waves(a) / a.n_kv;
    return (int)std::clamp<int64_t>(blocks * tiles / TILE8_LEAST, 1, std::max(slots, 1));
}

struct Tile8Ws {
    size_t first, parts, bytes;  // where they begin, behind the plan and its items
};
Tile8Ws tile8_ws(const ServeAttnArgs &a) {
    const size_t P = tile8_pieces(a), blocks = block_count(a.b.n_rows, a.b.n_seq, a.G, tile8_m(a));
    if (!P) return Tile8Ws{0, 0, 0};
    Tile8Ws w;
    w.first = sizeof(Tile8Plan) + blocks * sizeof(Tile8Item);
    w.parts = w.first + (P + 3) / 4 * 16;
    w.bytes = w.parts + a.n_kv * P * 2 * tile8_m(a) * (a.hd + 2) * sizeof(float);
    return w;
}

template <int HD, bool BF, int NW>
void launch_tile(const ServeAttn8Args &x, void *ws, hipStream_t st) {
    constexpr int M = 32 * NW;
    const ServeAttnArgs &a = x.a;
    const int P = tile8_pieces(a), grid = (P ? P : a.n_blocks) * a.n_kv;
    const Tile8Ws w = tile8_ws(a);
    Tile8Plan *plan = P ? (Tile8Plan *)ws : nullptr;
    Tile8Item *items = (Tile8Item *)(plan + 1);
    int *first = (int *)((uint8_t *)ws + w.first);
    float *parts = (float *)((uint8_t *)ws + w.parts);
    if (P) tile8_plan_kernel<M><<<1, 1024, 0, st>>>(a, TILE8_KT<HD>, plan, items, first, P);
    if (a.softcap > 0) attn8_tile_kernel<HD, BF, true, NW><<<grid, 64 * NW, 0, st>>>(x, plan, items, first, P, parts);
    else attn8_tile_kernel<HD, BF, false, NW><<<grid, 64 * NW, 0, st>>>(x, plan, items, first, P, parts);
    if (P) tile8_join_kernel<HD, BF, M><<<dim3(a.n_blocks * a.n_kv, NW), 256, 0, st>>>(a, TILE8_KT<HD>, plan, items, P, parts);
}

template <int HD, bool BF, int NB>
void launch_few(const ServeAttn8Args &x, void *ws, hipStream_t st) {
    const ServeAttnArgs &a = x.a;
    const Few8Cut cut = few8_cut(a);
    const int64_t grid = (int64_t)cut.P * a.n_kv;
    if (cut.S) {
        if (a.softcap > 0) attn8_few_kernel<HD, BF, true, NB, false><<<grid, 256, 0, st>>>(x, cut, (float *)ws);
        else attn8_few_kernel<HD, BF, false, NB, false><<<grid, 256, 0, st>>>(x, cut, (float *)ws);
    } else {
        if (a.softcap > 0) attn8_few_kernel<HD, BF, true, NB, true><<<grid, 256, 0, st>>>(x, cut, (float *)ws);
        else attn8_few_kernel<HD, BF, false, NB, true><<<grid, 256, 0, st>>>(x, cut, (float *)ws);
    }
    if (cut.S != 1) few8_join_kernel<HD, BF, 16 * NB><<<dim3(a.b.n_seq * a.n_kv, few8_rows_most(a)), 256, 0, st>>>(a, cut, (const float *)ws);
}

template <int HD, bool BF>
void launch_hd(const ServeAttn8Args &x, void *ws, hipStream_t st) {
    const ServeAttnArgs &a = x.a;
    const int few = few_row_blocks(true, a.b.max_new, a.G);
    if (few == 1) return launch_few<HD, BF, 1>(x, ws, st);
    if (few == 2) return launch_few<HD, BF, 2>(x, ws, st);
    if constexpr (HD <= 128) {
        if (tile8_waves(a) == 8) return launch_tile<HD, BF, 8>(x, ws, st);
    }
    launch_tile<HD, BF, 4>(x, ws, st);
}

template <bool BF>
void launch_ty(const ServeAttn8Args &x, void *ws, hipStream_t st) {
    switch (x.a.hd) {
    case 32: launch_hd<32, BF>(x, ws, st); break;
    case 64: launch_hd<64, BF>(x, ws, st); break;
    case 96: launch_hd<96, BF>(x, ws, st); break;
    case 128: launch_hd<128, BF>(x, ws, st); break;
    default: launch_hd<256, BF>(x, ws, st); break;
    }
}

template <int SRC>
void launch_append(const PagedAppend8Args &x, int grid, hipStream_t st) {
    switch (x.a.hd) {
    case 32: paged_append8_kernel<32, SRC><<<grid, 256, 0, st>>>(x); break;
    case 64: paged_append8_kernel<64, SRC><<<grid, 256, 0, st>>>(x); break;
    case 96: paged_append8_kernel<96, SRC><<<grid, 256, 0, st>>>(x); break;
    case 128: paged_append8_kernel<128, SRC><<<grid, 256, 0, st>>>(x); break;
    default: paged_append8_kernel<256, SRC><<<grid, 256, 0, st>>>(x); break;
    }
}

}  // namespace

size_t serve_attn8_ws(const ServeAttnArgs &a) {
    if (!few8(a)) return tile8_ws(a).bytes;
    const Few8Cut cut = few8_cut(a);
    return cut.S == 1 ? 0 : (size_t)cut.P * a.n_kv * (cut.S ? 1 : 2) * part_floats(few8_rows_most(a), a.hd) * sizeof(float);
}

void launch_serve_attn8(ServeAttn8Args x, void *ws, hipStream_t st) {
    ServeAttnArgs &a = x.a;
    if (!few8(a)) a.n_blocks = (int)block_count(a.b.n_rows, a.b.n_seq, a.G, tile8_m(a));
    if (a.ty == T_BF16) launch_ty<true>(x, ws, st);
    else launch_ty<false>(x, ws, st);
}

void launch_paged_append8(const PagedAppend8Args &x, hipStream_t st) {
    const int64_t waves = (int64_t)append8_count(x.a.b.n_rows, x.a.b.n_seq, x.s.block_shift) * x.a.n_kv * 2;
    const int grid = (int)((waves + 3) / 4);
    if (x.a.src_ty == T_F32) launch_append<T_F32>(x, grid, st);
    else if (x.a.src_ty == T_BF16) launch_append<T_BF16>(x, grid, st);
    else launch_append<T_F16>(x, grid, st);
}

}  // namespace rie
