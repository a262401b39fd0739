// serve_device.hpp — what the kernels of the batched serving operators share: matrix
// instructions on 16-bit operands, places in LDS, where a batch's sequences and pages lie,
// softcaps.
#pragma once

#include "device.hpp"
#include "serve.hpp"

#include <cfloat>

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

}  // namespace

}  // namespace rie
