// serve_index.hpp — where the sequences of a serving batch lie: their rows, positions
// and pages, the blocks of query rows that workgroups take, and the splits of long
// caches.  The starts, lengths and page tables are device memory that the host never
// reads, so everything taken from them is clamped here before it is used as an index;
// the same functions compile for the host, where tests check them.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#ifdef __HIPCC__
#define RIE_HD __host__ __device__ __forceinline__
#else
#define RIE_HD inline
#endif

namespace rie {

RIE_HD int iclamp(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }
RIE_HD int imin(int a, int b) { return a < b ? a : b; }
RIE_HD int imax(int a, int b) { return a > b ? a : b; }

// One sequence of a batch: rows [row0, row0 + n_new) hold its new tokens, the last of
// its len + over positions, of which the first len can be addressed.  Token t is at position
// pos0() + t (negative: before the sequence's first position, a token that sees nothing;
// len or more: a token that is written nowhere and sees the addressable ones before it).
struct SeqView {
    int row0, n_new, len, over = 0;
    RIE_HD int pos0() const { return len + over - n_new; }
};
// starts[i], starts[i + 1] and lens[i] as the device memory has them; n_rows rows exist,
// cap positions can be addressed
RIE_HD SeqView seq_view(int start, int end, int len, int n_rows, int cap) {
    SeqView s;
    s.row0 = iclamp(start, 0, n_rows);
    s.n_new = iclamp(end, s.row0, n_rows) - s.row0;
    s.len = iclamp(len, 0, cap);
    s.over = len > cap ? len - cap : 0;
    return s;
}

// First of the block ids that belong to the sequence starting at row `start`, number i
// of the batch, where a block is M consecutive query rows (token · G + head of the
// group).  Sequence i owns the ids up to the next one's first: at least ⌈n_new·G/M⌉, so
// that no list of blocks has to be made before the launch.
RIE_HD int block_base(int start, int i, int G, int M) { return (int)((int64_t)start * G / M) + i; }
inline int64_t block_count(int n_rows, int n_seq, int G, int M) { return (int64_t)n_rows * G / M + n_seq; }

// The same for blocks of 2^shift positions of a cache of 8 bits that a sequence's new tokens are
// written to: n of them touch at most ⌊n / 2^shift⌋ + 2 blocks, wherever the first one lies.
RIE_HD int append8_id(int start, int i, int shift) { return (start >> shift) + 2 * i; }
inline int64_t append8_count(int n_rows, int n_seq, int shift) { return ((int64_t)n_rows >> shift) + 2 * (int64_t)n_seq; }

// the last position before the window of a token at position p (window 0: none), for any p and
// any window of 31 bits
RIE_HD int before_window(int p, int window) { return window > 0 ? imax(p, -1) - window : -1; }
// Positions [lo, hi) that at least one of tokens t0..t1 of s sees (window 0: all up to its own)
struct KeyRange {
    int lo, hi;
};
RIE_HD KeyRange key_range(const SeqView &s, int t0, int t1, int window) {
    KeyRange r;
    const int p0 = s.pos0() + t0, p1 = s.pos0() + t1;
    r.hi = iclamp(p1 + 1, 0, s.len);
    r.lo = imax(before_window(p0, window) + 1, 0);
    if (r.lo > r.hi) r.lo = r.hi;
    return r;
}
// tiles of KT positions that hold [lo, hi): the first one, and how many
RIE_HD int first_tile(const KeyRange &r, int KT) { return r.lo / KT; }
RIE_HD int tile_count(const KeyRange &r, int KT) { return r.hi > r.lo ? (r.hi + KT - 1) / KT - r.lo / KT : 0; }
// splits of nt tiles when a split takes C of them and the last of S all that are left
RIE_HD int split_count(int nt, int C, int S) { return imax(1, imin(S, (nt + C - 1) / C)); }

// Which kernel a launch over sequences of at most max_new tokens takes, G query heads to a KV
// head: 1 or 2, the blocks of 16 query rows of the few-rows kernel, or 0, the tile kernel.  The
// few-rows kernel reads pages only; it keeps what a probability's rounding leaves.  Both
// sides, few rows and tiles, in us (bf16, 8 KV heads of 128): one sequence of 30000 positions, 4
// rows 28.8 and 38.4, 32 rows 37.3 and 40.2; 16 of 4000: 49.7 and 52.6, 70.2 and 51.5; 64 of
// 4000: 207 and 181, 270 and 184.  One KV head of 256, 64 of 4000: 47.0 and 74.3, 90.7 and 82.0.
// 36 rows, tiles: 41.5, 53.3, 264 and 81.5.
constexpr int FEW_ROWS = 32;
inline int few_row_blocks(bool paged, int max_new, int G) {
    const int64_t rows = (int64_t)max_new * G;
    return !paged || rows > FEW_ROWS ? 0 : rows <= 16 ? 1 : 2;
}

// Values in memory: `width` bytes each at p + i row + j head, i < n and j < heads (strides in bytes, not negative)
struct RowsAt {
    const void *p;
    int64_t n, row, heads, head, width;
};
// Whether two of them share a byte.  What decides is whether Σ k s, over the strides s and the
// differences k of the indexes, comes within the widths of the bases' distance: found from the
// largest stride on, of which only few k leave a distance that the others can make up.  For strides
// so crooked that this takes many steps the answer is yes.
inline bool rows_overlap(const RowsAt &a, const RowsAt &b) {
    typedef __int128 wide;
    struct Term {
        int64_t lo, hi, s;
    } t[4];
    int n = 0;
    auto add = [&](int64_t na, int64_t sa, int64_t nb, int64_t sb) {
        if (sa == sb && sa) {
            if (na > 1 || nb > 1) t[n++] = Term{1 - na, nb - 1, sa};
            return;
        }
        if (na > 1 && sa) t[n++] = Term{1 - na, 0, sa};
        if (nb > 1 && sb) t[n++] = Term{0, nb - 1, sb};
    };
    add(a.n, a.row, b.n, b.row);
    add(a.heads, a.head, b.heads, b.head);
    std::sort(t, t + n, [](const Term &x, const Term &y) { return x.s > y.s; });
    wide least[5], most[5];  // sums of the terms from i on
    least[n] = most[n] = 0;
    for (int i = n - 1; i >= 0; i--) {
        least[i] = least[i + 1] + (wide)t[i].lo * t[i].s;
        most[i] = most[i + 1] + (wide)t[i].hi * t[i].s;
    }
    int steps = 1 << 14;
    auto met = [&](auto &&self, int i, wide d) -> bool {  // b - a is d so far
        if (d + least[i] >= a.width || d + most[i] <= -b.width) return false;
        if (i == n) return true;
        // d + k s + (what the others make) has to come between -b.width and a.width
        auto down = [](wide x, int64_t s) { return x >= 0 ? x / s : -((-x + s - 1) / s); };
        const wide from = -down(-(1 - b.width - d - most[i + 1]), t[i].s), to = down(a.width - 1 - d - least[i + 1], t[i].s);
        const int64_t k1 = to < t[i].hi ? (int64_t)to : t[i].hi;
        for (int64_t k = from > t[i].lo ? (int64_t)from : t[i].lo; k <= k1; k++)
            if (--steps < 0 || self(self, i + 1, d + (wide)k * t[i].s)) return true;
        return false;
    };
    return met(met, 0, (wide)(intptr_t)b.p - (intptr_t)a.p);
}

// Waves of a workgroup of the tile kernel over 8-bit pages, 32 query rows each: 8 where there are so
// many rows, but not of so many blocks that a workgroup for each would make 2^32 threads
inline int tile8_wave_count(int n_rows, int n_seq, int max_new, int G, int n_kv, int hd) {
    return hd <= 128 && (int64_t)max_new * G > 128 && block_count(n_rows, n_seq, G, 256) * n_kv < 1 << 23 ? 8 : 4;
}

// Floats of a partial result of R rows of hd values, and each row's maximum and sum behind them all: whole
// 16-byte vectors, also of odd numbers of rows
RIE_HD int part_floats(int R, int hd) { return (R * (hd + 2) + 3) & ~3; }

// How a launch divides the positions of a block: every split takes C tiles, S at most.
struct SplitPlan {
    int C, S;
};
// wgs: workgroups without splits; tiles: those of the longest block; want: workgroups
// that fill the card; least: tiles that a split is worth
inline SplitPlan split_plan(int64_t wgs, int tiles, int want, int least, int most) {
    SplitPlan p{tiles > 0 ? tiles : 1, 1};
    if (wgs >= want || tiles < 2 * least) return p;
    int64_t s = (want + wgs - 1) / wgs;
    if (s > tiles / least) s = tiles / least;
    if (s > most) s = most;
    if (s < 2) return p;
    p.C = (int)((tiles + s - 1) / s);
    p.S = (tiles + p.C - 1) / p.C;
    return p;
}

// The same for blocks whose time is arithmetic: the number of splits with the least time by
// this estimate, in µs.  wgs workgroups without splits, slots of them at a time; tiles of the
// longest block, tile_us each; a second launch and the partials' way to memory and back
// (part_us per split) where there is more than one.
inline SplitPlan tile_plan(int64_t wgs, int slots, int tiles, double tile_us, double part_us, int most) {
    SplitPlan best{tiles > 0 ? tiles : 1, 1};
    double least = 0;
    for (int s = 1; s <= most && s <= tiles; s++) {
        const int C = (tiles + s - 1) / s;
        if (s > 1 && (tiles + C - 1) / C != s) continue;
        const double full = (double)wgs * s / slots, us = (full > 1 ? full : 1) * C * tile_us + (s > 1 ? 6 + s * part_us : 0);
        if (s == 1 || us < least) {
            least = us;
            best = SplitPlan{C, s};
        }
    }
    return best;
}

}  // namespace rie
