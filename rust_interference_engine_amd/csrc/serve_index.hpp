// serve_index.hpp — where the sequences of a serving batch lie: their rows, positions
// and pages, the blocks of query rows that workgroups take, and the splits of long
// caches.  The starts, lengths and page tables are device memory that the host never
// reads, so everything taken from them is clamped here before it is used as an index;
// the same functions compile for the host, where tests check them.
#pragma once

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
