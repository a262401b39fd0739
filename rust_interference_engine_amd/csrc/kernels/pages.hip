// pages.hip — a pool of pages whose bookkeeping stays on the device: pages given to sequences
// that grow, sequences forked and reordered (the beams of a search), freed, and a pool's pages
// moved together.
//
// refs[p] is the number of table rows that hold page p, and a page with none is free; nothing else
// says so, and a call that needs pages takes the free ones with the lowest numbers.  All choices
// go by row and page number, so that a call's results do not depend on timing: references change
// by integer additions, which may come in any order.
//
// Everything read from device memory is clamped before it is an index.
//
// The planning of a call is one workgroup's: it counts what is needed, finds pages by counting
// through refs 16 to a thread (16384 to a round), and leaves lists in the workspace.  Tables and
// pages are changed by a second and third launch over the whole card.
//
// Bound: for many or large pages HBM, every moved byte read and written once; else the launches
// and what the planning workgroup waits for.  24 searches of 8 beams forked, 44 MB read and written:
// 7.0 us to plan (loads requested before anything waits; state kept in registers over the steps;
// 9.5 before), 10 us for references and copies in one launch (13 in two), 3.9 us for the rows.  A pool
// of 120000 positions compacted, 430 MB read and written: 7 + 90 us (4.8 TB/s).  A reserve looks for
// free pages from number 0 on: 48 new pages of a pool of 10000, 9000 in use, 7.9 us for the call, of
// 300000 that are all but in use 36, of 4 million 430; with nothing to find 6.
#include "../common.hpp"
#include "../device.hpp"
#include "../serve.hpp"

#include <algorithm>

namespace rie {

namespace {

constexpr int PLAN = 1024;       // threads of a planning workgroup
constexpr int PER = 16;          // references of a thread in a round
constexpr int MAX_BUFS = 64;     // buffers of a launch
constexpr int PIECE = 256 * 16;  // bytes that a workgroup copies at a time

typedef int i32x4 __attribute__((ext_vector_type(4)));

// x of the threads before this one, and of all of them; s: 17 words.  All threads call this.
__device__ __forceinline__ int scan(int x, int *s, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int y = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int z = __shfl_up(y, o);
        if (lane >= o) y += z;
    }
    __syncthreads();
    if (lane == 63) s[w] = y;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < PLAN / 64; i++) {
        before += i < w ? s[i] : 0;
        all += s[i];
    }
    total = all;
    return before + y - x;
}

// Bit i: page p0 + i is free.  Behind the last page none is.
__device__ __forceinline__ uint32_t free_of(const int *refs, int p0, int n_pages) {
    uint32_t bits = 0;
    if (p0 + PER <= n_pages) {
        typedef i32x4 i32x4_a4 __attribute__((aligned(4)));
        i32x4 r[PER / 4];
#pragma unroll
        for (int i = 0; i < PER / 4; i++) r[i] = *(const i32x4_a4 *)(refs + p0 + 4 * i);
#pragma unroll
        for (int i = 0; i < PER; i++) bits |= r[i / 4][i % 4] == 0 ? 1u << i : 0;
    } else {
        for (int i = 0; i < PER; i++) bits |= p0 + i < n_pages && refs[p0 + i] == 0 ? 1u << i : 0;
    }
    return bits;
}

// The free pages with the lowest numbers, up to `want`, in order into list; how many there are.  All
// threads call this; bits0: of the first round, which callers read while they find out what they want.
__device__ __forceinline__ uint32_t free_in_round(const PoolView &p, int p0) {
    const int mine = p0 + (int)threadIdx.x * PER;
    return mine < p.n_pages ? free_of(p.refs, mine, p.n_pages) : 0;
}
__device__ __forceinline__ int find_free(const PoolView &p, uint32_t bits0, int want, int *list, int *s) {
    int found = 0;
    for (int p0 = 0; p0 < p.n_pages && found < want; p0 += PLAN * PER) {
        const int mine = p0 + (int)threadIdx.x * PER;
        uint32_t bits = p0 ? free_in_round(p, p0) : bits0;
        int total, at = found + scan(__popc(bits), s, total);
        for (; bits && at < want; bits &= bits - 1) list[at++] = mine + __builtin_ctz(bits);
        found += total;
    }
    return min(found, want);
}

struct Seq {  // of a row: pages that its positions fill, pages that they touch, and pages that it holds
    int full, touched, held;
};
__device__ __forceinline__ Seq seq_of(const PoolView &p, int i) {
    const int page = 1 << p.page_shift, len = (int)min((int64_t)max(p.lens[i], 0), (int64_t)p.cols << p.page_shift);
    return Seq{len >> p.page_shift, (len >> p.page_shift) + ((len & (page - 1)) != 0), min(max(p.held[i], 0), p.cols)};
}

// ---- pages for the positions that sequences have: row by row, the lowest free pages ----
__global__ __launch_bounds__(PLAN) void reserve_kernel(PoolView p, int *list) {
    __shared__ int s[PLAN / 64];
    __shared__ int s_at[POOL_MAX_SEQ + 1];  // pages that the rows before need, up to all there are
    __shared__ unsigned long long s_beyond;  // those that positions behind the columns need: lacking, whatever the pool has
    const uint32_t bits0 = free_in_round(p, 0);
    int64_t want = 0;
    if (threadIdx.x == 0) s_beyond = 0;
    for (int i0 = 0; i0 < p.n_seq; i0 += PLAN) {
        const int i = i0 + (int)threadIdx.x;
        int need = 0, beyond = 0, total;
        if (i < p.n_seq) {
            const Seq q = seq_of(p, i);
            need = max(q.touched - q.held, 0);
            const int len = max(p.lens[i], 0);
            beyond = max((len >> p.page_shift) + ((len & ((1 << p.page_shift) - 1)) != 0) - p.cols, 0);
        }
        const int before = scan(need, s, total);
        if (beyond) atomicAdd(&s_beyond, (unsigned long long)beyond);
        if (i < p.n_seq) s_at[i] = (int)min(want + before, (int64_t)p.n_pages);
        want += total;
    }
    const int most = (int)min(want, (int64_t)p.n_pages);
    if (threadIdx.x == 0) s_at[p.n_seq] = most;
    const int found = find_free(p, bits0, most, list, s);
    __syncthreads();
    for (int j = threadIdx.x; j < found; j += PLAN) {
        int lo = 0, hi = p.n_seq;  // the last row that begins at or before j
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (s_at[mid] <= j) lo = mid;
            else hi = mid;
        }
        const int page = list[j];
        p.table[lo * p.table_stride + seq_of(p, lo).held + (j - s_at[lo])] = page;
        p.refs[page] = 1;
    }
    __syncthreads();
    // a row gets what there is, from its first missing page on
    for (int i = threadIdx.x; i < p.n_seq; i += PLAN) {
        const Seq q = seq_of(p, i);
        const int got = max(min(s_at[i + 1], found) - s_at[i], 0);
        if (got) p.held[i] = q.held + got;
    }
    if (threadIdx.x == 0) p.counts[0] = (int)min(want - found + (int64_t)s_beyond, (int64_t)INT32_MAX);
}

// ---- fork ----
//
// Of those that take a row, its keeper (the row itself, or the first of them) goes on with what that
// row may write next: its partial last page, and the pages held behind it.  Others may hold these
// too, where a row has been cut back into pages that it shared.  Then no row goes on with them: a
// partial page that another row holds is copied for the keeper as well, even where all that hold it
// are in this call (one page more than it would take, but no choice among them), and of the pages
// behind, the keeper gets those before the first that another row holds.
struct Child {  // what becomes of a row
    int src, held, old_held, len;
    int at, fresh;  // place of the source's partial page where the row gets a copy of it (−1: none), and that copy (−1: the pool has none)
};
struct Lists {
    int n;  // pages to copy
    int pad[3];
};

// Of the lanes' rows r, the first of their pages [from, to) that more than one row holds, or to; `on`: the
// lane has a row.  A wave's lanes share its rows evenly, each with AHEAD loads on their way (192 rows with
// 37 pages ahead: 18 us for the call, a row after the other with all lanes 38, none ahead 11).
// place: 64 words of the wave's own.
__device__ __forceinline__ int first_shared(const PoolView &p, bool on, int r, int from, int to, int *place) {
    constexpr int AHEAD = 8;
    const int lane = threadIdx.x & 63;
    const uint64_t rows = __ballot(on);
    if (!rows) return to;
    const int n = (int)__popcll(rows), rank = (int)__popcll(rows & ((1ull << lane) - 1));
    int per = 64;  // lanes to a row
    while (64 / per < n) per /= 2;
    if (on) place[rank] = lane;
    wave_sync();
    const int mine = lane / per, of = place[min(mine, n - 1)];
    wave_sync();
    const int row = __shfl(r, of), end = __shfl(to, of), begin = __shfl(from, of);
    int first = end;
    if (mine < n) {
        const int *t = p.table + row * p.table_stride;
        for (int k0 = begin + lane % per; k0 < first; k0 += AHEAD * per) {
            int page[AHEAD];
            bool shared[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; a++) page[a] = k0 + a * per < end ? t[k0 + a * per] : -1;
#pragma unroll
            for (int a = 0; a < AHEAD; a++) shared[a] = (unsigned)page[a] < (unsigned)p.n_pages && p.refs[page[a]] > 1;
#pragma unroll
            for (int a = AHEAD - 1; a >= 0; a--) first = shared[a] ? k0 + a * per : first;
        }
    }
    for (int o = per / 2; o; o >>= 1) first = min(first, __shfl_xor(first, o));
    return __shfl(first, rank * per & 63);
}

__global__ __launch_bounds__(PLAN) void fork_plan_kernel(PoolView p, const int *src, Lists *lists, Child *child, int *children, int *kept, int *from, int *to, int *list) {
    __shared__ int s_count[POOL_MAX_SEQ], s_heir[POOL_MAX_SEQ];  // children of a row, and which of them inherits its partial page
    __shared__ int s[PLAN / 64], s_place[PLAN / 64][64];
    constexpr int ROUNDS = POOL_MAX_SEQ / PLAN;
    const uint32_t bits0 = free_in_round(p, 0);
    int r[ROUNDS];
#pragma unroll
    for (int u = 0; u < ROUNDS; u++) {
        const int i = u * PLAN + (int)threadIdx.x;
        r[u] = i < p.n_seq ? src[i] : -1;
        r[u] = (unsigned)r[u] < (unsigned)p.n_seq ? r[u] : -1;
        s_count[i] = 0;
        s_heir[i] = INT32_MAX;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; u++) {
        const int i = u * PLAN + (int)threadIdx.x;
        if (r[u] < 0) continue;
        atomicAdd(s_count + r[u], 1);
        atomicMin(s_heir + r[u], r[u] == i ? -1 : i);  // the row itself, or its first child
    }
    __syncthreads();
    int want = 0, copies = 0;
    Child c[ROUNDS];
    int old[ROUNDS], mine[ROUNDS];  // the source's partial page; which of the new ones goes in its place
#pragma unroll
    for (int u = 0; u < ROUNDS; u++) {
        const int i = u * PLAN + (int)threadIdx.x;
        c[u] = Child{r[u], 0, 0, 0, -1, -1};
        old[u] = -1;
        int ahead = -1;  // of a keeper with pages behind its last position, the first of them
        bool keeps = false, shared = false;
        if (u * PLAN >= p.n_seq) continue;
        if (i < p.n_seq) {
            children[i] = s_count[i];
            c[u].old_held = seq_of(p, i).held;
        }
        if (r[u] >= 0) {
            const Seq q = seq_of(p, r[u]);
            const bool keep = r[u] == i || s_heir[r[u]] == i;  // it takes the source's pages as they are
            c[u].held = keep ? q.held : min(q.touched, q.held);
            c[u].len = p.lens[r[u]];
            if (q.touched > q.full && q.held > q.full) {
                old[u] = p.table[r[u] * p.table_stride + q.full];
                shared = keep && (unsigned)old[u] < (unsigned)p.n_pages && p.refs[old[u]] > 1;
                if (!keep || shared) c[u].at = q.full;
            }
            keeps = keep;
            ahead = keep && q.held > q.touched ? q.touched : -1;
        }
        const int first = first_shared(p, ahead >= 0, r[u], ahead, c[u].held, s_place[threadIdx.x >> 6]);
        if (ahead >= 0) c[u].held = first;
        if (keeps) kept[r[u]] = shared ? ~c[u].held : c[u].held;
        int total;
        mine[u] = want + scan(c[u].at >= 0, s, total);
        want += total;
    }
    const int found = find_free(p, bits0, want, list, s);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < ROUNDS; u++) {
        const int i = u * PLAN + (int)threadIdx.x;
        if (u * PLAN >= p.n_seq) break;
        if (c[u].at >= 0 && mine[u] < found) {
            c[u].fresh = list[mine[u]];
            p.refs[c[u].fresh] = 1;
        }
        const bool copy = c[u].fresh >= 0 && (unsigned)old[u] < (unsigned)p.n_pages;
        int total;
        const int k = copies + scan(copy, s, total);
        if (copy) {
            from[k] = old[u];
            to[k] = c[u].fresh;
        }
        copies += total;
        if (i < p.n_seq) child[i] = c[u];
    }
    if (threadIdx.x == 0) {
        lists->n = copies;
        p.counts[0] = want - found;
    }
}

struct Bufs {
    PageBuf b[MAX_BUFS];
    int first[MAX_BUFS + 1];  // pieces of a page before buffer i
    int n;
};

// Copies pages: workgroup g of n takes every n-th piece of every page in the lists
__device__ void copy_pages(const Bufs &bufs, int g, int n, const int *from, const int *to, int n_copies, int n_pages) {
    const int per = bufs.first[bufs.n];
    for (int64_t i = g; i < (int64_t)n_copies * per; i += n) {
        const int j = (int)(i / per), piece = (int)(i - (int64_t)j * per);
        int b = 0;
        while (piece >= bufs.first[b + 1]) b++;
        const PageBuf &buf = bufs.b[b];
        const int f = from[j], t = to[j];
        if ((unsigned)f >= (unsigned)n_pages || (unsigned)t >= (unsigned)n_pages) continue;
        const int64_t at = (int64_t)(piece - bufs.first[b]) * PIECE;
        const uint8_t *x = buf.base + f * buf.stride + at;
        uint8_t *y = buf.base + t * buf.stride + at;
        const int len = (int)min((int64_t)PIECE, buf.bytes - at);
        if ((((uintptr_t)x | (uintptr_t)y | (unsigned)len) & 15) == 0) {
            const int o = threadIdx.x * 16;
            if (o < len) *(u32x4 *)(y + o) = *(const u32x4 *)(x + o);
        } else {
            for (int o = threadIdx.x * 4; o < len; o += 256 * 4) *(uint32_t *)(y + o) = *(const uint32_t *)(x + o);
        }
    }
}

// The old rows' references, and the rows that others go on from into `rows`, a workgroup each; and the copies
__global__ __launch_bounds__(256) void fork_refs_kernel(PoolView p, Bufs bufs, int row_wgs, const Lists *lists, const int *src, const int *children, const int *kept, const int *from, const int *to, int *rows) {
    if ((int)blockIdx.x >= row_wgs) {
        copy_pages(bufs, blockIdx.x - row_wgs, gridDim.x - row_wgs, from, to, lists->n, p.n_pages);
        return;
    }
    const int r = blockIdx.x, n = children[r];
    const bool stays = (unsigned)src[r] < (unsigned)p.n_seq && src[r] == r;
    const Seq q = seq_of(p, r);
    // pages before this one stay with the keeper; negative: ~ it, and the partial one does not
    const int k = n ? kept[r] : 0, stay = k < 0 ? ~k : k;
    if (n == 1 && stays && k == q.held) return;
    const int *t = p.table + r * p.table_stride;
    for (int c = threadIdx.x; c < q.held; c += 256) {
        const int page = t[c], change = c < q.full ? n - 1 : c >= stay || (k < 0 && c == q.full) ? -1 : 0;
        if (n) rows[(int64_t)r * p.cols + c] = page;
        if (change && (unsigned)page < (unsigned)p.n_pages) atomicAdd(p.refs + page, change);
    }
}

// The new rows, a workgroup each
__global__ __launch_bounds__(256) void fork_rows_kernel(PoolView p, const Child *child, const int *rows) {
    const int i = blockIdx.x;
    const Child c = child[i];
    if (c.src == i && c.at < 0 && c.held == c.old_held) return;  // and keeps its pages
    int *t = p.table + i * p.table_stride;
    const int *r = rows + (int64_t)max(c.src, 0) * p.cols;
    for (int k = threadIdx.x; k < max(c.held, c.old_held); k += 256) t[k] = k >= c.held ? -1 : k == c.at ? c.fresh : r[k];
    if (threadIdx.x == 0) {
        p.lens[i] = c.len;
        p.held[i] = c.held;
    }
}

// ---- free: a workgroup per row ----
__global__ __launch_bounds__(256) void free_kernel(PoolView p, const int *which) {
    const int i = blockIdx.x;
    if (!which[i]) return;
    const int held = seq_of(p, i).held;
    int *t = p.table + i * p.table_stride;
    for (int c = threadIdx.x; c < held; c += 256) {
        const int page = t[c];
        if ((unsigned)page < (unsigned)p.n_pages) atomicSub(p.refs + page, 1);
        t[c] = -1;
    }
    __syncthreads();
    if (threadIdx.x == 0) p.held[i] = p.lens[i] = 0;
}

// ---- compact: of n pages in use, those from number n on go to the free ones below it, in order ----
__global__ __launch_bounds__(PLAN) void compact_plan_kernel(PoolView p, Lists *lists, int *from, int *to, int *goes) {
    __shared__ int s[PLAN / 64];
    int used = 0;
    for (int p0 = 0; p0 < p.n_pages; p0 += PLAN * PER) {
        const int mine = p0 + (int)threadIdx.x * PER, n = min(max(p.n_pages - mine, 0), PER);
        int total;
        scan(n ? n - __popc(free_of(p.refs, mine, p.n_pages)) : 0, s, total);
        used += total;
    }
    int n_from = 0, n_to = 0;
    for (int p0 = 0; p0 < p.n_pages; p0 += PLAN * PER) {
        const int mine = p0 + (int)threadIdx.x * PER, n = min(max(p.n_pages - mine, 0), PER);
        const uint32_t all = (1u << n) - 1, low = mine >= used ? 0 : used - mine >= PER ? all : all & ((1u << (used - mine)) - 1);
        const uint32_t f = n ? free_of(p.refs, mine, p.n_pages) : 0;
        uint32_t a = ~f & all & ~low, b = f & low;
        for (uint32_t c = f & ~low; c; c &= c - 1) goes[mine + __builtin_ctz(c)] = mine + __builtin_ctz(c);
        int total;
        int at = n_from + scan(__popc(a), s, total);
        n_from += total;
        for (; a; a &= a - 1) from[at++] = mine + __builtin_ctz(a);
        at = n_to + scan(__popc(b), s, total);
        n_to += total;
        for (; b; b &= b - 1) to[at++] = mine + __builtin_ctz(b);
    }
    __syncthreads();
    const int n = min(n_from, n_to);  // the same
    for (int j = threadIdx.x; j < n; j += PLAN) {
        const int f = from[j], t = to[j];
        goes[f] = t;
        p.refs[t] = p.refs[f];
        p.refs[f] = 0;
    }
    if (threadIdx.x == 0) {
        lists->n = n;
        p.counts[1] = used;
    }
}

__global__ __launch_bounds__(256) void compact_rows_kernel(PoolView p, Bufs bufs, int row_wgs, const Lists *lists, const int *from, const int *to, const int *goes) {
    if ((int)blockIdx.x >= row_wgs) {
        copy_pages(bufs, blockIdx.x - row_wgs, gridDim.x - row_wgs, from, to, lists->n, p.n_pages);
        return;
    }
    const int i = blockIdx.x, used = p.counts[1];
    const Seq q = seq_of(p, i);
    int *t = p.table + i * p.table_stride;
    for (int c = threadIdx.x; c < q.held; c += 256) {
        const int page = t[c];
        if (page >= used && page < p.n_pages) t[c] = goes[page];
    }
}

__global__ __launch_bounds__(256) void copy_kernel(Bufs bufs, const int *from, const int *to, int n, int n_pages) {
    copy_pages(bufs, blockIdx.x, gridDim.x, from, to, n, n_pages);
}

Bufs bufs_of(const PageBuf *b, int n) {
    Bufs x;
    x.n = n;
    x.first[0] = 0;
    for (int i = 0; i < n; i++) {
        x.b[i] = b[i];
        x.first[i + 1] = x.first[i] + (int)((b[i].bytes + PIECE - 1) / PIECE);
    }
    return x;
}

constexpr int COPY_WGS = 2048;  // 8 to a CU

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace

size_t page_reserve_ws(const PoolView &p) { return up16((size_t)p.n_pages * sizeof(int)); }

size_t page_fork_ws(const PoolView &p) {
    return sizeof(Lists) + up16(p.n_seq * sizeof(Child)) + 5 * up16(p.n_seq * sizeof(int)) + up16((size_t)p.n_seq * p.cols * sizeof(int));
}

size_t page_compact_ws(const PoolView &p) { return sizeof(Lists) + 3 * up16((size_t)p.n_pages * sizeof(int)); }

void launch_page_reserve(const PoolView &p, void *ws, hipStream_t st) { reserve_kernel<<<1, PLAN, 0, st>>>(p, (int *)ws); }

void launch_page_fork(const PoolView &p, const int *src, const PageBuf *bufs, int n_bufs, void *ws, hipStream_t st) {
    uint8_t *w = (uint8_t *)ws;
    Lists *lists = (Lists *)w;
    w += sizeof(Lists);
    Child *child = (Child *)w;
    w += up16(p.n_seq * sizeof(Child));
    int *ints[5];  // children, pages that their keepers keep, pages copied from and to, free ones
    for (int *&x : ints) {
        x = (int *)w;
        w += up16(p.n_seq * sizeof(int));
    }
    int *rows = (int *)w;
    fork_plan_kernel<<<1, PLAN, 0, st>>>(p, src, lists, child, ints[0], ints[1], ints[2], ints[3], ints[4]);
    int done = 0;
    do {
        const int n = std::min(n_bufs - done, MAX_BUFS), row_wgs = done ? 0 : p.n_seq;
        fork_refs_kernel<<<row_wgs + (n ? COPY_WGS : 0), 256, 0, st>>>(p, bufs_of(bufs + done, n), row_wgs, lists, src, ints[0], ints[1], ints[2], ints[3], rows);
        done += n;
    } while (done < n_bufs);
    fork_rows_kernel<<<p.n_seq, 256, 0, st>>>(p, child, rows);
}

void launch_page_free(const PoolView &p, const int *which, hipStream_t st) { free_kernel<<<p.n_seq, 256, 0, st>>>(p, which); }

void launch_page_compact(const PoolView &p, const PageBuf *bufs, int n_bufs, void *ws, hipStream_t st) {
    uint8_t *w = (uint8_t *)ws;
    Lists *lists = (Lists *)w;
    w += sizeof(Lists);
    int *ints[3];  // pages moved from and to; where a page goes
    for (int *&x : ints) {
        x = (int *)w;
        w += up16((size_t)p.n_pages * sizeof(int));
    }
    compact_plan_kernel<<<1, PLAN, 0, st>>>(p, lists, ints[0], ints[1], ints[2]);
    int done = 0;
    do {
        const int n = std::min(n_bufs - done, MAX_BUFS), row_wgs = done ? 0 : p.n_seq;
        compact_rows_kernel<<<row_wgs + (n ? COPY_WGS : 0), 256, 0, st>>>(p, bufs_of(bufs + done, n), row_wgs, lists, ints[0], ints[1], ints[2]);
        done += n;
    } while (done < n_bufs);
}

void launch_page_copy(const PageBuf *bufs, int n_bufs, int n_pages, const int *src, const int *dst, int n, hipStream_t st) {
    for (int done = 0; done < n_bufs;) {
        const int m = std::min(n_bufs - done, MAX_BUFS);
        copy_kernel<<<COPY_WGS, 256, 0, st>>>(bufs_of(bufs + done, m), src, dst, n, n_pages);
        done += m;
    }
}

}  // namespace rie
