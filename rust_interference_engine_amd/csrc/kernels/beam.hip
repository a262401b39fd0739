// beam.hip — beam search's selection.  Of the candidates (beam b, token t) of a request, with
//
//   score_b + x_bt − m_b − ln Σ_t e^(x_bt − m_b),  m_b = max x_b,
//
// the best n_out in order, the lowest beam, then the lowest token first among equals.
//
// The logits are read once.  beam_part_kernel takes groups of consecutive logits, a wave per run
// of groups, with the run's maximum and sum, and keeps every group's maximum.  beam_row_kernel
// joins a row's runs and finds its own best n_out tokens: they lie in the n_out groups with the
// largest maxima (by value, then by place: a group ahead of theirs holds a logit ahead of them),
// so only those are read again.  The workgroup of a request that is done last merges its rows.
//
// Beams are compared by sums in f64: in f32 the candidates of two beams would be equal to the last
// bit too often, and their order that of the roundings.  ln Σ is f64 of an f32 sum
// (off by under 2^-22 of it in all rows measured; of 192 of 128256 logits by 3 · 2^-24).
//
// Bound: HBM, rows · V values, for the first launch, latency for the second.  192 rows of 128256
// bf16 logits, 16 wanted: 12.1 us (4.1 TB/s) + 14.7 us, of which 2.5 us wait for the groups'
// maxima, 4 us are the groups' loads and their candidates, 3.4 us the merge; 4 rows of 151936 f32
// logits, 4 wanted: 3.3 + 8.3 us.  The merge in a launch of its own: 5.5 us more.
#include "../common.hpp"
#include "../device.hpp"
#include "../serve.hpp"

#include <algorithm>
#include <cfloat>

namespace rie {

namespace {

constexpr int R = 16, STEP = 64 * R;  // logits of a lane and of a wave at a time
constexpr int MAX_GROUPS = 512;       // of a row: groups of 1024, 2048 or 4096 logits
constexpr float FAST_M = 1 << 20;     // size of a maximum below which an exponent is one fma

typedef f32x4 f32x4_a4 __attribute__((aligned(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef u16x8 u16x8_a2 __attribute__((aligned(2)));

template <int TY>
__device__ __forceinline__ float logit(const void *x, int i) {
    if constexpr (TY == T_F32) return ((const float *)x)[i];
    const uint16_t b = ((const uint16_t *)x)[i];
    return TY == T_BF16 ? __uint_as_float((uint32_t)b << 16) : h2f(b);
}

// Place of a lane's value j in its wave's 1024: runs of 16 bytes, the lanes' side by side
template <int TY>
__device__ __forceinline__ int place(int lane, int j) {
    constexpr int N = TY == T_F32 ? 4 : 8;
    return j / N * (64 * N) + lane * N + j % N;
}

// The lane's values of the 1024 from element e0 of the row on, −inf behind its end.  The same
// elements whatever the row's alignment, so that rows of equal logits have equal sums.
template <int TY>
__device__ __forceinline__ void load_step(const void *x, int e0, int V, int lane, float (&v)[R]) {
    if (e0 + STEP <= V) {
        if constexpr (TY == T_F32) {
            f32x4 a[R / 4];
#pragma unroll
            for (int i = 0; i < R / 4; i++) a[i] = *(const f32x4_a4 *)((const float *)x + e0 + place<TY>(lane, 4 * i));
#pragma unroll
            for (int j = 0; j < R; j++) v[j] = a[j / 4][j % 4];
        } else {
            u16x8 a[R / 8];
#pragma unroll
            for (int i = 0; i < R / 8; i++) a[i] = *(const u16x8_a2 *)((const uint16_t *)x + e0 + place<TY>(lane, 8 * i));
#pragma unroll
            for (int j = 0; j < R; j++) v[j] = TY == T_BF16 ? __uint_as_float((uint32_t)a[j / 8][j % 8] << 16) : h2f(a[j / 8][j % 8]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; j++) {
            const int e = e0 + place<TY>(lane, j);
            v[j] = e < V ? logit<TY>(x, e) : -INFINITY;
        }
    }
}

struct Run {  // maximum and Σ e^(x − m); s is NaN where there is a NaN or +inf
    float m, s;
};
__device__ __forceinline__ Run join(const Run &a, const Run &b) {
    const float m = fmaxf(a.m, b.m);
    return Run{m, a.s * exp2_hw((a.m - m) * LOG2E_F) + b.s * exp2_hw((b.m - m) * LOG2E_F)};
}

template <int TY>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a, int n_groups, int steps, int per, int n_parts, float *gmax, Run *runs, int *arrived) {
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = id / n_parts, part = id - row * n_parts;
    if (row >= a.n * a.n_beams) return;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int g0 = part * per, g1 = min(g0 + per, n_groups), u1 = min(g1 * steps, (a.V + STEP - 1) / STEP);
    // M is the wave's maximum so far, s the lane's sum.  fs is the sum of the steps since M moved, in
    // log2 units against −c, where c = −M · log2 e rounded: one fma forms an exponent, and the rounding
    // of c, r = M · log2 e + c exactly, is taken out of the sum when M moves or at the end (it holds
    // 2^r times its own).  From |M| = 2^20 on, r could pass 2^-4: those take a subtraction.
    float M = -FLT_MAX, s = 0, fs = 0, c = 0;
    bool plain = true;
    auto settle = [&] {
        s = fmaf(fs, plain ? 1.0f : exp2_hw(-fmaf(M, LOG2E_F, c)), s);
        fs = 0;
    };
    float v[R], nx[R], g = -INFINITY;
    load_step<TY>(x, g0 * steps * STEP, a.V, lane, v);
    for (int u = g0 * steps; u < u1; u++) {
        if (u + 1 < u1) load_step<TY>(x, (u + 1) * STEP, a.V, lane, nx);
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < R - 1; j += 2) mx = fmaxf(fmaxf(mx, v[j]), v[j + 1]);
        mx = fmaxf(mx, v[R - 1]);
        mx = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(xmax_f<64>(mx))));
        mx = mx == mx ? mx : -INFINITY;  // nothing but NaN
        g = fmaxf(g, mx);
        if ((u + 1) % steps == 0 || u + 1 == u1) {
            if (lane == 0) gmax[(int64_t)row * n_groups + u / steps] = g;
            g = -INFINITY;
        }
        if (mx > M) {
            settle();
            s *= exp2_hw((M - mx) * LOG2E_F);
            M = mx;
            plain = !(fabsf(M) < FAST_M);
            c = plain ? 0.0f : -(M * LOG2E_F);
        }
        float e[R];
        if (!plain) {
#pragma unroll
            for (int j = 0; j < R; j++) e[j] = exp2_hw(fmaf(v[j], LOG2E_F, c));
        } else {
#pragma unroll
            for (int j = 0; j < R; j++) e[j] = exp2_hw((v[j] - M) * LOG2E_F);
        }
#pragma unroll
        for (int o = R / 2; o; o >>= 1)
#pragma unroll
            for (int j = 0; j < o; j++) e[j] += e[j + o];
        fs += e[0];
#pragma unroll
        for (int j = 0; j < R; j++) v[j] = nx[j];
    }
    settle();
    s = xsum_f<64>(s);
    if (lane == 0) runs[(int64_t)row * n_parts + part] = Run{M, s};
    if (part == 0 && lane == 0 && row % a.n_beams == 0) arrived[row / a.n_beams] = 0;
}

constexpr int CAND = 1024;  // logits that are ranked at once

// Stores and loads that other XCDs' workgroups see, and are seen by
__device__ __forceinline__ void put(double *p, double v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put(int *p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Numbers in the order of the values, equal ones' lower index first
__device__ __forceinline__ uint64_t ordered(float v, int index) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ int64_t ordered(double v) {
    const int64_t b = __double_as_longlong(v + 0.0);
    return b < 0 ? b ^ INT64_MAX : b;
}

// A row's best k = min(n_out, V) tokens in order, with their sums: key[row][k], id[row][k].
//
// A few thousand cycles of one workgroup, so what counts is what waits for what: all loads are
// requested before anything is waited for; each wave finds the groups for itself, without a
// barrier; barriers are LDS's only, so that loads pass them; and ranks are counted with one
// comparison of whole numbers and an addition with its carry (masks of two comparisons joined in
// scalar registers took 75 cycles a candidate).
template <int TY>
__device__ void best_of_row(const BeamArgs &a, int row, int n_groups, int steps, int n_parts, const float *gmax, const Run *runs, double *key, int *id) {
    __shared__ Run s_run[4];
    __shared__ uint64_t s_cand[CAND];
    __shared__ int s_group[4][BEAM_MAX_OUT];
    __shared__ int s_n[4];  // candidates of each wave, in its quarter of the list
    __shared__ float s_mine[256];
    __shared__ float s_thr;
    constexpr int PART = CAND / 4;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t before = (1ull << lane) - 1;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int k = min(a.n_out, a.V), kg = min(k, n_groups);
    key += (int64_t)row * k;
    id += (int64_t)row * k;
    constexpr int NG = MAX_GROUPS / 64;
    float own[NG];
#pragma unroll
    for (int i = 0; i < NG; i++) own[i] = lane + 64 * i < n_groups ? fmaxf(gmax[(int64_t)row * n_groups + lane + 64 * i], -INFINITY) : NAN;
    Run p{-FLT_MAX, 0};
    for (int i = tid; i < n_parts; i += 256) p = join(p, runs[(int64_t)row * n_parts + i]);
    const float score = a.scores[row];
    const int finished = a.finished ? a.finished[row] : 0;

    // T, from which on a group is taken: at most the kg-th largest maximum, so that at least kg are.
    // That of the lanes' own largest maxima, found by counting; with more to come, or too many equal
    // ones, the kg-th largest maximum itself, one value after the other, the largest first (16 of
    // them 2.4 us, the counts 0.5).  NaN: no group.
    float T = -INFINITY;
    int sel = MAX_GROUPS;
    if (kg <= 64) {
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < NG; i++) most = fmaxf(most, own[i]);
        int ahead = 0;
#pragma unroll
        for (int j = 0; j < 64; j++) ahead += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(most), j)) > most;
        T = -xmax_f<64>(ahead < kg ? -most : -INFINITY);
        T = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(T)));
        sel = 0;
#pragma unroll
        for (int i = 0; i < NG; i++) {
            if (64 * i >= n_groups) break;
            sel += (int)__popcll(__ballot(own[i] >= T));
        }
    }
    if (sel > BEAM_MAX_OUT) {
        sel = kg;
        T = INFINITY;
        for (int n = 0; n < kg;) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                if (64 * i >= n_groups) break;
                m = n == 0 || own[i] < T ? fmaxf(m, own[i]) : m;
            }
            T = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(xmax_f<64>(m))));
#pragma unroll
            for (int i = 0; i < NG; i++) {
                if (64 * i >= n_groups) break;
                n += (int)__popcll(__ballot(own[i] == T));
            }
        }
    }
    // the groups above it, and of those that equal it the first
    int n_above = 0, n_equal = 0;
#pragma unroll
    for (int i = 0; i < NG; i++) {
        if (64 * i >= n_groups) break;
        n_above += (int)__popcll(__ballot(own[i] > T));
    }
    int at = 0;
#pragma unroll
    for (int i = 0; i < NG; i++) {
        if (64 * i >= n_groups) break;
        const uint64_t above = __ballot(own[i] > T), equal = __ballot(own[i] == T);
        const int pa = at + (int)__popcll(above & before), pe = n_above + n_equal + (int)__popcll(equal & before);
        if (own[i] > T) s_group[w][pa] = i * 64 + lane;
        else if (own[i] == T && pe < sel) s_group[w][pe] = i * 64 + lane;
        at += (int)__popcll(above);
        n_equal += (int)__popcll(equal);
    }
    wave_sync();
    // The logits of these from T on may be among the first k.  More than fit (few groups, or equal
    // logits): those from the k-th largest of the threads' own maxima on.
    constexpr int AT_ONCE = 4;  // steps that a wave reads at once
    float v[AT_ONCE][R];
    const int n_steps = sel * steps;
    auto first_of = [&](int u) { return (s_group[w][u / steps] * steps + u % steps) * STEP; };
    auto read = [&](int u0) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < AT_ONCE; q++)
            if (u0 + 4 * q < n_steps) load_step<TY>(x, first_of(u0 + 4 * q), a.V, lane, v[q]);
    };
    read(w);
    // the row's sum meanwhile
#pragma unroll
    for (int o = 32; o; o >>= 1) p = join(p, Run{__shfl_xor(p.m, o), __shfl_xor(p.s, o)});
    if (lane == 0) s_run[w] = p;
    lds_barrier();
    p = join(join(s_run[0], s_run[1]), join(s_run[2], s_run[3]));
    if (finished) {  // goes on as it is
        for (int i = tid; i < k; i += 256) {
            put(key + i, i == 0 && fabsf(score) <= FLT_MAX ? (double)score : -INFINITY);
            put(id + i, a.pad);
        }
        return;
    }
    if (!(p.s > 0) || !(p.m <= FLT_MAX) || !(fabsf(score) <= FLT_MAX)) {  // offers nothing
        for (int i = tid; i < k; i += 256) {
            put(key + i, -INFINITY);
            put(id + i, i);
        }
        return;
    }
    const double log_s = log((double)p.s);
    float thr = kg < k ? -FLT_MAX : fmaxf(T, -FLT_MAX), mine = -INFINITY;  // not those of −inf, nor what lies behind the row's end
    int n = 0;
    for (int attempt = 0; attempt < 2; attempt++) {
        int found = 0;
        for (int u0 = w; u0 < n_steps; u0 += 4 * AT_ONCE) {
            if (attempt || u0 > w) read(u0);
            uint64_t hits = 0;
#pragma unroll
            for (int q = 0; q < AT_ONCE; q++) {
                uint32_t h = 0;
                if (u0 + 4 * q < n_steps) {
#pragma unroll
                    for (int j = 0; j < R; j++) {
                        mine = fmaxf(mine, v[q][j]);
                        h |= v[q][j] >= thr ? 1u << j : 0;
                    }
                }
                hits |= (uint64_t)h << (16 * q);
            }
            while (__any(hits != 0)) {
                const uint64_t some = __ballot(hits != 0);
                const int c = found + (int)__popcll(some & before);
                if (hits) {
                    const int b = __builtin_ctzll(hits);
                    if (c < PART) s_cand[w * PART + c] = (uint32_t)(first_of(u0 + b / 16 * 4) + place<TY>(lane, b % 16));
                    hits &= hits - 1;
                }
                found += (int)__popcll(some);
            }
        }
        if (lane == 0) s_n[w] = found;
        lds_barrier();
        n = s_n[0] + s_n[1] + s_n[2] + s_n[3];
        if (max(max(s_n[0], s_n[1]), max(s_n[2], s_n[3])) > PART) n = CAND + 1;
        if (n <= CAND || attempt) break;
        s_mine[tid] = mine;
        lds_barrier();
        int ahead = 0;
        for (int j = 0; j < 256; j++) ahead += (s_mine[j] > mine) | ((s_mine[j] == mine) & (j < tid));
        if (ahead == k - 1) s_thr = mine;
        lds_barrier();
        thr = fmaxf(s_thr, -FLT_MAX);
    }
    if (n <= CAND) {
        // candidates by number: the i-th lies in the wave's quarter that holds it
        auto slot = [&](int i) {
            int g = 0;
            while (i >= s_n[g]) i -= s_n[g++];
            return g * PART + i;
        };
        float mine_v[CAND / 256];
        int mine_s[CAND / 256], mine_e[CAND / 256];
#pragma unroll
        for (int u = 0; u < CAND / 256; u++) {
            const int i = tid + 256 * u;
            mine_s[u] = mine_e[u] = 0;
            if (i >= n) continue;
            mine_s[u] = slot(i);
            mine_e[u] = (int)(uint32_t)s_cand[mine_s[u]];
            mine_v[u] = logit<TY>(x, mine_e[u]);
        }
#pragma unroll
        for (int u = 0; u < CAND / 256; u++) {
            if (tid + 256 * u >= n) continue;
            s_cand[mine_s[u]] = ordered(mine_v[u], mine_e[u]);
        }
        lds_barrier();
#pragma unroll
        for (int u = 0; u < CAND / 256; u++) {
            if (256 * u >= n) break;
            const bool on = tid + 256 * u < n;
            const uint64_t me = on ? s_cand[mine_s[u]] : 0;
            int ahead = 0;
            for (int g = 0; g < 4; g++) {
                const int m = s_n[g];
#pragma unroll 4
                for (int j = 0; j < m; j++) ahead += s_cand[g * PART + j] > me;
            }
            if (on && ahead < k) {
                put(key + ahead, (double)score + (((double)mine_v[u] - (double)p.m) - log_s));
                put(id + ahead, mine_e[u]);
            }
        }
        if (n >= k) return;
        // the first of the logits of −inf: under k of the row's are none, so they lie in its first 2 k
        const bool out = tid < a.V && logit<TY>(x, tid) == -INFINITY;
        const uint64_t m = __ballot(out);
        lds_barrier();
        if (lane == 0) s_n[w] = (int)__popcll(m);
        lds_barrier();
        int place_of = n + (int)__popcll(m & before);
        for (int i = 0; i < w; i++) place_of += s_n[i];
        if (out && place_of < k) {
            put(key + place_of, -INFINITY);
            put(id + place_of, tid);
        }
        return;
    }
    // more equal logits than fit: the next one of all of the groups' logits, k times
    float last = INFINITY;
    int last_e = -1;
    for (int r = 0; r < k; r++) {
        float bv = -INFINITY;
        int be = INT32_MAX;
        for (int i = tid; i < sel * steps * STEP; i += 256) {
            const int e = s_group[w][i / (steps * STEP)] * steps * STEP + i % (steps * STEP);
            if (e >= a.V) continue;
            const float v = logit<TY>(x, e);
            if ((v < last || (v == last && e > last_e)) && (v > bv || (v == bv && e < be))) {
                bv = v;
                be = e;
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            const float v = __shfl_xor(bv, o);
            const int e = __shfl_xor(be, o);
            if (v > bv || (v == bv && e < be)) {
                bv = v;
                be = e;
            }
        }
        __syncthreads();
        if (lane == 0) {
            s_mine[w] = bv;
            s_n[w] = be;
        }
        __syncthreads();
        for (int i = 0; i < 4; i++)
            if (s_mine[i] > bv || (s_mine[i] == bv && s_n[i] < be)) {
                bv = s_mine[i];
                be = s_n[i];
            }
        last = bv;
        last_e = be;
        if (tid == 0) {
            put(key + r, (double)score + (((double)bv - (double)p.m) - log_s));
            put(id + r, be);
        }
    }
}

// The rows of a request merged.  Each row's candidates are in order, so what is ahead of one in
// another row is found by halving.
__device__ void merge_rows(const BeamArgs &a, int req, const double *key, const int *id, double *s_key) {
    const int W = a.n_beams, k = min(a.n_out, a.V), n = W * k;
    key += (int64_t)req * n;
    id += (int64_t)req * n;
    auto chosen = [&](int i, int ahead, double v, int token) {
        if (ahead >= a.n_out) return;
        const int64_t o = (int64_t)req * a.n_out + ahead;
        a.next[o] = (float)v;
        a.parents[o] = req * W + i / k;
        a.tokens[o] = token;
    };
    constexpr int FEW = 256;  // that are ranked by counting (24 requests of 8 beams and 16 candidates: by halving 4.7 us)
    if (n <= FEW) {
        __shared__ int s_ahead[FEW], s_at[BEAM_MAX_OUT], s_tie;
        int64_t *s_ord = (int64_t *)s_key;
        const int i = threadIdx.x, at = i < n ? i : 0;
        const double v = __hip_atomic_load(key + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int token = __hip_atomic_load(id + at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        s_ahead[i] = 0;
        if (i < n) s_ord[i] = ordered(v);
        if (i == 0) s_tie = 0;
        lds_barrier();
        // as many threads to a candidate as there are, each with a share of the others
        const int per = n <= FEW / 4 ? 4 : n <= FEW / 2 ? 2 : 1, c = i / per, share = (n + per - 1) / per, from = i % per * share, to = min(from + share, n);
        if (c < n) {
            const int64_t me = s_ord[c];
            int ahead = 0;
#pragma unroll 4
            for (int j = from; j < to; j++) ahead += s_ord[j] > me;
            atomicAdd(s_ahead + c, ahead);
        }
        lds_barrier();
        // equal ones have one place: their order is that of the candidates
        int ahead = i < n ? s_ahead[i] : a.n_out;
        if (ahead < a.n_out) s_at[ahead] = i;
        lds_barrier();
        if (ahead < a.n_out && s_at[ahead] != i) s_tie = 1;
        lds_barrier();
        if (s_tie && i < n) {
            const int64_t me = s_ord[i];
            for (int j = 0; j < i; j++) ahead += s_ord[j] == me;
        }
        if (i < n) chosen(i, ahead, v, token);
        return;
    }
    for (int i = threadIdx.x; i < n; i += 256) s_key[i] = __hip_atomic_load(key + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const int b = i / k;
        const double v = s_key[i];
        int ahead = i - b * k;
        for (int c = 0; c < W && ahead < a.n_out; c++) {
            if (c == b) continue;
            int lo = 0, hi = k;  // candidates of row c that are ahead: larger, or as large and of a lower beam
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                const double y = s_key[c * k + mid];
                if (y > v || (y == v && c < b)) lo = mid + 1;
                else hi = mid;
            }
            ahead += lo;
        }
        chosen(i, ahead, v, __hip_atomic_load(id + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    }
}

// A workgroup for each row; the one of a request that is done last merges them.  Rows are passed on
// through atomic stores and loads, and counted when their stores have completed.
template <int TY>
__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a, int n_groups, int steps, int n_parts, const float *gmax, const Run *runs, double *key, int *id, int *arrived) {
    extern __shared__ double s_key[];
    __shared__ int s_last;
    const int row = blockIdx.x, req = row / a.n_beams;
    best_of_row<TY>(a, row, n_groups, steps, n_parts, gmax, runs, key, id);
    wait_vmem();
    __syncthreads();
    if (threadIdx.x == 0) s_last = __hip_atomic_fetch_add(arrived + req, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.n_beams - 1;
    __syncthreads();
    if (s_last) merge_rows(a, req, key, id, s_key);
}

struct BeamPlan {
    int steps, n_groups, per, n_parts;
};
BeamPlan beam_plan(int rows, int V) {
    BeamPlan p;
    const int n = (V + STEP - 1) / STEP;
    p.steps = (n + MAX_GROUPS - 1) / MAX_GROUPS;
    p.n_groups = (n + p.steps - 1) / p.steps;
    // groups per wave: enough waves to fill the card, and long runs beyond that
    p.per = (int)std::clamp<int64_t>(((int64_t)rows * p.n_groups + 8191) / 8192, 1, 32);
    p.n_parts = (p.n_groups + p.per - 1) / p.per;
    return p;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

constexpr size_t LDS_UNASKED = 32 << 10;  // dynamic LDS that, with what the kernel has itself, is under the 64 KiB that need not be asked for

template <int TY>
void launch_ty(const BeamArgs &a, void *ws, hipStream_t st) {
    const int rows = a.n * a.n_beams, k = std::min(a.n_out, a.V);
    const BeamPlan p = beam_plan(rows, a.V);
    uint8_t *w = (uint8_t *)ws;
    double *key = (double *)w;
    w += up16((size_t)rows * k * sizeof(double));
    int *id = (int *)w;
    w += up16((size_t)rows * k * sizeof(int));
    Run *runs = (Run *)w;
    w += up16((size_t)rows * p.n_parts * sizeof(Run));
    float *gmax = (float *)w;
    w += up16((size_t)rows * p.n_groups * sizeof(float));
    int *arrived = (int *)w;
    beam_part_kernel<TY><<<(int)(((int64_t)rows * p.n_parts + 3) / 4), 256, 0, st>>>(a, p.n_groups, p.steps, p.per, p.n_parts, gmax, runs, arrived);
    // the merge's sums: up to 64 KiB (64 beams of 128), beside 13 KiB that the rows take
    const size_t lds = (size_t)a.n_beams * k * sizeof(double);
    if (lds > LDS_UNASKED) RIE_HIP_CHECK(hipFuncSetAttribute((const void *)beam_row_kernel<TY>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    beam_row_kernel<TY><<<rows, 256, lds, st>>>(a, p.n_groups, p.steps, p.n_parts, gmax, runs, key, id, arrived);
}

}  // namespace

size_t beam_ws(int n, int n_beams, int V, int n_out) {
    const int64_t rows = (int64_t)n * n_beams;
    const int k = std::min(n_out, V);
    const BeamPlan p = beam_plan((int)rows, V);
    return up16(rows * k * sizeof(double)) + up16(rows * k * sizeof(int)) + up16(rows * p.n_parts * sizeof(Run)) + up16(rows * p.n_groups * sizeof(float)) + up16(n * sizeof(int));
}

void launch_beam(const BeamArgs &a, void *ws, hipStream_t st) {
    if (a.ty == T_F32) launch_ty<T_F32>(a, ws, st);
    else if (a.ty == T_F16) launch_ty<T_F16>(a, ws, st);
    else launch_ty<T_BF16>(a, ws, st);
}

}  // namespace rie
