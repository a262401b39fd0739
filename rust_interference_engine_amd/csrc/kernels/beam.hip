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
// so only those are read again.  beam_join_kernel merges the rows of a request.
//
// Beams are compared by sums in f64: in f32 the candidates of two beams would be equal to the last
// bit too often, and their order that of the roundings.  ln Σ is f64 of an f32 sum (2^-22 of it).
//
// Bound: HBM, rows · V values, and for a few rows the three launches.
#include "../common.hpp"
#include "../device.hpp"
#include "../serve.hpp"

#include <algorithm>
#include <cfloat>

namespace rie {

namespace {

constexpr int R = 16, STEP = 64 * R;  // logits of a lane and of a wave at a time
constexpr int MAX_GROUPS = 512;       // of a row: groups of 1024, 2048 or 4096 logits

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
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a, int n_groups, int steps, int per, int n_parts, float *gmax, Run *runs) {
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = id / n_parts, part = id - row * n_parts;
    if (row >= a.n * a.n_beams) return;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int g0 = part * per, g1 = min(g0 + per, n_groups), u1 = min(g1 * steps, (a.V + STEP - 1) / STEP);
    float M = -FLT_MAX, s = 0;  // the wave's maximum so far, and the lane's sum
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
            s *= exp2_hw((M - mx) * LOG2E_F);
            M = mx;
        }
#pragma unroll
        for (int j = 0; j < R; j++) s += exp2_hw((v[j] - M) * LOG2E_F);
#pragma unroll
        for (int j = 0; j < R; j++) v[j] = nx[j];
    }
    s = xsum_f<64>(s);
    if (lane == 0) runs[(int64_t)row * n_parts + part] = Run{M, s};
}

constexpr int CAND = 1024;  // logits that are ranked at once

// A row's best k = min(n_out, V) tokens in order, with their sums: key[row][k], id[row][k]
template <int TY>
__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a, int n_groups, int steps, int n_parts, const float *gmax, const Run *runs, double *key, int *id) {
    __shared__ Run s_run[4];
    __shared__ float s_val[CAND];
    __shared__ int s_idx[CAND];
    __shared__ float s_gmax[MAX_GROUPS];
    __shared__ int s_group[BEAM_MAX_OUT];
    __shared__ int s_n;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int k = min(a.n_out, a.V), kg = min(k, n_groups);
    key += (int64_t)row * k;
    id += (int64_t)row * k;
    const float score = a.scores[row];
    if (a.finished && a.finished[row]) {  // goes on as it is
        for (int i = tid; i < k; i += 256) {
            key[i] = i == 0 && fabsf(score) <= FLT_MAX ? (double)score : -INFINITY;
            id[i] = a.pad;
        }
        return;
    }
    Run p{-FLT_MAX, 0};
    for (int i = tid; i < n_parts; i += 256) p = join(p, runs[(int64_t)row * n_parts + i]);
    for (int i = tid; i < n_groups; i += 256) s_gmax[i] = gmax[(int64_t)row * n_groups + i];
#pragma unroll
    for (int o = 32; o; o >>= 1) p = join(p, Run{__shfl_xor(p.m, o), __shfl_xor(p.s, o)});
    if (lane == 0) s_run[w] = p;
    if (tid == 0) s_n = 0;
    __syncthreads();
    p = join(join(s_run[0], s_run[1]), join(s_run[2], s_run[3]));
    if (!(p.s > 0) || !(p.m <= FLT_MAX) || !(fabsf(score) <= FLT_MAX)) {  // offers nothing
        for (int i = tid; i < k; i += 256) {
            key[i] = -INFINITY;
            id[i] = i;
        }
        return;
    }
    const double log_s = log((double)p.s);
    // the groups with the largest maxima, by counting those ahead of each
    for (int i = tid; i < n_groups; i += 256) {
        const float v = s_gmax[i];
        int ahead = 0;
#pragma unroll 8
        for (int j = 0; j < n_groups; j++) ahead += (s_gmax[j] > v) | ((s_gmax[j] == v) & (j < i));
        if (ahead < kg) s_group[ahead] = i;
    }
    __syncthreads();
    // Their logits from the k-th largest group maximum on may be among the first k.  More than fit
    // (few groups, or equal logits): those from the k-th largest of the threads' own maxima on.
    float thr = kg < k ? -INFINITY : s_gmax[s_group[kg - 1]], mine = -INFINITY;
    for (int attempt = 0; attempt < 2; attempt++) {
        for (int u = w; u < kg * steps; u += 4) {
            float v[R];
            const int e0 = (s_group[u / steps] * steps + u % steps) * STEP;
            if (e0 >= a.V) continue;
            load_step<TY>(x, e0, a.V, lane, v);
#pragma unroll
            for (int j = 0; j < R; j++) {
                mine = fmaxf(mine, v[j]);
                if (!(v[j] >= thr) || v[j] == -INFINITY) continue;
                const int c = atomicAdd(&s_n, 1);
                if (c < CAND) {
                    s_val[c] = v[j];
                    s_idx[c] = e0 + place<TY>(lane, j);
                }
            }
        }
        __syncthreads();
        if (s_n <= CAND || attempt) break;
        __syncthreads();
        s_val[tid] = mine;
        if (tid == 0) s_n = 0;
        __syncthreads();
        int ahead = 0;
        for (int j = 0; j < 256; j++) ahead += (s_val[j] > mine) | ((s_val[j] == mine) & (j < tid));
        if (ahead == k - 1) s_val[256] = mine;
        __syncthreads();
        thr = s_val[256];
        __syncthreads();
    }
    const int n = s_n;
    if (n <= CAND) {
        for (int i = tid; i < n; i += 256) {
            const float v = s_val[i];
            const int e = s_idx[i];
            int ahead = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) ahead += (s_val[j] > v) | ((s_val[j] == v) & (s_idx[j] < e));
            if (ahead < k) {
                key[ahead] = (double)score + (((double)v - (double)p.m) - log_s);
                id[ahead] = e;
            }
        }
        if (n >= k) return;
        // the first of the logits of −inf: under k of the row's are none, so they lie in its first 2 k
        const bool out = tid < a.V && logit<TY>(x, tid) == -INFINITY;
        const uint64_t m = __ballot(out);
        __syncthreads();
        if (lane == 0) s_idx[w] = (int)__popcll(m);
        __syncthreads();
        int at = n + (int)__popcll(m & ((1ull << lane) - 1));
        for (int i = 0; i < w; i++) at += s_idx[i];
        if (out && at < k) {
            key[at] = -INFINITY;
            id[at] = tid;
        }
        return;
    }
    // more equal logits than fit: the next one of all of the groups' logits, k times
    float last = INFINITY;
    int last_e = -1;
    for (int r = 0; r < k; r++) {
        float bv = -INFINITY;
        int be = INT32_MAX;
        for (int i = tid; i < kg * steps * STEP; i += 256) {
            const int e = s_group[i / (steps * STEP)] * steps * STEP + i % (steps * STEP);
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
            s_val[w] = bv;
            s_idx[w] = be;
        }
        __syncthreads();
        for (int i = 0; i < 4; i++)
            if (s_val[i] > bv || (s_val[i] == bv && s_idx[i] < be)) {
                bv = s_val[i];
                be = s_idx[i];
            }
        last = bv;
        last_e = be;
        if (tid == 0) {
            key[r] = (double)score + (((double)bv - (double)p.m) - log_s);
            id[r] = be;
        }
    }
}

// The rows of a request merged.  Each row's candidates are in order, so what is ahead of one in
// another row is found by halving.
__global__ __launch_bounds__(256) void beam_join_kernel(BeamArgs a, const double *key, const int *id) {
    extern __shared__ double s_key[];
    const int W = a.n_beams, k = min(a.n_out, a.V), n = W * k, req = blockIdx.x;
    key += (int64_t)req * n;
    id += (int64_t)req * n;
    for (int i = threadIdx.x; i < n; i += 256) s_key[i] = key[i];
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
        if (ahead >= a.n_out) continue;
        const int64_t o = (int64_t)req * a.n_out + ahead;
        a.next[o] = (float)v;
        a.parents[o] = req * W + b;
        a.tokens[o] = id[i];
    }
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
    p.per = (int)std::clamp<int64_t>((int64_t)rows * p.n_groups / 8192, 1, 32);
    p.n_parts = (p.n_groups + p.per - 1) / p.per;
    return p;
}

size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

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
    beam_part_kernel<TY><<<(int)(((int64_t)rows * p.n_parts + 3) / 4), 256, 0, st>>>(a, p.n_groups, p.steps, p.per, p.n_parts, gmax, runs);
    beam_row_kernel<TY><<<rows, 256, 0, st>>>(a, p.n_groups, p.steps, p.n_parts, gmax, runs, key, id);
    beam_join_kernel<<<a.n, 256, (size_t)a.n_beams * k * sizeof(double), st>>>(a, key, id);
}

}  // namespace

size_t beam_ws(int n, int n_beams, int V, int n_out) {
    const int64_t rows = (int64_t)n * n_beams;
    const int k = std::min(n_out, V);
    const BeamPlan p = beam_plan((int)rows, V);
    return up16(rows * k * sizeof(double)) + up16(rows * k * sizeof(int)) + up16(rows * p.n_parts * sizeof(Run)) + up16(rows * p.n_groups * sizeof(float));
}

void launch_beam(const BeamArgs &a, void *ws, hipStream_t st) {
    if (a.ty == T_F32) launch_ty<T_F32>(a, ws, st);
    else if (a.ty == T_F16) launch_ty<T_F16>(a, ws, st);
    else launch_ty<T_BF16>(a, ws, st);
}

}  // namespace rie
