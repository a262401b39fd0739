// logprobs.hip — log probabilities of given tokens, the entropy and the most likely tokens
// of rows of logits x[0..V):
//
//   m = max x, S = Σ e^(x − m):  ln p_t = x_t − m − ln S,  H = ln S + Σ e^(x − m) (m − x) / S
//
// The logits are read once.  logprob_part_kernel takes groups of 1024 consecutive logits, a
// wave per run of groups, with the running maximum, the sum and the weighted sum in f32, and
// keeps every group's maximum; logprob_row_kernel joins a row's runs.  The k most likely
// tokens lie in the k groups with the largest maxima (by value, then by place: a group ahead
// of theirs holds a logit ahead of them), so only those are read again.
//
// Accuracy: the elements that equal the maximum are counted and left out of the sum, so that
// ln S = ln count + ln(1 + rest / count) keeps its digits where one token takes nearly all of
// the probability; every term of H is positive.
//
// −inf logits have probability 0 and add nothing to H.  A row that holds a NaN or +inf, or
// nothing above −inf, has NaN for all of its numbers; its top_ids still rank by logit, with
// NaN as −inf, and the lowest index first among equals.
//
// Bound: HBM, rows · V values.  512 rows of 128256 f32 (263 MB): 51 us and 5 for the second
// kernel, 5.1 TB/s and 4.7 together; 1021 rows of 151936 bf16 with 20 alternatives (310 MB): 70
// us, 4.4 TB/s (the exponentials' vector work beside it), and 26, of which 41 MB read again; one
// row with 5: 3.4 and 7.8, latency.  Groups of 512 and exponents by a subtraction and a product:
// 57, 83 and 49 us, and 23 for the one row's second kernel, which ranked all maxima.
#include "../common.hpp"
#include "../device.hpp"
#include "../serve.hpp"

#include <algorithm>
#include <cfloat>

namespace rie {

namespace {

constexpr int R = 16, GROUP = 64 * R;  // logits of a lane and of a group
constexpr float FAST_M = 1 << 20;      // size of a maximum below which an exponent is one fma
constexpr float D_MIN = -200;          // e^-200 is 0 in f32: the weighted sum's factor is cut there, so that 0 · -inf is not NaN

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

template <int TY>
__device__ __forceinline__ float logit(const void *x, int64_t i) {
    if constexpr (TY == T_F32) return ((const float *)x)[i];
    const uint16_t b = ((const uint16_t *)x)[i];
    return TY == T_BF16 ? __uint_as_float((uint32_t)b << 16) : h2f(b);
}

// Place of a lane's value j of a group: runs of 16 bytes, the lanes' side by side
template <int TY>
__device__ __forceinline__ int place(int lane, int j) {
    constexpr int N = TY == T_F32 ? 4 : 8;
    return j / N * (64 * N) + lane * N + j % N;
}

// The lane's values of the group that starts at element e0 of the row; −inf behind the row's
// ends (e0 is negative in the first group of a row that is not 16-byte aligned)
template <int TY>
__device__ __forceinline__ void load_group(const void *x, int e0, int V, int lane, float (&v)[R]) {
    if (e0 >= 0 && e0 + GROUP <= V) {
        if constexpr (TY == T_F32) {
            f32x4 a[R / 4];
#pragma unroll
            for (int i = 0; i < R / 4; i++) a[i] = *(const f32x4 *)((const float *)x + e0 + place<TY>(lane, 4 * i));
#pragma unroll
            for (int j = 0; j < R; j++) v[j] = a[j / 4][j % 4];
        } else {
            u16x8 a[R / 8];
#pragma unroll
            for (int i = 0; i < R / 8; i++) a[i] = *(const u16x8 *)((const uint16_t *)x + e0 + place<TY>(lane, 8 * i));
#pragma unroll
            for (int j = 0; j < R; j++) v[j] = TY == T_BF16 ? __uint_as_float((uint32_t)a[j / 8][j % 8] << 16) : h2f(a[j / 8][j % 8]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < R; j++) {
            const int e = e0 + place<TY>(lane, j);
            v[j] = e >= 0 && e < V ? logit<TY>(x, e) : -INFINITY;
        }
    }
}

// the elements by which a row's start lies behind a 16-byte boundary
template <int TY>
__device__ __forceinline__ int misplaced(const void *x) {
    return (int)((uintptr_t)x & 15) / (TY == T_F32 ? 4 : 2);
}

struct Part {  // of a run of logits: maximum, Σ e^(x − m) without the elements that equal it, their count, Σ e^(x − m) (x − m)
    float m, s, c, t;
};
__device__ __forceinline__ Part join(const Part &a, const Part &b) {
    const bool ab = a.m >= b.m;
    const float m = ab ? a.m : b.m, d = ab ? b.m - a.m : a.m - b.m;
    Part r;
    r.m = m;
    if (d == 0) {
        r.s = a.s + b.s;
        r.c = a.c + b.c;
        r.t = a.t + b.t;
        return r;
    }
    const float f = exp2_hw(fmaxf(d, D_MIN) * LOG2E_F), ls = ab ? b.s : a.s, lc = ab ? b.c : a.c, lt = ab ? b.t : a.t;
    r.s = (ab ? a.s : b.s) + f * (ls + lc);
    r.c = ab ? a.c : b.c;
    r.t = (ab ? a.t : b.t) + f * (lt + (ls + lc) * fmaxf(d, D_MIN));
    return r;
}

template <int TY>
__global__ __launch_bounds__(256) void logprob_part_kernel(LogprobArgs a, int n_groups, int per, int n_parts, float *gmax, Part *parts) {
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = id / n_parts, part = id - row * n_parts;
    if (row >= a.n) return;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int off = misplaced<TY>(x), g0 = part * per, g1 = min(g0 + per, n_groups);
    // M is the wave's maximum so far; s, t and cnt are the lane's.  fs and ft are the same sums of
    // the groups that hold no element equal to M, in log2 units against the reference −c, where
    // c = −M · log2 e rounded: one fma forms an exponent, and the rounding of c, r = M · log2 e + c
    // exactly, is taken out of the sums when M moves or at the end (they hold 2^r times theirs).
    // r is at most half a step of c, 2^-4 for |M| < 2^20; from 3e9 on it could pass 128, and 2^-r
    // be infinite.  Larger M (a run of masked logits, say) take the form with a subtraction.
    float M = -FLT_MAX, s = 0, t = 0, cnt = 0, fs = 0, ft = 0, c = 0;
    bool plain = true;  // no fast form for this M
    auto settle = [&] {
        const float r = plain ? 0.0f : fmaf(M, LOG2E_F, c), f = exp2_hw(-r);
        s = fmaf(fs, f, s);
        t = fmaf(LN2_F * f, ft - r * fs, t);
        fs = ft = 0;
    };
    float v[R], nx[R];
    load_group<TY>(x, g0 * GROUP - off, a.V, lane, v);
    for (int g = g0; g < g1; g++) {
        if (g + 1 < g1) load_group<TY>(x, (g + 1) * GROUP - off, a.V, lane, nx);
        float mx = v[0];
#pragma unroll
        for (int j = 1; j < R - 1; j += 2) mx = fmaxf(fmaxf(mx, v[j]), v[j + 1]);
        mx = fmaxf(mx, v[R - 1]);
        mx = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(xmax_f<64>(mx))));
        mx = mx == mx ? mx : -INFINITY;  // nothing but NaN
        if (lane == 0) gmax[(int64_t)row * n_groups + g] = mx;
        bool slow = mx >= M || plain;
        if (mx > M) {
            settle();
            const float d = fmaxf(M - mx, D_MIN), f = exp2_hw(d * LOG2E_F);
            t = f * (t + (s + cnt) * d);
            s = f * (s + cnt);
            cnt = 0;
            M = mx;
            plain = !(fabsf(M) < FAST_M);
            c = plain ? 0.0f : -(M * LOG2E_F);
        }
        if (!slow) {
            float gs = 0, gt = 0;
#pragma unroll
            for (int j = 0; j < R; j++) {
                const float d = fmaf(v[j], LOG2E_F, c), e = exp2_hw(d);
                gs += e;
                gt = fmaf(e, d, gt);
            }
            slow = __any(gt != gt);  // a −inf (0 · −inf) or a NaN: the other form
            if (!slow) {
                fs += gs;
                ft += gt;
            }
        }
        if (slow) {
#pragma unroll
            for (int j = 0; j < R; j++) {
                const bool eq = v[j] == M;
                const float d = v[j] - M, e = eq ? 0.0f : exp2_hw(d * LOG2E_F);
                cnt += eq ? 1.0f : 0.0f;
                s += e;
                t = fmaf(e, eq ? 0.0f : fmaxf(d, D_MIN), t);
            }
        }
#pragma unroll
        for (int j = 0; j < R; j++) v[j] = nx[j];
    }
    settle();
    s = xsum_f<64>(s);
    t = xsum_f<64>(t);
    cnt = xsum_f<64>(cnt);
    if (lane == 0) parts[(int64_t)row * n_parts + part] = Part{M, s, cnt, t};
}

constexpr int CAND = 1024;  // logits that are ranked at once

template <int TY>
__global__ __launch_bounds__(256) void logprob_row_kernel(LogprobArgs a, int n_groups, int n_parts, const float *gmax, const Part *parts) {
    __shared__ Part s_part[4];
    __shared__ float s_val[CAND];
    __shared__ int s_idx[CAND];
    __shared__ int s_n;
    __shared__ int s_group[LOGPROB_MAX_TOP];
    __shared__ float s_thr;
    extern __shared__ float s_gmax[];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, row = blockIdx.x;
    const void *x = (const uint8_t *)a.x + row * a.ld * (TY == T_F32 ? 4 : 2);
    const int target = a.targets ? a.targets[row] : -1;
    const float xt = target >= 0 && target < a.V ? logit<TY>(x, target) : 0.0f;

    // The k groups with the largest maxima: the first wave takes them out one by one, the lowest
    // group among equals, a lane holding every 64th group's maximum in registers (in LDS beyond
    // 512 groups).  The other waves join the runs meanwhile.
    const int k = a.n_top, kg = min(k, n_groups);
    if (w == 0 && k) {
        constexpr int NREG = 8;
        const bool many = n_groups > 64 * NREG;
        const float *gm = gmax + (int64_t)row * n_groups;
        float own[NREG], best = -INFINITY;
        int at = INT32_MAX;
#pragma unroll
        for (int i = 0; i < NREG; i++) own[i] = lane + 64 * i < n_groups ? gm[lane + 64 * i] : NAN;
        if (many)
            for (int i = lane; i < n_groups; i += 64) s_gmax[i] = gm[i];
        auto look = [&] {  // NaN (taken, or no group) compares with nothing
            best = -INFINITY;
            at = INT32_MAX;
            if (!many) {
#pragma unroll
                for (int i = 0; i < NREG; i++) {
                    const bool better = own[i] > best || (at == INT32_MAX && own[i] == best);
                    best = better ? own[i] : best;
                    at = better ? lane + 64 * i : at;
                }
            } else {
                for (int i = lane; i < n_groups; i += 64) {
                    const float v = s_gmax[i];
                    if (v > best || (at == INT32_MAX && v == best)) {
                        best = v;
                        at = i;
                    }
                }
            }
        };
        look();
        float thr = -INFINITY;
        for (int r = 0; r < kg; r++) {
            thr = xmax_f<64>(best);
            const int first = xreduce<64>(best == thr ? at : INT32_MAX, [](int x, int y) { return x < y ? x : y; });
            if (lane == 0) s_group[r] = first;
            if (at == first) {
                if (many) s_gmax[at] = NAN;
#pragma unroll
                for (int i = 0; i < NREG; i++) own[i] = at == lane + 64 * i ? NAN : own[i];
                look();
            }
        }
        if (lane == 0) s_thr = n_groups < k ? -INFINITY : thr;
    }
    Part p{-FLT_MAX, 0, 0, 0};
    const int first = k ? 64 : 0;  // thread that joins the first run
    for (int i = tid - first; i >= 0 && i < n_parts; i += 256 - first) p = join(p, parts[(int64_t)row * n_parts + i]);
#pragma unroll
    for (int o = 32; o; o >>= 1) p = join(p, Part{__shfl_xor(p.m, o), __shfl_xor(p.s, o), __shfl_xor(p.c, o), __shfl_xor(p.t, o)});
    if (lane == 0) s_part[w] = p;
    if (tid == 0) s_n = 0;
    __syncthreads();
    p = join(join(s_part[0], s_part[1]), join(s_part[2], s_part[3]));
    const bool none = !(p.c > 0) || !(p.m <= FLT_MAX);
    const float log_s = none ? NAN : logf(p.c) + log1pf(p.s / p.c);
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = log_s - p.t / (p.c + p.s);
        if (a.logprob) a.logprob[row] = target >= 0 && target < a.V ? xt - p.m - log_s : NAN;
    }
    if (!k) return;

    // their logits that may be among the first k
    const float thr = s_thr;
    const bool all = thr == -INFINITY;
    const int off = misplaced<TY>(x);
    constexpr int AT_ONCE = 3;  // groups that a wave reads at once
    for (int i0 = w; i0 < kg; i0 += 4 * AT_ONCE) {
        float v[AT_ONCE][R];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
            if (i0 + 4 * u < kg) load_group<TY>(x, s_group[i0 + 4 * u] * GROUP - off, a.V, lane, v[u]);
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            if (i0 + 4 * u >= kg) break;
            const int e0 = s_group[i0 + 4 * u] * GROUP - off;
#pragma unroll
            for (int j = 0; j < R; j++) {
                if (!(v[u][j] >= thr) && !(all && v[u][j] != v[u][j])) continue;
                const int e = e0 + place<TY>(lane, j);
                if (all && (e < 0 || e >= a.V)) continue;  // the −inf behind the row's ends
                const int c = atomicAdd(&s_n, 1);
                if (c < CAND) {
                    s_val[c] = v[u][j] == v[u][j] ? v[u][j] : -INFINITY;
                    s_idx[c] = e;
                }
            }
        }
    }
    __syncthreads();
    const int n = s_n;
    if (n <= CAND) {
        for (int i = tid; i < n; i += 256) {
            const float v = s_val[i];
            const int e = s_idx[i];
            int ahead = 0;
#pragma unroll 8
            for (int j = 0; j < n; j++) ahead += (s_val[j] > v) | ((s_val[j] == v) & (s_idx[j] < e));
            if (ahead < k) {
                a.top_ids[(int64_t)row * k + ahead] = e;
                a.top_logprobs[(int64_t)row * k + ahead] = v - p.m - log_s;
            }
        }
        return;
    }
    // more equal logits than fit: the next one of all of the groups' logits, k times
    float last = INFINITY;
    int last_e = -1;
    for (int r = 0; r < k; r++) {
        float bv = -INFINITY;
        int be = INT32_MAX;
        for (int i = tid; i < kg * GROUP; i += 256) {
            const int e = s_group[i / GROUP] * GROUP - off + i % GROUP;
            if (e < 0 || e >= a.V) continue;
            float v = logit<TY>(x, e);
            v = v != v ? -INFINITY : v;
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
            a.top_ids[(int64_t)row * k + r] = be;
            a.top_logprobs[(int64_t)row * k + r] = bv - p.m - log_s;
        }
    }
}

// groups of a row: one more than its logits fill, for rows that begin inside 16 bytes
int groups_of(int V) { return (V + 7 + GROUP - 1) / GROUP; }

}  // namespace

size_t logprobs_ws(int n, int V) { return (size_t)n * groups_of(V) * (sizeof(float) + sizeof(Part)); }

void launch_logprobs(const LogprobArgs &a, void *ws, hipStream_t st) {
    const int ng = groups_of(a.V);
    // groups per wave: enough waves to fill the card, and long runs beyond that
    const int per = (int)std::clamp<int64_t>((int64_t)a.n * ng / 8192, 1, 32), np = (ng + per - 1) / per;
    Part *parts = (Part *)ws;
    float *gmax = (float *)(parts + (size_t)a.n * np);
    const int grid = (int)(((int64_t)a.n * np + 3) / 4);
    const size_t lds = a.n_top && ng > 512 ? ng * sizeof(float) : 0;
    if (a.ty == T_F32) {
        logprob_part_kernel<T_F32><<<grid, 256, 0, st>>>(a, ng, per, np, gmax, parts);
        logprob_row_kernel<T_F32><<<a.n, 256, lds, st>>>(a, ng, np, gmax, parts);
    } else if (a.ty == T_F16) {
        logprob_part_kernel<T_F16><<<grid, 256, 0, st>>>(a, ng, per, np, gmax, parts);
        logprob_row_kernel<T_F16><<<a.n, 256, lds, st>>>(a, ng, np, gmax, parts);
    } else {
        logprob_part_kernel<T_BF16><<<grid, 256, 0, st>>>(a, ng, per, np, gmax, parts);
        logprob_row_kernel<T_BF16><<<a.n, 256, lds, st>>>(a, ng, np, gmax, parts);
    }
}

}  // namespace rie
