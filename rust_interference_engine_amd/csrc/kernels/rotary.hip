// rotary.hip — rotary positions for rows of queries and keys: of the first `dims` values of a
// head, pair i is turned by the angle a = p · f_i of its token's position p,
//
//   (x, y) → m · (x cos a − y sin a, x sin a + y cos a),
//
// where a pair is values i and i + dims/2 (halves) or 2i and 2i + 1 (interleaved).  The values
// behind are copied.
//
// Angles are formed and reduced to a quarter turn in f64: at position 10^6 the product in f32
// would be off by 0.06.  They depend on the token and the pair only, so a workgroup forms its
// rows' sines and cosines once, one or two to a thread, into LDS, and all heads use them.
//
// Bound: HBM (a launch and the chain position → angle → rows for a step's few tokens).  A thread
// takes 16 values at a time and requests four such items before it works on the first.
#include "../common.hpp"
#include "../serve_device.hpp"

namespace rie {

namespace {

constexpr int AT_ONCE = 4;

// cos and sin of position · freq.  The quarter turns' multiple of π/2 is taken out in two parts, the first of which
// is exact for up to 2^31 of them: 33 bits of π/2, and what is left.
__device__ __forceinline__ f32x2 turn(int position, double freq) {
    constexpr double P1 = 0x1.921fb544p+0, P2 = 0x1.0b4611a626331p-34;
    const double a = (double)position * freq, n = rint(a * 0x1.45f306dc9c883p-1);
    const float r = (float)fma(-n, P2, fma(-n, P1, a));
    const int quarter = (int)(n - 4.0 * floor(n * 0.25));
    const float s = sinf(r), c = cosf(r);
    const float x = quarter & 1 ? s : c, y = quarter & 1 ? c : s;
    return f32x2{(quarter + 1) & 2 ? -x : x, quarter & 2 ? -y : y};
}

template <int TY, int N>
__device__ __forceinline__ void get(const uint8_t *p, float (&v)[N]) {
    if constexpr (N == 8 && TY == T_F32) {
        const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 16);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[e] = a[e];
            v[4 + e] = b[e];
        }
    } else if constexpr (N == 8) {
        const u32x4 a = *(const u32x4 *)p;
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = value16<TY == T_BF16>(a[e / 2] >> (e & 1) * 16 & 0xFFFF);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = TY == T_F32 ? ((const float *)p)[e] : value16<TY == T_BF16>(((const uint16_t *)p)[e]);
    }
}
template <int TY, int N>
__device__ __forceinline__ void put(uint8_t *p, const float (&v)[N]) {
    if constexpr (N == 8 && TY == T_F32) {
        *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4 *)(p + 16) = f32x4{v[4], v[5], v[6], v[7]};
    } else if constexpr (N == 8) {
        constexpr bool BF = TY == T_BF16;
        *(u32x4 *)p = u32x4{pack2<BF>(v[0], v[1]), pack2<BF>(v[2], v[3]), pack2<BF>(v[4], v[5]), pack2<BF>(v[6], v[7])};
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) {
            if constexpr (TY == T_F32) ((float *)p)[e] = v[e];
            else ((uint16_t *)p)[e] = (uint16_t)pack2<TY == T_BF16>(v[e], v[e]);
        }
    }
}

// V: values of a piece, 8 or (rows of any alignment) 1.  An item is two pieces: of halves, the
// pairs' first and second values, else 2 V consecutive ones.
template <int SRC, int DST, int V, bool PAIRS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int R) {
    constexpr int ES = SRC == T_F32 ? 4 : 2, ED = DST == T_F32 ? 4 : 2;
    extern __shared__ f32x2 s_turn[];  // [row][pair]
    __shared__ int s_pos[16];
    __shared__ bool s_on[16];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), row0 = blockIdx.x * R, half = a.dims / 2;
    if (a.positions) {
        if (tid < R) {
            s_on[tid] = row0 + tid < a.b.n_rows;
            s_pos[tid] = s_on[tid] ? a.positions[row0 + tid] : 0;
        }
    } else {
        for (int i = w; i < R; i += 4) {
            const int row = row0 + i;
            int si;
            const SeqView sv = find_seq(a.b, a.kv, imin(row, a.b.n_rows - 1), si, [&](int s, int) { return iclamp(s, 0, a.b.n_rows); });
            s_on[i] = row < a.b.n_rows && row >= sv.row0 && row < sv.row0 + sv.n_new;
            s_pos[i] = sv.pos0() + row - sv.row0;
        }
    }
    __syncthreads();
    for (int i = tid; i < R * half; i += 256) {
        const int r = i / half, p = i - r * half;
        const f32x2 t = turn(s_pos[r], a.freqs[p]);
        s_turn[i] = f32x2{t[0] * a.magnitude, t[1] * a.magnitude};
    }
    __syncthreads();
    // items of a head: rotated ones, then the rest, which a call in place leaves alone
    const int turned = (half + V - 1) / V, rest = a.in_place ? 0 : (a.hd - a.dims + 2 * V - 1) / (2 * V), per = turned + rest;
    const int heads = a.n_q + a.n_k, n = R * heads * per;
    for (int i0 = tid; i0 < n; i0 += 256 * AT_ONCE) {
        float x[AT_ONCE][V], y[AT_ONCE][V];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int i = i0 + 256 * u;
            if (i >= n) break;
            const int it = i % per, rh = i / per, h = rh % heads, r = rh / heads;
            if (!s_on[r]) continue;
            const uint8_t *p = (h < a.n_q ? a.q + h * a.q_head + (row0 + r) * a.q_row : a.k + (h - a.n_q) * a.k_head + (row0 + r) * a.k_row);
            const int at = it < turned ? (PAIRS ? 2 * V * it : V * it) : a.dims + 2 * V * (it - turned);
            const int next = it < turned && !PAIRS ? half : V;
            get<SRC>(p + at * ES, x[u]);
            if (it < turned || at + V < a.hd) get<SRC>(p + (at + next) * ES, y[u]);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++) {
            const int i = i0 + 256 * u;
            if (i >= n) break;
            const int it = i % per, rh = i / per, h = rh % heads, r = rh / heads;
            if (!s_on[r]) continue;
            uint8_t *p = (h < a.n_q ? a.q_out + h * a.qo_head + (row0 + r) * a.qo_row : a.k_out + (h - a.n_q) * a.ko_head + (row0 + r) * a.ko_row);
            const int at = it < turned ? (PAIRS ? 2 * V * it : V * it) : a.dims + 2 * V * (it - turned);
            const int next = it < turned && !PAIRS ? half : V;
            if (it < turned) {
                const f32x2 *t = s_turn + r * half + it * V;
                if constexpr (PAIRS && V == 8) {
                    float z[16];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float b = e < 4 ? x[u][2 * e] : y[u][2 * e - 8], d = e < 4 ? x[u][2 * e + 1] : y[u][2 * e - 7];
                        z[2 * e] = b * t[e][0] - d * t[e][1];
                        z[2 * e + 1] = b * t[e][1] + d * t[e][0];
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        x[u][e] = z[e];
                        y[u][e] = z[8 + e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; e++) {
                        const float b = x[u][e], d = y[u][e];
                        x[u][e] = b * t[e][0] - d * t[e][1];
                        y[u][e] = b * t[e][1] + d * t[e][0];
                    }
                }
            }
            put<DST>(p + at * ED, x[u]);
            if (it < turned || at + V < a.hd) put<DST>(p + (at + next) * ED, y[u]);
        }
    }
}

template <int SRC, int DST>
void launch_types(const RotaryArgs &a, int R, int grid, size_t lds, hipStream_t st) {
    if (a.wide) {
        if (a.interleaved) rotary_kernel<SRC, DST, 8, true><<<grid, 256, lds, st>>>(a, R);
        else rotary_kernel<SRC, DST, 8, false><<<grid, 256, lds, st>>>(a, R);
    } else {
        if (a.interleaved) rotary_kernel<SRC, DST, 1, true><<<grid, 256, lds, st>>>(a, R);
        else rotary_kernel<SRC, DST, 1, false><<<grid, 256, lds, st>>>(a, R);
    }
}

template <int SRC>
void launch_src(const RotaryArgs &a, int R, int grid, size_t lds, hipStream_t st) {
    if (a.dst_ty == T_F32) launch_types<SRC, T_F32>(a, R, grid, lds, st);
    else if (a.dst_ty == T_F16) launch_types<SRC, T_F16>(a, R, grid, lds, st);
    else launch_types<SRC, T_BF16>(a, R, grid, lds, st);
}

}  // namespace

void launch_rotary(const RotaryArgs &a, hipStream_t st) {
    // a workgroup's rows: four where that leaves enough workgroups to fill the card
    const int R = a.b.n_rows >= 2048 ? 4 : 1, grid = (a.b.n_rows + R - 1) / R;
    const size_t lds = (size_t)R * (a.dims / 2) * sizeof(f32x2);
    if (a.src_ty == T_F32) launch_src<T_F32>(a, R, grid, lds, st);
    else if (a.src_ty == T_F16) launch_src<T_F16>(a, R, grid, lds, st);
    else launch_src<T_BF16>(a, R, grid, lds, st);
}

}  // namespace rie
