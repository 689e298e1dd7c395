// The joint of a residual block, one pass over the rows:
//     y = x + s * a(g) * N_post(f)        (the block's output f normed, gated, scaled and added to the stream x)
//     h = N_pre(y)                        (the next block's input)
// with N = layernorm (v - mean) / (std_unbiased + eps) * gain + shift -- the framework's own form (models/attn.py:39-42) -- or rmsnorm
// v / sqrt(mean(v^2) + eps) * gain (+ shift), a = identity, sigmoid or silu, g one gate per element or per row, s a number or one per column.
// Bound by HBM: forward reads x, f, g and writes y, h; backward reads x, f, g, d_y, d_h and writes d_x, d_f, d_g.  The backward pass reads x and
// recomputes y in float32 (reading the rounded y instead would move the same bytes).  Measured: 16,384 x 2048 bf16 forward with a full gate 66 us (5.1 TB/s; a large copy 5.2);
// 512,000 x 256 f16 with a row gate 202 us forward (5.2 TB/s) and 307 backward (5.1); 60,000 x 1000 float32 without a gate 188 and 242 (5.1, 6.0).
//
// A row lies in the registers of G lanes, eight elements each (G = the power of two that covers the width): sums over a row are DPP steps inside a
// wave, one LDS exchange where a row takes several waves.  Norms in two passes over the registers (mean, then squares): no cancellation.
#include "block_types.h"

namespace {

constexpr int E = 8;                              // elements of a row per lane

// (a DPP operand that the compiler may fold into the addition)
#define LANES(v, ctrl) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float (*lds)[N][16], int& turn) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
        v[n] += LANES(v[n], 0xB1);
        v[n] += LANES(v[n], 0x4E);
        if (G >= 8) v[n] += LANES(v[n], 0x141);
        if (G >= 16) v[n] += LANES(v[n], 0x140);
        if (G >= 32) v[n] += __shfl_xor(v[n], 16);
        if (G >= 64) v[n] += __shfl_xor(v[n], 32);
    }
    if (G > 64) {                                 // (two turns of the table: a wave writes one while slower waves still read the other)
        const int wave = threadIdx.x >> 6;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int n = 0; n < N; ++n) lds[turn][n][wave] = v[n];
        __syncthreads();
        const int first = wave / (G / 64) * (G / 64);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float s = 0.f;
#pragma unroll
            for (int w = 0; w < G / 64; ++w) s += lds[turn][n][first + w];
            v[n] = s;
        }
    }
}

template <typename T, int V, int G>
struct Row {
    static constexpr int CH = E / V;
    // column of element i of lane j
    static __device__ __forceinline__ int col(int j, int i) { return (i / V * G + j) * V + i % V; }
    struct Raw { papr_pack<T, V> t[CH]; };         // a row on its way: in the rows' type, a third of the registers
    static __device__ __forceinline__ void fetch(Raw& r, const T* row, int width, int j) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + j) * V;
            if (at < width) r.t[c] = *reinterpret_cast<const papr_pack<T, V>*>(row + at);
        }
    }
    // whole: (uniform) every lane's chunks lie inside the row
    static __device__ __forceinline__ void values(float (&v)[E], const Raw& r, int width, int j, bool whole) {
        if (whole) {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = (float)r.t[i / V].v[i % V];
            return;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const bool in = (c * G + j) * V < width;
#pragma unroll
            for (int i = 0; i < V; ++i) v[c * V + i] = in ? (float)r.t[c].v[i] : 0.f;
        }
    }
    static __device__ __forceinline__ void store(const float (&v)[E], T* row, int width, int j) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + j) * V;
            if (at >= width) continue;
            papr_pack<T, V> t;
#pragma unroll
            for (int i = 0; i < V; ++i) t.v[i] = (T)v[c * V + i];
            *reinterpret_cast<papr_pack<T, V>*>(row + at) = t;
        }
    }
    static __device__ __forceinline__ void param(float (&v)[E], const void* p, int type, int width, int j, float absent) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = (c * G + j) * V;
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = absent;
            if (p && at < width) load_param<V>(t, p, type, at);
#pragma unroll
            for (int i = 0; i < V; ++i) v[c * V + i] = at < width ? t[i] : 0.f;
        }
    }
};

// a(g) and a'(g)
template <bool EXACT>
__device__ __forceinline__ void gate_of(float g, int act, float& value, float& slope) {
    if (act == PAPR_GATE_NONE) { value = g; slope = 1.f; return; }
    const float p = papr_sigmoid<EXACT>(g);
    value = act == PAPR_GATE_SIGMOID ? p : g * p;
    slope = act == PAPR_GATE_SIGMOID ? p * (1.f - p) : p * __builtin_fmaf(g, 1.f - p, 1.f);
}

// v <- standardised rows; stats = {mean, 1 / divisor, factor of the correlation term in the backward pass}
template <int G, int V>
__device__ __forceinline__ void standardise(float (&v)[E], int kind, float eps, int width, int j, float (&stats)[3], float (*lds)[1][16], int& turn) {
    if (kind == PAPR_NORM_NONE) return;
    const float rw = 1.f / (float)width;
    float s[1] = {0.f};
    stats[0] = 0.f;
    if (kind == PAPR_NORM_LAYER) {
#pragma unroll
        for (int i = 0; i < E; ++i) s[0] += v[i];
        group_sum<G, 1>(s, lds, turn);
        stats[0] = s[0] * rw;
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = (i / V * G + j) * V < width ? v[i] - stats[0] : 0.f;
    }
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] = __builtin_fmaf(v[i], v[i], s[0]);
    group_sum<G, 1>(s, lds, turn);
    if (kind == PAPR_NORM_LAYER) {
        // (hardware square root and reciprocals, an ulp each: the precise forms were a fifth of the forward kernel's instructions at 256 columns)
        const float rest = __builtin_amdgcn_rcpf((float)(width - 1)), std = __builtin_amdgcn_sqrtf(s[0] * rest), div = std + eps;
        stats[1] = __builtin_amdgcn_rcpf(div);
        stats[2] = std > 0.f ? div * rest * __builtin_amdgcn_rcpf(std) : 0.f;      // (a constant row: the deviation's slope is taken as zero, like torch's)
    } else {
        stats[1] = __builtin_amdgcn_rsqf(__builtin_fmaf(s[0], rw, eps));
        stats[2] = rw;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= stats[1];
}

// (four waves a SIMD, the four workgroups a compute unit that join_blocks counts on: with registers for three the last quarter ran alone, 79,282 x 712 float32 315 us for 175)
template <typename T, int V, int G>
__global__ __launch_bounds__(G > 256 ? G : 256, 4) void join_fwd_kernel(papr_join_desc d, T* __restrict__ y_out, T* __restrict__ h_out, float* __restrict__ stats_out) {
    typedef Row<T, V, G> R;
    constexpr int THREADS = G > 256 ? G : 256, RPB = THREADS / G;
    __shared__ float lds[2][1][16];
    int turn = 0;
    const int j = threadIdx.x % G, width = d.width;
    float pa[E], pb[E], qa[E], qb[E], sc[E];
    R::param(pa, d.post.gain, d.post.type, width, j, 1.f);
    R::param(pb, d.post.shift, d.post.type, width, j, 0.f);
    R::param(qa, d.pre.gain, d.pre.type, width, j, 1.f);
    R::param(qb, d.pre.shift, d.pre.type, width, j, 0.f);
    R::param(sc, d.scale_cols, d.scale_type, width, j, d.scale);
    // the next row's loads are on their way while this one is computed: a wave has 2 to 3 KB in flight all the time
    const bool whole = width == G * E;
    typename R::Raw rx, rf, rg;
    float g1 = 0.f;
    const int64_t step = (int64_t)gridDim.x * RPB, first = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
    auto fetch = [&](int64_t at) {
        const int64_t row = at < d.rows ? at : d.rows - 1;
        R::fetch(rx, reinterpret_cast<const T*>(d.x) + row * d.ldx, width, j);
        if (d.f) R::fetch(rf, reinterpret_cast<const T*>(d.f) + row * d.ldf, width, j);
        if (d.gate_form == PAPR_GATE_FULL) R::fetch(rg, reinterpret_cast<const T*>(d.gate) + row * d.ldg, width, j);
        if (d.gate_form == PAPR_GATE_ROW) g1 = (float)reinterpret_cast<const T*>(d.gate)[row * d.ldg];
    };
    fetch(first);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB, at = first; r0 < d.rows; r0 += step, at += step) {
        const bool live = at < d.rows;
        const int64_t row = live ? at : d.rows - 1;
        float y[E], f[E], ga[E], st[6] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, slope;
        R::values(y, rx, width, j, whole);
        if (d.f) {
            R::values(f, rf, width, j, whole);
            if (d.gate_form == PAPR_GATE_FULL) {
                R::values(ga, rg, width, j, whole);
#pragma unroll
                for (int i = 0; i < E; ++i) gate_of<sizeof(T) == 4>(ga[i], d.gate_act, ga[i], slope);
            } else {
                float g = 1.f;
                if (d.gate_form == PAPR_GATE_ROW) gate_of<sizeof(T) == 4>(g1, d.gate_act, g, slope);
#pragma unroll
                for (int i = 0; i < E; ++i) ga[i] = g;
            }
        }
        if (r0 + step < d.rows) fetch(at + step);
        __builtin_amdgcn_sched_barrier(0);
        if (d.f) {
            float s3[3] = {0.f, 0.f, 0.f};
            standardise<G, V>(f, d.post.kind, d.post.eps, width, j, s3, lds, turn);
            st[0] = s3[0]; st[1] = s3[1]; st[2] = s3[2];
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] += sc[i] * ga[i] * __builtin_fmaf(f[i], pa[i], pb[i]);
            if (live && y_out) R::store(y, y_out + row * width, width, j);
        }
        if (h_out) {
            float s3[3] = {0.f, 0.f, 0.f};
            standardise<G, V>(y, d.pre.kind, d.pre.eps, width, j, s3, lds, turn);
            st[3] = s3[0]; st[4] = s3[1]; st[5] = s3[2];
#pragma unroll
            for (int i = 0; i < E; ++i) y[i] = __builtin_fmaf(y[i], qa[i], qb[i]);
            if (live) R::store(y, h_out + row * width, width, j);
        }
        if (stats_out && live && j == 0) {
#pragma unroll
            for (int i = 0; i < 6; ++i) stats_out[row * 6 + i] = st[i];
        }
    }
}

template <typename T, int V, int G>
__global__ __launch_bounds__(G > 256 ? G : 256, 2) void join_bwd_kernel(papr_join_desc d, const float* __restrict__ stats, const T* __restrict__ d_y, const T* __restrict__ d_h,
                                                                     T* __restrict__ d_x, T* __restrict__ d_f, T* __restrict__ d_g, float* __restrict__ part) {
    typedef Row<T, V, G> R;
    constexpr int THREADS = G > 256 ? G : 256, RPB = THREADS / G;
    __shared__ float lds[2][3][16], lds2[2][2][16];
    __shared__ float fold[RPB > 1 ? RPB * G * E : 1];
    int turn = 0;
    const int j = threadIdx.x % G, width = d.width;
    const float rw = 1.f / (float)width;
    // What a compute unit has on its way is what bounds this kernel (eight waves; 512,000 x 256 float16 with one row's operands each 352 us, 4.5 TB/s, with two 311, 5.1): two rows ahead of the arithmetic,
    // with the parameters read again from LDS row by row instead of sitting in 32 registers.  float32 rows (twice the bytes) and odd ones: one row ahead.
    constexpr int AHEAD = G == 512 || sizeof(T) == 4 || V == 1 ? 1 : 2;
    // Rows of eight waves: gates and p are computed again behind the next norm's sums instead of being carried over them (32 registers).
    constexpr bool AGAIN = G == 512;
    __shared__ __attribute__((aligned(16))) float par[4][G * E];
    float pa[E], pb[E], qa[E], sc[E];
    R::param(pa, d.post.gain, d.post.type, width, j, 1.f);
    R::param(pb, d.post.shift, d.post.type, width, j, 0.f);
    R::param(qa, d.pre.gain, d.pre.type, width, j, 1.f);
    R::param(sc, d.scale_cols, d.scale_type, width, j, d.scale);
    auto param = [&](int q, float (&v)[E], bool put) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            float4* at = (float4*)&par[q][(i / 4 * G + j) * 4];
            if (put) *at = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            else { const float4 t = *at; v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w; }
        }
    };
    if (threadIdx.x < G) { param(0, pa, true); param(1, pb, true); param(2, qa, true); param(3, sc, true); }
    __syncthreads();
    float acc[5][E];                              // column sums: d(pre gain), d(pre shift), d(post gain), d(post shift), d(scale)
#pragma unroll
    for (int a = 0; a < 5; ++a)
#pragma unroll
        for (int i = 0; i < E; ++i) acc[a][i] = 0.f;
    struct Operands { typename R::Raw x, f, g, y, h; T gate; float st[6]; } w0, w1;
    const int64_t step = (int64_t)gridDim.x * RPB, first = (int64_t)blockIdx.x * RPB + threadIdx.x / G;
    auto fetch = [&](Operands& w, int64_t at) __attribute__((always_inline)) {
        const int64_t row = at < d.rows ? at : d.rows - 1;
        R::fetch(w.x, reinterpret_cast<const T*>(d.x) + row * d.ldx, width, j);
        if (d.f) R::fetch(w.f, reinterpret_cast<const T*>(d.f) + row * d.ldf, width, j);
        if (d.gate_form == PAPR_GATE_FULL) R::fetch(w.g, reinterpret_cast<const T*>(d.gate) + row * d.ldg, width, j);
        if (d.gate_form == PAPR_GATE_ROW) w.gate = reinterpret_cast<const T*>(d.gate)[row * d.ldg];
        if (d_y) R::fetch(w.y, d_y + row * width, width, j);
        if (d_h) R::fetch(w.h, d_h + row * width, width, j);
#pragma unroll
        for (int i = 0; i < 6; ++i) w.st[i] = stats[row * 6 + i];
    };
    const bool whole = width == G * E;
    auto one_row = [&](Operands& w, int64_t r0, int64_t at) __attribute__((always_inline)) {
        const bool live = at < d.rows;
        const int64_t row = live ? at : d.rows - 1;
        float x[E], f[E], g[E], dy[E], dh[E];
        const bool all_live = r0 + RPB <= d.rows;      // (uniform)
        const int seen = live ? width : 0;        // (a row past the end: zero gradients, nothing reaches the sums)
        R::values(x, w.x, width, j, whole);
        if (d.f) R::values(f, w.f, width, j, whole);
        if (d.gate_form == PAPR_GATE_FULL) R::values(g, w.g, width, j, whole);
        if (d_y) R::values(dy, w.y, seen, j, whole && all_live);
        if (d_h) R::values(dh, w.h, seen, j, whole && all_live);
        const float g1 = d.gate_form == PAPR_GATE_ROW ? (float)w.gate : 0.f, m1 = w.st[0], r1 = w.st[1], c1 = w.st[2], m2 = w.st[3], r2 = w.st[4], c2 = w.st[5];
        fetch(w, at + AHEAD * step);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");            // (the parameters are read where they are used, row by row)
        param(0, pa, false);
        param(1, pb, false);
        param(3, sc, false);
        // (columns past the end need no care here: their gains, scale and incoming gradients are zero, so nothing of them reaches a row's sums, and their own results are
        // never stored)
        const bool post = d.post.kind != PAPR_NORM_NONE;
        float ga[E], gn[E], gs[E], p[E];
        auto gates = [&]() __attribute__((always_inline)) {
            if (d.gate_form == PAPR_GATE_FULL) {
#pragma unroll
                for (int i = 0; i < E; ++i) gate_of<sizeof(T) == 4>(g[i], d.gate_act, ga[i], gs[i]);
            } else {
                float gv = 1.f, sv = 0.f;
                if (d.gate_form == PAPR_GATE_ROW) gate_of<sizeof(T) == 4>(g1, d.gate_act, gv, sv);
#pragma unroll
                for (int i = 0; i < E; ++i) { ga[i] = gv; gs[i] = sv; }
            }
        };
        if (d.f) {
            gates();
            if (post)
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = (f[i] - m1) * r1;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                p[i] = __builtin_fmaf(f[i], pa[i], pb[i]);
                gn[i] = ga[i];
                ga[i] *= sc[i];
                x[i] = __builtin_fmaf(ga[i], p[i], x[i]);
            }
        }
        if (!d_y)
#pragma unroll
            for (int i = 0; i < E; ++i) dy[i] = 0.f;
        if (d_h) {
            asm volatile("" ::: "memory");
            param(2, qa, false);
            if (d.pre.kind == PAPR_NORM_NONE) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    acc[0][i] = __builtin_fmaf(dh[i], x[i], acc[0][i]);
                    acc[1][i] += dh[i];
                    dy[i] = __builtin_fmaf(dh[i], qa[i], dy[i]);
                }
            } else {
                float s[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    x[i] = (x[i] - m2) * r2;
                    acc[0][i] = __builtin_fmaf(dh[i], x[i], acc[0][i]);
                    acc[1][i] += dh[i];
                    dh[i] *= qa[i];
                    s[0] = __builtin_fmaf(dh[i], x[i], s[0]);
                    s[1] += dh[i];
                }
                group_sum<G, 2>(s, lds2, turn);
                const float t = s[0] * c2 * r2, m = d.pre.kind == PAPR_NORM_LAYER ? s[1] * rw * r2 : 0.f;
#pragma unroll
                for (int i = 0; i < E; ++i) dy[i] += __builtin_fmaf(dh[i], r2, -__builtin_fmaf(x[i], t, m));
            }
        }
        if (live && d_x) R::store(dy, d_x + row * width, width, j);
        if (!d.f) return;
        float s[3] = {0.f, 0.f, 0.f}, dp[E];
        asm volatile("" ::: "memory");
        param(0, pa, false);
        param(3, sc, false);
        if (AGAIN) {
            param(1, pb, false);
#pragma unroll
            for (int i = 0; i < E; ++i) asm volatile("" : "+v"(g[i]), "+v"(f[i]));       // (computed here, not carried)
            gates();
#pragma unroll
            for (int i = 0; i < E; ++i) {
                p[i] = __builtin_fmaf(f[i], pa[i], pb[i]);
                gn[i] = ga[i];
                ga[i] *= sc[i];
            }
        }
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float w = dy[i] * p[i];
            dp[i] = dy[i] * ga[i];
            acc[4][i] = __builtin_fmaf(gn[i], w, acc[4][i]);
            g[i] = sc[i] * w * gs[i];
            s[2] += g[i];
            acc[2][i] = __builtin_fmaf(dp[i], f[i], acc[2][i]);
            acc[3][i] += dp[i];
            dp[i] *= pa[i];
            s[0] = __builtin_fmaf(dp[i], f[i], s[0]);
            s[1] += dp[i];
        }
        if (post || d.gate_form == PAPR_GATE_ROW) group_sum<G, 3>(s, lds, turn);
        if (d_g) {
            if (d.gate_form == PAPR_GATE_FULL) { if (live) R::store(g, d_g + row * width, width, j); }
            else if (live && j == 0) d_g[row] = (T)s[2];
        }
        if (post) {
            const float t = s[0] * c1 * r1, m = d.post.kind == PAPR_NORM_LAYER ? s[1] * rw * r1 : 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) dp[i] = __builtin_fmaf(dp[i], r1, -__builtin_fmaf(f[i], t, m));
        }
        if (live && d_f) R::store(dp, d_f + row * width, width, j);
    };
    fetch(w0, first);
    if (AHEAD > 1) fetch(w1, first + step);
    for (int64_t r0 = (int64_t)blockIdx.x * RPB, at = first; r0 < d.rows; r0 += AHEAD * step, at += AHEAD * step) {
        one_row(w0, r0, at);
        if (AHEAD > 1 && r0 + step < d.rows) one_row(w1, r0 + step, at + step);
    }
    if (!part) return;
    // the workgroup's row groups meet in LDS, in group order; one partial row per workgroup and array
    float* out = part + (int64_t)blockIdx.x * 5 * width;
#pragma unroll
    for (int a = 0; a < 5; ++a) {
        if (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i) fold[(threadIdx.x / G * E + i) * G + j] = acc[a][i];
            __syncthreads();
            for (int q = threadIdx.x; q < E * G; q += THREADS) {
                float s = 0.f;
                for (int k = 0; k < RPB; ++k) s += fold[k * E * G + q];
                const int c = R::col(q % G, q / G);
                if (c < width) out[(int64_t)a * width + c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int c = R::col(j, i);
                if (c < width) out[(int64_t)a * width + c] = acc[a][i];
            }
        }
    }
}

// The backward pass of rows above 4096 columns: sixteen waves a row, so 128 registers a lane in all, 40 of them column sums.  The row is held as it lies in memory and
// everything made of it is made again in each of the three stages (the next norm's sums; d_x, d_g and the other norm's sums; d_f), four elements at a time; the
// parameters lie in LDS.  9000 x 5000 in bf16 272 us, in float32 273 (4.0 TB/s; the next row's loads have no registers to wait in); with the values carried between the
// stages 600 bytes a lane were spilled: 2007 and 1191 us.
template <typename T, int V>
__global__ __launch_bounds__(1024, 4) void join_bwd_wide_kernel(papr_join_desc d, const float* __restrict__ stats, const T* __restrict__ d_y, const T* __restrict__ d_h,
                                                                T* __restrict__ d_x, T* __restrict__ d_f, T* __restrict__ d_g, float* __restrict__ part) {
    constexpr int G = 1024;
    typedef Row<T, V, G> R;
    __shared__ float lds[2][3][16], lds2[2][2][16];
    __shared__ __attribute__((aligned(16))) float par[4][G * E];
    int turn = 0;
    const int j = threadIdx.x, width = d.width;
    const float rw = 1.f / (float)width;
    {
        float v[E];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const void* p = q == 0 ? d.post.gain : q == 1 ? d.post.shift : q == 2 ? d.pre.gain : d.scale_cols;
            R::param(v, p, q < 2 ? d.post.type : q == 2 ? d.pre.type : d.scale_type, width, j, q == 1 ? 0.f : q == 3 ? d.scale : 1.f);
#pragma unroll
            for (int i = 0; i < E; i += 4) *(float4*)&par[q][(i / 4 * G + j) * 4] = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
    }                                             // (a lane's own places: no barrier)
    float acc[5][E];
#pragma unroll
    for (int a = 0; a < 5; ++a)
#pragma unroll
        for (int i = 0; i < E; ++i) acc[a][i] = 0.f;
    const bool post = d.post.kind != PAPR_NORM_NONE, pre = d.pre.kind != PAPR_NORM_NONE, full = d.gate_form == PAPR_GATE_FULL;
    auto fetch = [&](typename R::Raw& r, const T* row) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < R::CH; ++c) {
            const int at = (c * G + j) * V;
            if (row && at < width) r.t[c] = *reinterpret_cast<const papr_pack<T, V>*>(row + at);
            else
#pragma unroll
                for (int i = 0; i < V; ++i) r.t[c].v[i] = (T)0.f;
        }
    };
    auto put = [&](const typename R::Raw& r, T* row) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < R::CH; ++c) {
            const int at = (c * G + j) * V;
            if (at < width) *reinterpret_cast<papr_pack<T, V>*>(row + at) = r.t[c];
        }
    };
    for (int64_t row = blockIdx.x; row < d.rows; row += gridDim.x) {
        typename R::Raw rx, rf, rg, ry, rh;
        fetch(rx, reinterpret_cast<const T*>(d.x) + row * d.ldx);
        fetch(rf, d.f ? reinterpret_cast<const T*>(d.f) + row * d.ldf : nullptr);
        fetch(rg, full ? reinterpret_cast<const T*>(d.gate) + row * d.ldg : nullptr);
        fetch(ry, d_y ? d_y + row * width : nullptr);
        fetch(rh, d_h ? d_h + row * width : nullptr);
        const float m1 = stats[row * 6], r1 = stats[row * 6 + 1], c1 = stats[row * 6 + 2], m2 = stats[row * 6 + 3], r2 = stats[row * 6 + 4], c2 = stats[row * 6 + 5];
        float row_gate = 1.f, row_slope = 0.f;
        if (d.gate_form == PAPR_GATE_ROW) gate_of<sizeof(T) == 4>((float)reinterpret_cast<const T*>(d.gate)[row * d.ldg], d.gate_act, row_gate, row_slope);
        auto four = [&](int q, int i) __attribute__((always_inline)) { return *(const float4*)&par[q][(i / 4 * G + j) * 4]; };
        // element i: y and f (standardised where there is a norm), p = N_post(f), the gate and its slope
        auto made = [&](int i, float gain, float shift, float s, float& y, float& f, float& p, float& a, float& slope) __attribute__((always_inline)) {
            y = (float)rx.t[i / V].v[i % V];
            f = (float)rf.t[i / V].v[i % V];
            a = row_gate; slope = row_slope;
            if (full) gate_of<sizeof(T) == 4>((float)rg.t[i / V].v[i % V], d.gate_act, a, slope);
            if (post) f = (f - m1) * r1;
            p = __builtin_fmaf(f, gain, shift);
            if (d.f) y = __builtin_fmaf(a * s, p, y);
            if (pre) y = (y - m2) * r2;
        };
#define PAPR_OF(t, b) ((b) == 0 ? t.x : (b) == 1 ? t.y : (b) == 2 ? t.z : t.w)
        float t2 = 0.f, m = 0.f;
        if (d_h && pre) {
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int i0 = 0; i0 < E; i0 += 4) {
                const float4 pa = four(0, i0), pb = four(1, i0), qa = four(2, i0), sc = four(3, i0);
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int i = i0 + b;
                    float y, f, p, a, slope;
                    made(i, PAPR_OF(pa, b), PAPR_OF(pb, b), PAPR_OF(sc, b), y, f, p, a, slope);
                    const float q = (float)rh.t[i / V].v[i % V] * PAPR_OF(qa, b);
                    s[0] = __builtin_fmaf(q, y, s[0]);
                    s[1] += q;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            group_sum<G, 2>(s, lds2, turn);
            t2 = s[0] * c2 * r2;
            m = d.pre.kind == PAPR_NORM_LAYER ? s[1] * rw * r2 : 0.f;
        }
        typename R::Raw ox, og;
        float dp[E], s[3] = {0.f, 0.f, 0.f};
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i0 = 0; i0 < E; i0 += 4) {
            const float4 pa = four(0, i0), pb = four(1, i0), qa = four(2, i0), sc = four(3, i0);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int i = i0 + b;
                float y, f, p, a, slope;
                made(i, PAPR_OF(pa, b), PAPR_OF(pb, b), PAPR_OF(sc, b), y, f, p, a, slope);
                const float dh = (float)rh.t[i / V].v[i % V], q = dh * PAPR_OF(qa, b);
                float g = (float)ry.t[i / V].v[i % V];
                if (d_h) {
                    acc[0][i] = __builtin_fmaf(dh, y, acc[0][i]);
                    acc[1][i] += dh;
                    g += pre ? __builtin_fmaf(q, r2, -__builtin_fmaf(y, t2, m)) : q;
                }
                ox.t[i / V].v[i % V] = (T)g;
                const float w = g * p, v = g * a * PAPR_OF(sc, b);
                acc[4][i] = __builtin_fmaf(a, w, acc[4][i]);
                const float u = PAPR_OF(sc, b) * w * slope;
                og.t[i / V].v[i % V] = (T)u;
                s[2] += u;
                acc[2][i] = __builtin_fmaf(v, f, acc[2][i]);
                acc[3][i] += v;
                dp[i] = v * PAPR_OF(pa, b);
                s[0] = __builtin_fmaf(dp[i], f, s[0]);
                s[1] += dp[i];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (d_x) put(ox, d_x + row * width);
        if (!d.f) continue;                       // (uniform)
        if (d_g && full) put(og, d_g + row * width);
        if (post || d.gate_form == PAPR_GATE_ROW) group_sum<G, 3>(s, lds, turn);
        if (d_g && !full && j == 0) d_g[row] = (T)s[2];
        if (!d_f) continue;
        const float t1 = s[0] * c1 * r1, n = d.post.kind == PAPR_NORM_LAYER ? s[1] * rw * r1 : 0.f;
        if (post)
#pragma unroll
            for (int i = 0; i < E; ++i) dp[i] = __builtin_fmaf(dp[i], r1, -__builtin_fmaf(((float)rf.t[i / V].v[i % V] - m1) * r1, t1, n));
        R::store(dp, d_f + row * width, width, j);
    }
#undef PAPR_OF
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 5 * width;
#pragma unroll
    for (int a = 0; a < 5; ++a)
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const int c = R::col(j, i);
            if (c < width) out[(int64_t)a * width + c] = acc[a][i];
        }
}

int lanes_for(int width) {
    const int need = (width + E - 1) / E;
    for (int g = 8; g <= 1024; g *= 2)
        if (g >= need) return g;
    return 0;
}

template <typename T, int V, int G>
int launch_join(const papr_join_desc& d, bool bwd, void* y, void* h, float* stats, const void* d_y, const void* d_h, void* d_x, void* d_f, void* d_g, float* part,
                int64_t blocks, hipStream_t s) {
    constexpr int THREADS = G > 256 ? G : 256;
    if (bwd) {
        if constexpr (G > 512) join_bwd_wide_kernel<T, V><<<dim3((unsigned)blocks), dim3(THREADS), 0, s>>>(d, stats, (const T*)d_y, (const T*)d_h, (T*)d_x, (T*)d_f, (T*)d_g, part);
        else join_bwd_kernel<T, V, G><<<dim3((unsigned)blocks), dim3(THREADS), 0, s>>>(d, stats, (const T*)d_y, (const T*)d_h, (T*)d_x, (T*)d_f, (T*)d_g, part);
    } else
        join_fwd_kernel<T, V, G><<<dim3((unsigned)blocks), dim3(THREADS), 0, s>>>(d, (T*)y, (T*)h, stats);
    PAPR_CHECK_LAUNCH(bwd ? "papr_join_bwd" : "papr_join_fwd");
    return 0;
}

template <typename T, int V>
int pick_join(int G, const papr_join_desc& d, bool bwd, void* y, void* h, float* stats, const void* d_y, const void* d_h, void* d_x, void* d_f, void* d_g, float* part,
              int64_t blocks, hipStream_t s) {
#define PAPR_JOIN_CASE(g) case g: return launch_join<T, V, g>(d, bwd, y, h, stats, d_y, d_h, d_x, d_f, d_g, part, blocks, s);
    switch (G) { PAPR_JOIN_CASE(8) PAPR_JOIN_CASE(16) PAPR_JOIN_CASE(32) PAPR_JOIN_CASE(64) PAPR_JOIN_CASE(128) PAPR_JOIN_CASE(256) PAPR_JOIN_CASE(512) PAPR_JOIN_CASE(1024) }
#undef PAPR_JOIN_CASE
    papr_set_error("papr_join: no kernel for %d lanes a row", G);
    return 1;
}

// Bytes of a vector that every row may be read in: 16, 4 (two 16-bit values), or one value.  (16 bytes at any address, which the hardware takes too, measured less than
// single values: 320,000 x 117 in float32 187 us forward against 151, in bf16 backward 208 against 151.)
int join_vector(const papr_join_desc& d, const void* const* more, int n_more) {
    const int b = papr_type_bytes(d.type);
    uintptr_t bits = (uintptr_t)d.x | (uintptr_t)d.f | (uintptr_t)(d.ldx * b) | (uintptr_t)(d.f ? d.ldf * b : 0) | (uintptr_t)((int64_t)d.width * b);
    if (d.gate_form == PAPR_GATE_FULL) bits |= (uintptr_t)d.gate | (uintptr_t)(d.ldg * b);
    for (int i = 0; i < n_more; ++i) bits |= (uintptr_t)more[i];
    const void* params[5] = {d.post.gain, d.post.shift, d.pre.gain, d.pre.shift, d.scale_cols};
    uintptr_t at = 0;                              // (a parameter's vector may be twice a row's: float32 beside 16-bit rows)
    for (const void* p : params) at |= (uintptr_t)p;
    return (bits & 15) == 0 && (at & 31) == 0 ? 16 : (bits & 3) == 0 && (at & 7) == 0 ? 4 : b;
}

int64_t join_blocks(const papr_join_desc& d, int G, bool bwd) {
    const int64_t rpb = G > 256 ? 1 : 256 / G, need = (d.rows + rpb - 1) / rpb;
    // (the waves that are resident at once: the backward kernel's registers allow eight a compute unit, the forward kernel's sixteen)
    const int64_t cap = (int64_t)papr_cu_count() * (G >= 512 ? (bwd ? 1 : 2) : bwd ? 2 : 4);
    return need < cap ? need : cap;
}

int join_check(const papr_join_desc* d, const char* who) {
    PAPR_REQUIRE(d, "%s: no descriptor", who);
    PAPR_REQUIRE(papr_type_ok(d->type), "%s: unknown row type %d", who, d->type);
    PAPR_REQUIRE(d->rows >= 0 && d->width >= 1 && d->width <= PAPR_JOIN_MAX_WIDTH, "%s: rows %lld, width %d (1 .. %d)", who, (long long)d->rows, d->width, PAPR_JOIN_MAX_WIDTH);
    PAPR_REQUIRE(d->gate_form >= PAPR_GATE_ABSENT && d->gate_form <= PAPR_GATE_FULL, "%s: unknown gate form %d", who, d->gate_form);
    PAPR_REQUIRE(d->gate_act >= PAPR_GATE_NONE && d->gate_act <= PAPR_GATE_SILU, "%s: unknown gate activation %d", who, d->gate_act);
    PAPR_REQUIRE(d->rows == 0 || d->x, "%s: x is missing", who);
    PAPR_REQUIRE(d->rows == 0 || (d->gate_form != PAPR_GATE_ABSENT) == (d->gate != nullptr), "%s: gate and gate_form disagree", who);
    PAPR_REQUIRE(d->gate_form == PAPR_GATE_ABSENT || d->f || d->rows == 0, "%s: a gate without the block's output f", who);
    PAPR_REQUIRE(d->rows <= 1 || (d->ldx >= d->width && (!d->f || d->ldf >= d->width) && (!d->gate || d->ldg >= (d->gate_form == PAPR_GATE_FULL ? d->width : 1))),
                 "%s: row strides %lld, %lld, %lld do not cover the rows", who, (long long)d->ldx, (long long)d->ldf, (long long)d->ldg);
    const papr_block_norm* norms[2] = {&d->post, &d->pre};
    for (const papr_block_norm* n : norms) {
        PAPR_REQUIRE(n->kind >= PAPR_NORM_NONE && n->kind <= PAPR_NORM_RMS, "%s: unknown norm %d", who, n->kind);
        PAPR_REQUIRE(n->kind != PAPR_NORM_LAYER || d->width >= 2, "%s: layernorm's unbiased deviation needs two columns", who);
        PAPR_REQUIRE(papr_type_ok(n->type), "%s: unknown parameter type %d", who, n->type);
    }
    PAPR_REQUIRE(papr_type_ok(d->scale_type), "%s: unknown scale type %d", who, d->scale_type);
    return 0;
}

__global__ __launch_bounds__(1024) void colsum_kernel(const float* __restrict__ part, int64_t n_blocks, int32_t width, int32_t n_arrays, papr_colsum_out out) {
    __shared__ float lds[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, a = blockIdx.y;
    if (!out.p[a]) return;                        // (uniform over the workgroup)
    const int c = blockIdx.x * 64 + lane;
    const int64_t step = (int64_t)n_arrays * width, per = (n_blocks + 15) / 16;
    int64_t b = wave * per, end = b + per < n_blocks ? b + per : n_blocks;
    const float* p = part + (int64_t)a * width + (c < width ? c : 0);
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (; b + 8 <= end; b += 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += p[(b + i) * step];
    for (; b < end; ++b) s[0] += p[b * step];
    lds[wave][lane] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (wave == 0 && c < width) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum += lds[w][lane];
        store_param(out.p[a], out.type[a], c, sum);
    }
}

}  // namespace

int papr_colsum_reduce(const float* part, int64_t n_blocks, int32_t width, int32_t n_arrays, const papr_colsum_out& out, hipStream_t s) {
    colsum_kernel<<<dim3((width + 63) / 64, n_arrays), dim3(1024), 0, s>>>(part, n_blocks, width, n_arrays, out);
    PAPR_CHECK_LAUNCH("papr column sums");
    return 0;
}

extern "C" int papr_join_fwd(const papr_join_desc* d, void* y, void* h, float* stats, papr_stream_t stream) {
    if (int rc = join_check(d, "papr_join_fwd")) return rc;
    if (d->rows == 0) return 0;
    PAPR_REQUIRE(y || h, "papr_join_fwd: neither y nor h is asked for");
    PAPR_REQUIRE(!y || d->f, "papr_join_fwd: y without the block's output f (it would be x)");
    PAPR_REQUIRE(((uintptr_t)stats & 3) == 0, "papr_join_fwd: the stats start on 4 bytes");
    const void* rows_out[2] = {y, h};
    const int vec = join_vector(*d, rows_out, 2);
    const int G = lanes_for(d->width);
    const int64_t blocks = join_blocks(*d, G, false);
    PAPR_TYPE_SWITCH(d->type, {
        if (vec == 16) return pick_join<T, 16 / sizeof(T)>(G, *d, false, y, h, stats, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, blocks, as_stream(stream));
        if (vec == 4 && sizeof(T) == 2) return pick_join<T, 4 / sizeof(T)>(G, *d, false, y, h, stats, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, blocks, as_stream(stream));
        return pick_join<T, 1>(G, *d, false, y, h, stats, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, blocks, as_stream(stream));
    });
}

extern "C" size_t papr_join_bwd_workspace_bytes(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    papr_join_desc d = {};
    d.rows = rows; d.width = width;
    const int G = lanes_for(width);
    return G ? (size_t)join_blocks(d, G, true) * 5 * (size_t)width * sizeof(float) : 0;
}

extern "C" int papr_join_bwd(const papr_join_desc* d, const float* stats, const void* d_y, const void* d_h, void* d_x, void* d_f, void* d_g,
                             const papr_join_grads* g, void* workspace, papr_stream_t stream) {
    if (int rc = join_check(d, "papr_join_bwd")) return rc;
    papr_colsum_out out = {};
    bool sums = false;
    if (g) {
        void* p[5] = {g->pre_gain, g->pre_shift, g->post_gain, g->post_shift, g->scale_cols};
        const int32_t t[5] = {d->pre.type, d->pre.type, d->post.type, d->post.type, d->scale_type};
        for (int i = 0; i < 5; ++i) { out.p[i] = p[i]; out.type[i] = t[i]; sums = sums || p[i]; }
    }
    PAPR_REQUIRE(!sums || d->rows == 0 || workspace, "papr_join_bwd: parameter gradients need the workspace");
    if (d->rows == 0) return sums ? papr_colsum_reduce(nullptr, 0, d->width, 5, out, as_stream(stream)) : 0;
    PAPR_REQUIRE(stats && ((uintptr_t)stats & 3) == 0, "papr_join_bwd: the forward call's stats are missing or do not start on 4 bytes");
    PAPR_REQUIRE(!sums || ((uintptr_t)workspace & 15) == 0, "papr_join_bwd: the workspace starts on 16 bytes");
    PAPR_REQUIRE(d_y || d_h, "papr_join_bwd: neither d_y nor d_h is given");
    PAPR_REQUIRE(d->f || (!d_f && !d_g), "papr_join_bwd: gradients of f or its gate without f");
    const void* rows_out[5] = {d_y, d_h, d_x, d_f, d->gate_form == PAPR_GATE_FULL ? d_g : nullptr};
    const int vec = join_vector(*d, rows_out, 5);
    const int G = lanes_for(d->width);
    const int64_t blocks = join_blocks(*d, G, true);
    float* part = sums ? (float*)workspace : nullptr;
    int rc = 0;
    PAPR_TYPE_SWITCH(d->type, {
        rc = vec == 16 ? pick_join<T, 16 / sizeof(T)>(G, *d, true, nullptr, nullptr, const_cast<float*>(stats), d_y, d_h, d_x, d_f, d_g, part, blocks, as_stream(stream))
             : vec == 4 && sizeof(T) == 2 ? pick_join<T, 4 / sizeof(T)>(G, *d, true, nullptr, nullptr, const_cast<float*>(stats), d_y, d_h, d_x, d_f, d_g, part, blocks, as_stream(stream))
             : pick_join<T, 1>(G, *d, true, nullptr, nullptr, const_cast<float*>(stats), d_y, d_h, d_x, d_f, d_g, part, blocks, as_stream(stream));
    });
    if (rc || !sums) return rc;
    return papr_colsum_reduce(part, blocks, d->width, 5, out, as_stream(stream));
}
