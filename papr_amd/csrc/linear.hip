// Linear layers over rows with their epilogue, and their backward pass, on the matrix pipe:
//     z = x W^T + b,  y = act(z) + r          d_z = d_y act'(z),  d_x = d_z W,  d_W = d_z^T x,  d_b = sum of the rows of d_z
// x (M, K), W (N, K) in float32, float16 or bfloat16; sums in float32.  One kernel, C(m, n) = sum_k A(m, k) B(n, k), serves the three products; an operand
// lies with k contiguous (x and W forward, d_z in d_x) or with its rows contiguous (W in d_x, both in d_W), or it is a set of 8-bit rows (rows8.hip: d_W).
//   * float16 / bfloat16: the values themselves are the matrix operands.
//   * float32: every value is cut into three bfloat16 parts (8 + 8 + 8 bits, rounded to nearest: exact for every normal number) on its way into LDS, and the six
//     products of weight 2^-18 and more are summed -- what is left out is below 2^-26 of a term, less than float32's own rounding.  2.5 PFLOP/s / 6 = 416 TFLOP/s
//     against 157 of the float32 matrix instructions.  Infinities and NaN give NaN (inf - inf), magnitudes above 2^128 (1 - 2^-9) count as infinite.
//   * d_z is an operand of two products and is kept in the rows' type (rounded once, to nearest): float32 for float32 rows; for 16-bit rows its rounding is of the
//     size of the gradients' own.  d_b sums it in float32 before that rounding.
#include "block_types.h"
#include <atomic>

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

// Phi(z) and phi(z) of the erf form of gelu.  float32 rows: the library's erf and exp.  16-bit rows: erfc(x) = t (a1 + ... + a5 t^4) exp(-x^2), t = 1 / (1 + p x)
// (Abramowitz and Stegun 7.1.26, 1.5e-7 absolute), a sixteenth of the rows' own rounding and a third of erf's instructions: erf in the epilogue of an
// 8192 x 1024 -> 4096 layer took longer than its matrix instructions.
template <bool EXACT>
__device__ __forceinline__ void gauss(float z, float& cdf, float& pdf) {
    if (EXACT) {
        cdf = 0.5f * erfcf(z * -0.70710678f);
        pdf = 0.39894228f * expf(-0.5f * z * z);
    } else {
        const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, x, 1.f));
        const float e = __builtin_amdgcn_exp2f(x * x * -1.44269504f);
        const float q = 0.5f * t * e * __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
        cdf = z < 0.f ? q : 1.f - q;
        pdf = 0.39894228f * e;
    }
}
// v <- act(v)
template <bool EXACT, int N>
__device__ __forceinline__ void act_values(float (&v)[N], int act) {
    if (act == PAPR_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] > 0.f ? v[i] : (v[i] == v[i] ? 0.f : v[i]);
    } else if (act == PAPR_ACT_LEAKY_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = v[i] > 0.f ? v[i] : 0.2f * v[i];
    } else if (act == PAPR_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float cdf, pdf;
            gauss<EXACT>(v[i], cdf, pdf);
            v[i] *= cdf;
        }
    } else if (act == PAPR_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= papr_sigmoid(v[i]);
    }
}
// g <- g act'(z)
template <bool EXACT, int N>
__device__ __forceinline__ void act_slopes(float (&g)[N], const float (&z)[N], int act) {
    if (act == PAPR_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = z[i] > 0.f ? g[i] : 0.f;
    } else if (act == PAPR_ACT_LEAKY_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = z[i] > 0.f ? g[i] : 0.2f * g[i];
    } else if (act == PAPR_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float cdf, pdf;
            gauss<EXACT>(z[i], cdf, pdf);
            g[i] *= __builtin_fmaf(z[i], pdf, cdf);
        }
    } else if (act == PAPR_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float p = papr_sigmoid(z[i]);
            g[i] *= p * __builtin_fmaf(z[i], 1.f - p, 1.f);
        }
    }
}

enum { K_RUNS = 0, ROWS_RUN = 1 };                // which index of an operand is contiguous in memory
enum { OUT_FORWARD = 0, OUT_ROWS = 1, OUT_SLAB = 2 };

struct Operand { const void* p; int64_t ld; int64_t rows; const uint8_t* exps; };       // exps: 8-bit rows only (ld in codes)
struct Epilogue {                                  // out and z (M, N) contiguous
    void* out;
    const void* bias; const void* res; int64_t ld_res; void* z;
    int act;
    int wide;                                      // whole 16-byte vectors in every row of out, z and res
};

template <typename T> struct Matrix { typedef bf16x8 frag; };
template <> struct Matrix<f16> { typedef f16x8 frag; };
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"      // (an LDS address is a 32-bit offset: the host pass sees a 64-bit pointer type)
__device__ __forceinline__ s16x4 read_tr4(unsigned a) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a); }
#pragma clang diagnostic pop

// One operand's tile of R rows x BK in LDS, `PLANES` of them, and the registers its next tile waits in.
//   K_RUNS:   image [R][BK] halfs, 16-byte pieces exchanged by the row number so that 16 rows' reads of one piece cover all 64 banks.
//   ROWS_RUN: image [BK][R + pad] halfs as it lies in memory; the transposing LDS read hands a lane 8 consecutive k of its row.  The row stride is
//             64 bytes modulo 256: the four k a 16-lane group reads lie on different quarters of the banks.
// FMT: 0 rows of type T, else 8-bit rows (ROWS_RUN only).  A thread's pieces sit at fixed 32-bit offsets from a uniform tile address that advances with k.
template <typename T, int LAYOUT, int FMT, bool VEC, int R, int BK, int THREADS>
struct Tile {
    static constexpr bool SPLIT = sizeof(T) == 4 && FMT == 0;
    static constexpr int PLANES = SPLIT ? 3 : 1;
    static constexpr int PIECE = SPLIT ? 4 : 8;                                   // elements of one load
    static constexpr int BYTES = FMT ? 1 : sizeof(T);
    static constexpr int N = R * BK / PIECE / THREADS;
    static constexpr int STRIDE = LAYOUT == K_RUNS ? BK : (R * 2 % 256 == 64 ? R : R + 32);
    static constexpr int PLANE = (LAYOUT == K_RUNS ? R : BK) * STRIDE;            // halfs
    static constexpr int HALFS = PLANES * PLANE;
    static_assert(R * BK % (PIECE * THREADS) == 0, "whole pieces per thread");
    typedef typename Matrix<T>::frag frag;

    uint4 reg[N];
    unsigned off[N];                                                              // bytes from the tile's address
    uint8_t ex[FMT ? N : 1];
    unsigned exo[FMT ? N : 1];
    const char* base;                                                             // (uniform) rows r0, the next k
    const uint8_t* exb;
    int64_t ld;

    // piece q of this thread: (row, k) of its first element inside the tile
    static __device__ __forceinline__ void where(int q, int& r, int& k) {
        const int id = q * THREADS + threadIdx.x;
        if (LAYOUT == K_RUNS) { r = id / (BK / PIECE); k = id % (BK / PIECE) * PIECE; }
        else { k = id / (R / PIECE); r = id % (R / PIECE) * PIECE; }
    }
    // swizzled place of 16-byte piece c of row r (halfs)
    static __device__ __forceinline__ int place(int r, int c) {
        const int sw = BK == 64 ? (r >> 1) & 7 : BK == 32 ? (r >> 2) & 3 : (r >> 3) & 1;
        return r * STRIDE + ((c ^ sw) << 3);
    }

    __device__ __forceinline__ void start(const Operand& o, int64_t r0, int64_t k0) {
        ld = o.ld;
        base = reinterpret_cast<const char*>(o.p) + (LAYOUT == K_RUNS ? r0 * ld + k0 : k0 * ld + r0) * BYTES;
        if (FMT) exb = o.exps + k0 * (ld >> 5) + (r0 >> 5);
        const int64_t left = (FMT ? ld : o.rows) - r0;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            if (r >= left) r = LAYOUT == K_RUNS ? (int)left - 1 : 0;              // (rows past the end: some row of the operand, its results are never stored)
            off[q] = (unsigned)((LAYOUT == K_RUNS ? (int64_t)r * ld + k : (int64_t)k * ld + r) * BYTES);
            if (FMT) exo[q] = (unsigned)(k * (ld >> 5) + (r >> 5));
        }
    }
    // the next tile: k0 .. k0 + BK of K terms.  `inside`: every piece may be read whole.  A piece that crosses the end of a contiguous row of rows reads the start
    // of the next one (those rows of the product are never stored), but behind the last k there is no next one.
    __device__ __forceinline__ void load(const Operand& o, int64_t r0, int64_t k0, int64_t K) {
        bool inside = k0 + BK <= K;
        if (LAYOUT == ROWS_RUN && !VEC && FMT == 0) inside = k0 + BK < K && o.rows >= PIECE;
        if (inside) {
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const char* src = base + off[q];
                if (FMT) {
                    const uint2 c = *reinterpret_cast<const uint2*>(src);
                    reg[q].x = c.x; reg[q].y = c.y;
                    ex[q] = exb[exo[q]];
                } else if (VEC) reg[q] = *reinterpret_cast<const uint4*>(src);
                else __builtin_memcpy(&reg[q], __builtin_assume_aligned(src, sizeof(T)), 16);
            }
        } else {
#pragma unroll
            for (int q = 0; q < N; ++q) {
                int r, k;
                where(q, r, k);
                const bool in = k0 + k < K;
                const char* src = in ? base + off[q] : base;                      // (base: rows r0, the tile's first k < K)
                if (FMT) {
                    const uint2 c = *reinterpret_cast<const uint2*>(src);
                    reg[q].x = in ? c.x : 0u; reg[q].y = in ? c.y : 0u;
                    ex[q] = exb[in ? exo[q] : 0u];
                } else if (VEC) {
                    const uint4 t = *reinterpret_cast<const uint4*>(src);
                    reg[q].x = in ? t.x : 0u; reg[q].y = in ? t.y : 0u; reg[q].z = in ? t.z : 0u; reg[q].w = in ? t.w : 0u;
                } else {
                    papr_pack<T, PIECE> t;
                    if (LAYOUT == ROWS_RUN && r0 + r >= o.rows) r = 0;
#pragma unroll
                    for (int i = 0; i < PIECE; ++i) {
                        const bool ok = LAYOUT == K_RUNS ? k0 + k + i < K : in && r0 + r + i < o.rows;
                        t.v[i] = ok ? reinterpret_cast<const T*>(src)[i] : (T)0.f;
                    }
                    __builtin_memcpy(&reg[q], &t, 16);
                }
            }
        }
        base += (LAYOUT == K_RUNS ? (int64_t)BK : BK * ld) * BYTES;
        if (FMT) exb += BK * (ld >> 5);
    }

    __device__ __forceinline__ void store(short* lds) const {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            const int at = LAYOUT == K_RUNS ? place(r, k >> 3) + (k & 7) : k * STRIDE + r;
            if (FMT) {
                float v[4], w[4];
                const float scale = __uint_as_float((unsigned)ex[q] << 23);
                papr_codes_to_float<FMT>(reg[q].x, scale, v);
                papr_codes_to_float<FMT>(reg[q].y, scale, w);
                frag h;
#pragma unroll
                for (int i = 0; i < 4; ++i) { h[i] = v[i]; h[4 + i] = w[i]; }     // (exact: at most 8 significant bits)
                *reinterpret_cast<frag*>(lds + at) = h;
            } else if (SPLIT) {
                const float f[4] = {__uint_as_float(reg[q].x), __uint_as_float(reg[q].y), __uint_as_float(reg[q].z), __uint_as_float(reg[q].w)};
                papr_pack<bf16, 4> p[3];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[0].v[i] = (bf16)f[i];
                    const float rest = f[i] - (float)p[0].v[i];
                    p[1].v[i] = (bf16)rest;
                    p[2].v[i] = (bf16)(rest - (float)p[1].v[i]);
                }
#pragma unroll
                for (int n = 0; n < PLANES; ++n) *reinterpret_cast<papr_pack<bf16, 4>*>(lds + n * PLANE + at) = p[n];
            } else *reinterpret_cast<uint4*>(lds + at) = reg[q];
        }
    }

    // this lane's operand of the 16-term step ks: row base + (lane & 31), k = 8 (lane >> 5) + 0 .. 7
    static __device__ __forceinline__ frag read(const short* lds, int plane, int row, int ks) {
        const int lane = threadIdx.x & 63;
        s16x8 v;
        if (LAYOUT == K_RUNS) {
            v = *reinterpret_cast<const s16x8*>(lds + plane * PLANE + place(row + (lane & 31), ks * 2 + (lane >> 5)));
        } else {
            const unsigned a = (unsigned)(size_t)(lds + plane * PLANE) +
                               2u * (unsigned)((ks * 16 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * STRIDE + row + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
            const s16x4 lo = read_tr4(a), hi = read_tr4(a + 8 * STRIDE);
            v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return __builtin_bit_cast(frag, v);
    }
};

// Workgroup -> (row tile, column tile, part of the sum).  Workgroups go to the eight XCDs in turn: each takes a contiguous run of tiles, and the run walks
// GROUP row tiles down before it steps to the next column tile, so that an XCD's workgroups of one moment share operand tiles in its L2.
struct Place { int m, n, part; };
__device__ __forceinline__ Place place_of(unsigned id, unsigned total, unsigned tm, unsigned tn) {
    constexpr unsigned XCDS = 8, GROUP = 8;
    const unsigned x = id % XCDS, q = id / XCDS, per = total / XCDS, rem = total % XCDS;
    const unsigned t = x * per + (x < rem ? x : rem) + q;
    Place p;
    p.part = (int)(t / (tm * tn));
    const unsigned r = t % (tm * tn), g = r / (GROUP * tn), in = r % (GROUP * tn), high = tm - g * GROUP < GROUP ? tm - g * GROUP : GROUP;
    p.m = (int)(g * GROUP + in % high);
    p.n = (int)(in / high);
    return p;
}

// Tile shapes: waves WM x WN, each IM x IN blocks of 32 x 32.
template <int WM_, int WN_, int IM_, int IN_>
struct Shape {
    static constexpr int WM = WM_, WN = WN_, IM = IM_, IN = IN_, THREADS = 64 * WM * WN, TM = WM * IM * 32, TN = WN * IN * 32;
};

template <typename T, int LA, int LB, int FMT, bool VEC, typename S>
struct Plan {
    static constexpr int BK = sizeof(T) == 2 ? 64 : S::TM > 64 ? 16 : 32;       // (divides step_of)
    typedef Tile<T, LA, 0, VEC, S::TM, BK, S::THREADS> TA;
    typedef Tile<T, LB, FMT, VEC, S::TN, BK, S::THREADS> TB;
    static constexpr int BUF = TA::HALFS + TB::HALFS;
    static constexpr int EPI_STRIDE = S::IN * 32 + 8;                             // floats: rows four apart lie on the other half of the banks
    static constexpr size_t EPI = (size_t)S::WM * S::WN * 32 * EPI_STRIDE * 4, LOOP = (size_t)2 * BUF * 2;
    static constexpr size_t LDS = EPI > LOOP ? EPI : LOOP;
};

// E consecutive results of row m from column n on
template <typename T, int OUT, int E>
__device__ __forceinline__ void finish(float (&v)[E], int64_t m, int64_t n, int64_t N, const float (&bias)[E], const papr_pack<T, E>& res, const Epilogue& ep) {
    if (OUT == OUT_FORWARD) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] += bias[i];
        if (ep.z) {
            papr_pack<T, E> t;
#pragma unroll
            for (int i = 0; i < E; ++i) t.v[i] = (T)v[i];
            *reinterpret_cast<papr_pack<T, E>*>(reinterpret_cast<T*>(ep.z) + m * N + n) = t;
        }
        act_values<sizeof(T) == 4>(v, ep.act);
        if (ep.res)
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += (float)res.v[i];
    }
    papr_pack<T, E> t;
#pragma unroll
    for (int i = 0; i < E; ++i) t.v[i] = (T)v[i];
    *reinterpret_cast<papr_pack<T, E>*>(reinterpret_cast<T*>(ep.out) + m * N + n) = t;
}

template <typename T, int LA, int LB, int FMT, bool VEC, int OUT, typename S>
__global__ __launch_bounds__(S::THREADS, 2) void product_kernel(Operand A, Operand B, int64_t K, int64_t k_per_part, unsigned tiles_m, unsigned tiles_n, Epilogue ep) {
    typedef Plan<T, LA, LB, FMT, VEC, S> P;
    typedef typename P::TA TA;
    typedef typename P::TB TB;
    constexpr int IM = S::IM, IN = S::IN, BK = P::BK;
    extern __shared__ __attribute__((aligned(16))) short smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
    const Place at = place_of(blockIdx.x, gridDim.x, tiles_m, tiles_n);
    const int64_t m0 = (int64_t)at.m * S::TM, n0 = (int64_t)at.n * S::TN;
    const int64_t kb = at.part * k_per_part, ke = kb + k_per_part < K ? kb + k_per_part : K;
    f32x16 acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    TA a;
    TB b;
    a.start(A, m0, kb);
    b.start(B, n0, kb);
    a.load(A, m0, kb, K);
    b.load(B, n0, kb, K);
    a.store(smem);
    b.store(smem + TA::HALFS);
    __syncthreads();
    int buf = 0;
    for (int64_t k0 = kb; k0 < ke; k0 += BK, buf ^= 1) {
        const bool more = k0 + BK < ke;
        if (more) {
            a.load(A, m0, k0 + BK, K);
            b.load(B, n0, k0 + BK, K);
        }
        const short *la = smem + buf * P::BUF, *lb = la + TA::HALFS;
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            typename TA::frag fa[TA::PLANES][IM];
            typename TB::frag fb[TB::PLANES][IN];
#pragma unroll
            for (int p = 0; p < TA::PLANES; ++p)
#pragma unroll
                for (int i = 0; i < IM; ++i) fa[p][i] = TA::read(la, p, (wm * IM + i) * 32, ks);
#pragma unroll
            for (int p = 0; p < TB::PLANES; ++p)
#pragma unroll
                for (int j = 0; j < IN; ++j) fb[p][j] = TB::read(lb, p, (wn * IN + j) * 32, ks);
#pragma unroll
            for (int p = 0; p < TA::PLANES; ++p)
#pragma unroll
                for (int q = 0; q < TB::PLANES; ++q)
                    if (p + q < 3)                // (the parts' products below 2^-26 are left out)
#pragma unroll
                        for (int i = 0; i < IM; ++i)
#pragma unroll
                            for (int j = 0; j < IN; ++j) acc[i][j] = mfma(fa[p][i], fb[q][j], acc[i][j]);
        }
        if (more) {
            a.store(smem + (buf ^ 1) * P::BUF);
            b.store(smem + (buf ^ 1) * P::BUF + TA::HALFS);
        }
        __syncthreads();
    }
    const int64_t M = A.rows, N = B.rows;
    if (OUT == OUT_SLAB) {
        // float32, as it lies: a lane holds column lane & 31 of a 32 x 32 block, rows (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
        float* out = reinterpret_cast<float*>(ep.out) + (int64_t)at.part * M * N;
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const int64_t n = n0 + (wn * IN + j) * 32 + (lane & 31);
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int64_t m = m0 + (wm * IM + i) * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
                    if (n < N && m < M) out[m * N + n] = acc[i][j][e];
                }
        }
        return;
    }
    // Through LDS, 32 rows of the wave's own at a time (no barrier), so that a lane takes 16 bytes of a row: 16-byte loads and stores of whole lines.  Rows that do not
    // start on 16 bytes: a lane takes single columns, 64 (32) lanes a row.
    float* epi = reinterpret_cast<float*>(smem) + wave * 32 * P::EPI_STRIDE;
    constexpr int COLS = IN * 32, E = 16 / sizeof(T), LPR = COLS / E, RPP = 64 / LPR;
    const int64_t nw = n0 + wn * COLS;
    const bool wide = ep.wide;
    const int64_t n = nw + (wide ? lane % LPR * E : lane % COLS);
    float bias[E];
#pragma unroll
    for (int i = 0; i < E; ++i) bias[i] = 0.f;
    if (OUT == OUT_FORWARD && ep.bias && n < N) {
        const T* src = reinterpret_cast<const T*>(ep.bias) + n;
        if (wide) {
#pragma unroll
            for (int i = 0; i < E; ++i) bias[i] = (float)src[i];
        } else bias[0] = (float)src[0];
    }
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int64_t mw = m0 + (wm * IM + i) * 32;
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) epi[((e & 3) + 8 * (e >> 2) + 4 * (lane >> 5)) * P::EPI_STRIDE + j * 32 + (lane & 31)] = acc[i][j][e];
        if (wide) {
            papr_pack<T, E> res[32 / RPP];
#pragma unroll
            for (int r = 0; r < 32 / RPP; ++r) {
                const int64_t m = mw + r * RPP + lane / LPR;
                if (OUT == OUT_FORWARD && ep.res && m < M && n < N) res[r] = *reinterpret_cast<const papr_pack<T, E>*>(reinterpret_cast<const T*>(ep.res) + m * ep.ld_res + n);
            }
#pragma unroll
            for (int r = 0; r < 32 / RPP; ++r) {
                const int64_t m = mw + r * RPP + lane / LPR;
                float v[E];
#pragma unroll
                for (int c = 0; c < E; c += 4) {
                    const float4 t = *reinterpret_cast<const float4*>(epi + (r * RPP + lane / LPR) * P::EPI_STRIDE + lane % LPR * E + c);
                    v[c] = t.x; v[c + 1] = t.y; v[c + 2] = t.z; v[c + 3] = t.w;
                }
                if (m < M && n < N) finish<T, OUT, E>(v, m, n, N, bias, res[r], ep);
            }
        } else {
            constexpr int ROWS = 64 / COLS;
#pragma unroll 4
            for (int r = 0; r < 32; r += ROWS) {
                const int64_t m = mw + r + lane / COLS;
                float v[1] = {epi[(r + lane / COLS) * P::EPI_STRIDE + lane % COLS]};
                const float b1[1] = {bias[0]};
                if (m < M && n < N) {
                    papr_pack<T, 1> res;
                    if (OUT == OUT_FORWARD && ep.res) res.v[0] = reinterpret_cast<const T*>(ep.res)[m * ep.ld_res + n];
                    finish<T, OUT, 1>(v, m, n, N, b1, res, ep);
                }
            }
        }
    }
}

// The slabs of a sum in parts: a workgroup takes 64 results, its four waves a quarter of the parts each, quarters added in order.
template <typename T>
__global__ __launch_bounds__(256) void join_slabs_kernel(const float* __restrict__ slab, int64_t n, int parts, T* __restrict__ out) {
    __shared__ float lds[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (parts + 3) / 4;
    for (int64_t i0 = (int64_t)blockIdx.x * 64; i0 < n; i0 += (int64_t)gridDim.x * 64) {
        const int64_t i = i0 + lane < n ? i0 + lane : n - 1;
        const int end = (wave + 1) * per < parts ? (wave + 1) * per : parts;
        float s = 0.f;
#pragma unroll 8
        for (int k = wave * per; k < end; ++k) s += slab[k * n + i];
        lds[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && i0 + lane < n) out[i] = (T)((lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]));
        __syncthreads();
    }
}

// d_z = d_y act'(z) in the rows' type (none: d_y as it is, nothing is written) and the column sums of it in float32, one partial row per workgroup.
// A thread holds PIECE columns; the threads of a workgroup beyond one row's take further rows.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ d_y, int64_t ld, const T* __restrict__ z, int64_t M, int N, int act, int lanes, T* __restrict__ d_z,
                                                    float* __restrict__ part, int64_t rows_per_block) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    __shared__ float fold[256 * V];
    const int per = 256 / lanes, cg = threadIdx.x % lanes, rl = threadIdx.x / lanes;
    const int c = (blockIdx.y * lanes + cg) * V;
    const int64_t beg = (int64_t)blockIdx.x * rows_per_block, end = beg + rows_per_block < M ? beg + rows_per_block : M;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    if (c < N)
#pragma unroll 4
        for (int64_t m = beg + rl; m < end; m += per) {
            auto g = *reinterpret_cast<const papr_pack<T, V>*>(d_y + m * ld + c);
            if (d_z) {
                const auto t = *reinterpret_cast<const papr_pack<T, V>*>(z + m * N + c);
                float v[V], zv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) { v[i] = (float)g.v[i]; zv[i] = (float)t.v[i]; }
                act_slopes<sizeof(T) == 4>(v, zv, act);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum[i] += v[i];
                    g.v[i] = (T)v[i];
                }
                *reinterpret_cast<papr_pack<T, V>*>(d_z + m * N + c) = g;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += (float)g.v[i];
            }
        }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) fold[threadIdx.x * V + i] = sum[i];
    __syncthreads();
    for (int q = threadIdx.x; q < lanes * V; q += 256) {
        const int col = blockIdx.y * lanes * V + q;
        float s = 0.f;
        for (int k = 0; k < per; ++k) s += fold[k * lanes * V + q];
        if (col < N) part[(int64_t)blockIdx.x * N + col] = s;
    }
}

typedef Shape<2, 4, 4, 2> Large;                   // 256 x 256, eight waves
typedef Shape<2, 2, 2, 2> Middle;                  // 128 x 128, four waves
typedef Shape<2, 2, 1, 1> Small;                   // 64 x 64, four waves

// Which tile, and into how many parts the sum is cut: the least estimated time.  A tile's time is its area times the steps of its part over the rate its shape
// reaches, the launch as many of them in turn as a compute unit gets; parts cost their slabs' way to memory and back.
struct Choice { int shape; int64_t parts, per; };      // per: terms of a part
int step_of(int type) { return type == PAPR_TYPE_F32 ? 32 : 64; }
Choice choose(int64_t M, int64_t N, int64_t K, int type, bool may_split) {
    const int bk = step_of(type);
    const int64_t cus = papr_cu_count(), steps = (K + bk - 1) / bk;
    static const int side[3] = {256, 128, 64}, resident[3] = {1, 2, 4};
    static const double rate[3] = {1.0, 0.8, 0.45};
    Choice best = {0, 1, 0};
    double least = 0;
    for (int s = 0; s < 3; ++s) {
        const int64_t tiles = ((M + side[s] - 1) / side[s]) * ((N + side[s] - 1) / side[s]), slots = cus * resident[s];
        int64_t tried[3] = {1, slots / tiles, 2 * slots / tiles};
        for (int64_t parts : tried) {
            if (parts > steps / 4) parts = steps / 4;
            if (parts > 1024) parts = 1024;
            if (parts < 1 || !may_split) parts = 1;
            const int64_t per = (steps + parts - 1) / parts;
            parts = (steps + per - 1) / per;
            const int64_t turns = (tiles * parts + slots - 1) / slots;
            // (in matrix instruction time of one compute unit: 4096 products of a 16-bit type a cycle; slabs at 2 KB a cycle over the chip; 3 us a launch)
            double t = (double)turns * resident[s] * ((double)side[s] * side[s] * (per + 3) * bk / (4096 * rate[s]));
            if (parts > 1) t += 2.0 * parts * M * N * 4 / 2048 + 7000;
            if (least == 0 || t < least) { least = t; best = {s, parts, per * bk}; }
        }
    }
    return best;
}

template <typename T, int LA, int LB, int FMT, bool VEC, int OUT, typename S>
int launch_shape(const Operand& A, const Operand& B, int64_t K, const Choice& c, const Epilogue& ep, hipStream_t s) {
    typedef Plan<T, LA, LB, FMT, VEC, S> P;
    static_assert(P::LDS <= 160 * 1024, "a compute unit's LDS");
    auto kernel = product_kernel<T, LA, LB, FMT, VEC, OUT, S>;
    static_assert(32 % P::BK == 0 || 64 % P::BK == 0, "parts are whole steps");
    const int64_t tm = (A.rows + S::TM - 1) / S::TM, tn = (B.rows + S::TN - 1) / S::TN, grid = tm * tn * c.parts;
    PAPR_REQUIRE(grid < (int64_t)1 << 31, "papr_linear: %lld tiles", (long long)grid);
    static std::atomic<uint64_t> ready{0};            // (devices on which this kernel may already use more than 64 KB of LDS)
    int dev = 0;
    (void)hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (P::LDS > 65536 && !(ready.load(std::memory_order_relaxed) & bit)) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)P::LDS);
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    kernel<<<dim3((unsigned)grid), dim3(S::THREADS), P::LDS, s>>>(A, B, K, c.per, (unsigned)tm, (unsigned)tn, ep);
    PAPR_CHECK_LAUNCH("papr_linear product");
    return 0;
}

template <typename T, int LA, int LB, int FMT, int OUT>
int launch_product(const Choice& c, bool vec, const Operand& A, const Operand& B, int64_t K, const Epilogue& ep, hipStream_t s) {
    if (c.shape == 0) return vec ? launch_shape<T, LA, LB, FMT, true, OUT, Large>(A, B, K, c, ep, s) : launch_shape<T, LA, LB, FMT, false, OUT, Large>(A, B, K, c, ep, s);
    if (c.shape == 1) return vec ? launch_shape<T, LA, LB, FMT, true, OUT, Middle>(A, B, K, c, ep, s) : launch_shape<T, LA, LB, FMT, false, OUT, Middle>(A, B, K, c, ep, s);
    return vec ? launch_shape<T, LA, LB, FMT, true, OUT, Small>(A, B, K, c, ep, s) : launch_shape<T, LA, LB, FMT, false, OUT, Small>(A, B, K, c, ep, s);
}

// C = A B^T into contiguous rows of type T, the sum in parts where the tiles alone do not fill the chip
template <typename T, int LA, int LB, int FMT>
int rows_product(bool vec, const Operand& A, const Operand& B, int64_t K, void* out, float* slab, hipStream_t s) {
    const Choice c = choose(A.rows, B.rows, K, sizeof(T) == 4 ? PAPR_TYPE_F32 : PAPR_TYPE_F16, true);
    Epilogue ep = {};
    if (c.parts == 1) {
        ep.out = out;
        ep.wide = ((uintptr_t)out & 15) == 0 && (B.rows * sizeof(T)) % 16 == 0;
        return launch_product<T, LA, LB, FMT, OUT_ROWS>(c, vec, A, B, K, ep, s);
    }
    ep.out = slab;
    if (int rc = launch_product<T, LA, LB, FMT, OUT_SLAB>(c, vec, A, B, K, ep, s)) return rc;
    const int64_t n = A.rows * B.rows, need = (n + 63) / 64, cap = (int64_t)papr_cu_count() * 16;
    join_slabs_kernel<T><<<dim3((unsigned)(need < cap ? need : cap)), dim3(256), 0, s>>>(slab, n, (int)c.parts, (T*)out);
    PAPR_CHECK_LAUNCH("papr_linear slabs");
    return 0;
}

// float32 slabs of one product
size_t slab_floats(int type, int64_t M, int64_t N, int64_t K) {
    const int64_t parts = choose(M, N, K, type, true).parts;
    return parts > 1 ? (size_t)(parts * M * N) : 0;
}

struct SlopeGrid { int lanes; int64_t blocks, rows_per_block; unsigned cols; };
SlopeGrid slope_grid(int64_t M, int N, int piece) {
    SlopeGrid g;
    const int groups = (N + piece - 1) / piece;
    g.lanes = 1;
    while (g.lanes < groups && g.lanes < 256) g.lanes *= 2;
    g.cols = (unsigned)((groups + g.lanes - 1) / g.lanes);
    const int64_t per = 256 / g.lanes;
    int64_t blocks = (M + 8 * per - 1) / (8 * per), cap = (int64_t)papr_cu_count() * 8 / g.cols;
    if (cap < 1) cap = 1;
    if (blocks > cap) blocks = cap;
    g.rows_per_block = (M + blocks - 1) / blocks;
    g.blocks = (M + g.rows_per_block - 1) / g.rows_per_block;
    return g;
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

int linear_check(const char* who, int type, int64_t M, int64_t N, int64_t K, int act) {
    PAPR_REQUIRE(papr_type_ok(type), "%s: unknown row type %d", who, type);
    PAPR_REQUIRE(M >= 0 && N >= 1 && K >= 1 && N <= (1 << 20) && K <= (1 << 20), "%s: M %lld, N %lld, K %lld", who, (long long)M, (long long)N, (long long)K);
    PAPR_REQUIRE(M < (int64_t)1 << 31, "%s: %lld rows", who, (long long)M);
    PAPR_REQUIRE(act >= PAPR_ACT_NONE && act <= PAPR_ACT_SILU, "%s: unknown activation %d", who, act);
    return 0;
}

}  // namespace

extern "C" int papr_linear_fwd(const papr_linear_desc* d, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ld_res,
                               void* y, void* z, papr_stream_t stream) {
    PAPR_REQUIRE(d, "papr_linear_fwd: no descriptor");
    if (int rc = linear_check("papr_linear_fwd", d->type, d->M, d->N, d->K, d->act)) return rc;
    if (d->M == 0) return 0;
    PAPR_REQUIRE(x && w && y, "papr_linear_fwd: a pointer is missing");
    const int b = papr_type_bytes(d->type);
    const bool vec = papr_rows_aligned(x, ldx, d->K, b) && papr_rows_aligned(w, ldw, d->K, b);
    const Operand A = {x, ldx, d->M, nullptr}, B = {w, ldw, d->N, nullptr};
    const Epilogue ep = {y, bias, res, ld_res, z, d->act,
                         papr_rows_aligned(y, d->N, d->N, b) && (!z || ((uintptr_t)z & 15) == 0) && (!res || papr_rows_aligned(res, ld_res, d->N, b))};
    const Choice c = choose(d->M, d->N, d->K, d->type, false);
    PAPR_TYPE_SWITCH(d->type, return (launch_product<T, K_RUNS, K_RUNS, 0, OUT_FORWARD>(c, vec, A, B, d->K, ep, as_stream(stream))));
}

extern "C" size_t papr_linear_bwd_workspace_bytes(const papr_linear_desc* d) {
    if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0 || !papr_type_ok(d->type)) return 0;
    const size_t dz = d->act == PAPR_ACT_NONE ? 0 : up16((size_t)d->M * d->N * papr_type_bytes(d->type));
    size_t part = 0;
    for (int piece = 1; piece <= 8; piece *= 2) {
        const size_t p = (size_t)slope_grid(d->M, (int)d->N, piece).blocks * d->N * sizeof(float);
        part = p > part ? p : part;
    }
    const size_t sx = slab_floats(d->type, d->M, d->K, d->N), sw = slab_floats(d->type, d->N, d->K, d->M);
    return dz + up16(part) + (sx > sw ? sx : sw) * sizeof(float);
}

extern "C" int papr_linear_bwd(const papr_linear_desc* d, const void* d_y, int64_t ld_dy, const void* z, const void* x, int64_t ldx, const void* exps, const void* w, int64_t ldw,
                               void* d_x, void* d_w, void* d_b, void* workspace, papr_stream_t stream) {
    PAPR_REQUIRE(d, "papr_linear_bwd: no descriptor");
    if (int rc = linear_check("papr_linear_bwd", d->type, d->M, d->N, d->K, d->act)) return rc;
    PAPR_REQUIRE(d->keep == 0 || d->keep == PAPR_KEEP_E4M3 || d->keep == PAPR_KEEP_INT8, "papr_linear_bwd: unknown format %d of the kept rows", d->keep);
    const int64_t M = d->M, N = d->N, K = d->K;
    hipStream_t s = as_stream(stream);
    PAPR_REQUIRE(M > 0, "papr_linear_bwd: no rows (the gradients of the weight and the bias are zero: the caller's)");
    PAPR_REQUIRE(d_y && workspace && (d->act == PAPR_ACT_NONE || z), "papr_linear_bwd: a pointer is missing");
    PAPR_REQUIRE(!d_x || w, "papr_linear_bwd: d_x needs the weight");
    PAPR_REQUIRE(!d_w || (x && (!d->keep || exps)), "papr_linear_bwd: d_w needs the rows");
    const int b = papr_type_bytes(d->type);
    const bool slope = d->act != PAPR_ACT_NONE;
    char* ws = reinterpret_cast<char*>(workspace);
    void* dz = slope ? ws : nullptr;
    if (slope) ws += up16((size_t)M * N * b);
    float* part = reinterpret_cast<float*>(ws);
    if (slope || d_b) {
        const bool vec = papr_rows_aligned(d_y, ld_dy, N, b) && ((uintptr_t)z & 15) == 0;
        const SlopeGrid g = slope_grid(M, (int)N, vec ? 16 / b : 1);
        const dim3 grid((unsigned)g.blocks, g.cols);
        PAPR_TYPE_SWITCH(d->type, {
            if (vec) slope_kernel<T, true><<<grid, 256, 0, s>>>((const T*)d_y, ld_dy, (const T*)z, M, (int)N, d->act, g.lanes, (T*)dz, d_b ? part : nullptr, g.rows_per_block);
            else slope_kernel<T, false><<<grid, 256, 0, s>>>((const T*)d_y, ld_dy, (const T*)z, M, (int)N, d->act, g.lanes, (T*)dz, d_b ? part : nullptr, g.rows_per_block);
        });
        PAPR_CHECK_LAUNCH("papr_linear_bwd");
        if (d_b) {
            papr_colsum_out out = {};
            out.p[0] = d_b;
            out.type[0] = d->type;
            if (int rc = papr_colsum_reduce(part, g.blocks, (int)N, 1, out, s)) return rc;
        }
    }
    size_t most = 0;
    for (int piece = 1; piece <= 8; piece *= 2) {
        const size_t p = (size_t)slope_grid(M, (int)N, piece).blocks * N * sizeof(float);
        most = p > most ? p : most;
    }
    float* slab = reinterpret_cast<float*>(ws + up16(most));
    const void* g = slope ? dz : d_y;
    const int64_t ldg = slope ? N : ld_dy;
    const bool vg = papr_rows_aligned(g, ldg, N, b);
    if (d_x) {
        const Operand A = {g, ldg, M, nullptr}, B = {w, ldw, K, nullptr};
        const bool vec = vg && papr_rows_aligned(w, ldw, K, b);
        int rc = 0;
        PAPR_TYPE_SWITCH(d->type, rc = (rows_product<T, K_RUNS, ROWS_RUN, 0>(vec, A, B, N, d_x, slab, s)));
        if (rc) return rc;
    }
    if (d_w) {
        const Operand A = {g, ldg, N, nullptr}, B = {x, ldx, K, (const uint8_t*)exps};
        const bool vec = vg && (d->keep || papr_rows_aligned(x, ldx, K, b));
        int rc = 0;
        PAPR_TYPE_SWITCH(d->type, {
            if (d->keep == PAPR_KEEP_E4M3) rc = rows_product<T, ROWS_RUN, ROWS_RUN, PAPR_KEEP_E4M3>(vec, A, B, M, d_w, slab, s);
            else if (d->keep == PAPR_KEEP_INT8) rc = rows_product<T, ROWS_RUN, ROWS_RUN, PAPR_KEEP_INT8>(vec, A, B, M, d_w, slab, s);
            else rc = rows_product<T, ROWS_RUN, ROWS_RUN, 0>(vec, A, B, M, d_w, slab, s);
        });
        if (rc) return rc;
    }
    return 0;
}
