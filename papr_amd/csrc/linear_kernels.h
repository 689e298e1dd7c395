// Linear layers over rows with their epilogue, and their backward pass, on the matrix pipe:
//     z = x W^T + b,  y = act(z) + r          d_z = d_y act'(z),  d_x = d_z W,  d_W = d_z^T x,  d_b = sum of the rows of d_z
// x (M, K), W (N, K) in float32, float16 or bfloat16; sums in float32.  One kernel, C(m, n) = sum_k A(m, k) B(n, k), serves the three products; an operand
// lies with k contiguous (x and W forward, d_z in d_x) or with its rows contiguous (W in d_x, both in d_W), or it is a set of 8-bit rows (rows8.hip: d_W).
//   * float16 / bfloat16: the values themselves are the matrix operands.
//   * float32: every value is cut into three bfloat16 parts (8 + 8 + 8 bits, rounded to nearest, the first kept finite: exact for every magnitude of 2^-109 and more, below that
//     off by 2^-134 at most, bfloat16's smallest half step) on its way into LDS, and six of the nine products are summed.  The parts are at most 1, 2^-8 and 2^-17 of a value, so
//     what is left out (second times third, twice, and third times third) is at most 2^-24 of a term: float32's own rounding.  Summed from the small products up: the first two
//     parts of the largest number alone add to 2^128, which is infinite.  2.5 PFLOP/s / 6 = 416 TFLOP/s against 157 of the float32 matrix instructions.  The third part of an
//     infinity is NaN, and so are its products: a result that is NaN is summed again from the values themselves (sum_again).
//   * z is kept for the backward pass, which makes a slope of it and nothing else, in the bytes of the rows' type.  A slope moves by at most 0.8 of z's rounding: bfloat16 rows hold gelu's
//     and silu's z in float16, an eighth of bfloat16's step (its smaller range costs nothing: beyond 65,504 the slopes are their limits, below 2^-14 they move by 2^-25); relu and
//     leakyrelu look at the sign alone, which float16 loses below 2^-25.
//   * d_z is an operand of two products.  For 16-bit rows with an activation that bends it (leakyrelu, gelu, silu) it is kept as the sum of two values of the rows' type, high
//     and low (16 significant bits or more), and both products take both: rounded to one such value it would be an error of the gradients' own rounding's size in each
//     of them (measured 1.45 times that rounding together; so 1.05 in float16 and 1.00 in bfloat16, which is z's part), and a slope up to 1.13 can take it past float16's largest number.  Twice the matrix instructions: 8192 x 1024
//     -> 4096 in bfloat16, forward and backward, 450 us; with d_z rounded once it was 332.
//     d_b sums it in float32.
#pragma once
#include "linear.h"
#include <atomic>
#include <type_traits>

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace papr_linear {

template <typename T> __device__ __forceinline__ float largest() { return __is_same(T, f16) ? 65504.f : 3.38953139e38f; }      // of the 16-bit types

// Phi(z) and phi(z) of the erf form of gelu.  float32 rows: the library's erf and exp.  16-bit rows: erfc(x) = t P(t) exp(-x^2), t = 1 / (1 + 0.375 x), P of
// degree 6 fitted for the least relative error over 0 <= x <= 9.6 (6.4e-7; with float32's steps 1.4e-6 to |z| = 3, 7.4e-6 to 9, most of it x^2's rounding in the exponent): relative, since
// a negative z's value is z times it, and at most a 60th of float16's own rounding.  A third of erf's instructions: erf in the epilogue of an 8192 x 1024 -> 4096 layer took longer
// than its matrix instructions.
template <bool EXACT>
__device__ __forceinline__ void gauss(float z, float& cdf, float& pdf) {
    if (EXACT) {
        cdf = 0.5f * erfcf(z * -0.70710678f);
        pdf = 0.39894228f * expf(-0.5f * z * z);
    } else {
        const float x = fabsf(z) * 0.70710678f, t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.375f, x, 1.f));
        const float e = __builtin_amdgcn_exp2f(x * x * -1.44269504f);
        float P = -0.1350959092f;
        const float c[6] = {0.3879378438f, -0.1295973212f, 0.2830615640f, 0.1666645557f, 0.2156891823f, 0.2113394439f};
#pragma unroll
        for (int i = 0; i < 6; ++i) P = __builtin_fmaf(t, P, c[i]);
        const float q = 0.5f * t * e * P;
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
        for (int i = 0; i < N; ++i) v[i] *= papr_sigmoid<EXACT>(v[i]);
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
            const float p = papr_sigmoid<EXACT>(z[i]);
            g[i] *= p * __builtin_fmaf(z[i], 1.f - p, 1.f);
        }
    }
}

// a float32 value in three bfloat16 parts (of an infinity the third is NaN)
__device__ __forceinline__ void cut_float(float v, bf16 (&part)[3]) {
    const float most = largest<bf16>();
    part[0] = (bf16)__builtin_amdgcn_fmed3f(v, -most, most);
    v -= (float)part[0];
    part[1] = (bf16)v;
    v -= (float)part[1];
    part[2] = (bf16)v;
}

enum { K_RUNS = 0, ROWS_RUN = 1 };                // which index of an operand is contiguous in memory
enum { OUT_FORWARD = 0, OUT_ROWS = 1, OUT_SLAB = 2, OUT_FORWARD_LOOSE = 3 };      // (loose: rows of the results that start anywhere)

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
// FMT: 0 rows of type T; PAPR_KEEP_* 8-bit rows (ROWS_RUN only); PAIR rows that are the sum of two sets of rows of type T, Operand::low bytes apart.
// A thread's pieces sit at fixed 32-bit offsets from a uniform tile address that advances with k.
constexpr int PAIR = 3;
template <typename T, int LAYOUT, int FMT, bool VEC, int R, int BK, int THREADS>
struct Tile {
    static constexpr bool PACKED = FMT == PAPR_KEEP_E4M3 || FMT == PAPR_KEEP_INT8, SPLIT = sizeof(T) == 4 && FMT == 0;
    static constexpr int SOURCES = FMT == PAIR ? 2 : 1, PLANES = SPLIT ? 3 : SOURCES;
    static constexpr int PIECE = SPLIT ? 4 : 8;                                   // elements of one load
    static constexpr int BYTES = PACKED ? 1 : sizeof(T);
    static constexpr int N = R * BK / PIECE / THREADS;
    static constexpr int STRIDE = LAYOUT == K_RUNS ? BK : (R * 2 % 256 == 64 ? R : R + 32);
    static constexpr int PLANE = (LAYOUT == K_RUNS ? R : BK) * STRIDE;            // halfs
    static constexpr int HALFS = PLANES * PLANE;
    static_assert(R * BK % (PIECE * THREADS) == 0, "whole pieces per thread");
    typedef typename Matrix<T>::frag frag;

    struct Held { uint4 reg[SOURCES][N]; uint8_t ex[PACKED ? N : 1]; };           // a tile on its way
    unsigned off[N];                                                              // bytes from the tile's address
    unsigned exo[PACKED ? N : 1];
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
        if (PACKED) exb = o.exps + k0 * (ld >> 5) + (r0 >> 5);
        const int64_t left = (PACKED ? ld : o.rows) - r0;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            if (r >= left) r = LAYOUT == K_RUNS ? (int)left - 1 : 0;              // (rows past the end: some row of the operand, its results are never stored)
            off[q] = (unsigned)((LAYOUT == K_RUNS ? (int64_t)r * ld + k : (int64_t)k * ld + r) * BYTES);
            if (PACKED) exo[q] = (unsigned)(k * (ld >> 5) + (r >> 5));
        }
    }
    // the next tile: k0 .. k0 + BK of K terms.  `inside`: every piece may be read whole.  A piece that crosses the end of a contiguous row of rows reads the start
    // of the next one (those rows of the product are never stored), but behind the last k there is no next one.
    __device__ __forceinline__ void load(Held& h, const Operand& o, int64_t r0, int64_t k0, int64_t K) {
        bool inside = k0 + BK <= K;
        if (LAYOUT == ROWS_RUN && !VEC && !PACKED) inside = k0 + BK < K && o.rows >= PIECE;
#pragma unroll
        for (int n = 0; n < SOURCES; ++n) {
            const char* const at = base + (n ? o.low : 0);
            if (inside) {
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    const char* src = at + off[q];
                    if (PACKED) {
                        const uint2 c = *reinterpret_cast<const uint2*>(src);
                        h.reg[n][q].x = c.x; h.reg[n][q].y = c.y;
                        h.ex[q] = exb[exo[q]];
                    } else if (VEC) h.reg[n][q] = *reinterpret_cast<const uint4*>(src);
                    else __builtin_memcpy(&h.reg[n][q], __builtin_assume_aligned(src, sizeof(T)), 16);
                }
            } else {
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    int r, k;
                    where(q, r, k);
                    const bool in = k0 + k < K;
                    const char* src = in ? at + off[q] : at;                      // (at: rows r0, the tile's first k < K)
                    if (PACKED) {
                        const uint2 c = *reinterpret_cast<const uint2*>(src);
                        h.reg[n][q].x = in ? c.x : 0u; h.reg[n][q].y = in ? c.y : 0u;
                        h.ex[q] = exb[in ? exo[q] : 0u];
                    } else if (VEC) {
                        const uint4 t = *reinterpret_cast<const uint4*>(src);
                        h.reg[n][q].x = in ? t.x : 0u; h.reg[n][q].y = in ? t.y : 0u; h.reg[n][q].z = in ? t.z : 0u; h.reg[n][q].w = in ? t.w : 0u;
                    } else {
                        papr_pack<T, PIECE> t;
                        if (LAYOUT == ROWS_RUN && r0 + r >= o.rows) r = 0;
#pragma unroll
                        for (int i = 0; i < PIECE; ++i) {
                            const bool ok = LAYOUT == K_RUNS ? k0 + k + i < K : in && r0 + r + i < o.rows;
                            t.v[i] = ok ? reinterpret_cast<const T*>(src)[i] : (T)0.f;
                        }
                        __builtin_memcpy(&h.reg[n][q], &t, 16);
                    }
                }
            }
        }
        base += (LAYOUT == K_RUNS ? (int64_t)BK : BK * ld) * BYTES;
        if (PACKED) exb += BK * (ld >> 5);
    }

    __device__ __forceinline__ void store(const Held& h, short* lds) const {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            const int at = LAYOUT == K_RUNS ? place(r, k >> 3) + (k & 7) : k * STRIDE + r;
            if constexpr (PACKED) {
                float v[4], w[4];
                const float scale = __uint_as_float((unsigned)h.ex[q] << 23);
                papr_codes_to_float<FMT>(h.reg[0][q].x, scale, v);
                papr_codes_to_float<FMT>(h.reg[0][q].y, scale, w);
                frag to;
#pragma unroll
                for (int i = 0; i < 4; ++i) { to[i] = v[i]; to[4 + i] = w[i]; }     // (exact: at most 8 significant bits)
                *reinterpret_cast<frag*>(lds + at) = to;
            } else if (SPLIT) {
                const uint4 t = h.reg[0][q];
                const float f[4] = {__uint_as_float(t.x), __uint_as_float(t.y), __uint_as_float(t.z), __uint_as_float(t.w)};
                papr_pack<bf16, 4> p[PLANES];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bf16 cut[3];
                    cut_float(f[i], cut);
#pragma unroll
                    for (int n = 0; n < PLANES; ++n) p[n].v[i] = cut[n];
                }
#pragma unroll
                for (int n = 0; n < PLANES; ++n) *reinterpret_cast<papr_pack<bf16, 4>*>(lds + n * PLANE + at) = p[n];
            } else {
#pragma unroll
                for (int n = 0; n < SOURCES; ++n) *reinterpret_cast<uint4*>(lds + n * PLANE + at) = h.reg[n][q];
            }
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

// Tile shapes: waves WM x WN, each IM x IN blocks of 32 x 32; DEPTH stages of a streaming kernel.
template <int WM_, int WN_, int IM_, int IN_, int DEPTH_>
struct Shape {
    static constexpr int DEPTH = DEPTH_, WM = WM_, WN = WN_, IM = IM_, IN = IN_, THREADS = 64 * WM * WN, TM = WM * IM * 32, TN = WN * IN * 32;
    static constexpr int EPI_STRIDE = IN * 32 + 8;                                // floats: rows four apart lie on the other half of the banks
    static constexpr size_t EPI = (size_t)WM * WN * 32 * EPI_STRIDE * 4;
};

template <typename T, int LA, int LB, int FA, int FMT, bool VEC, typename S>
struct Plan {
    static constexpr int BK = sizeof(T) == 2 ? 64 : 32, BUFFERS = (sizeof(T) == 4 || FA == PAIR) && S::TM > 64 ? 1 : 2;
    typedef Tile<T, LA, FA, VEC, S::TM, BK, S::THREADS> TA;
    typedef Tile<T, LB, FMT, VEC, S::TN, BK, S::THREADS> TB;
    static constexpr int BUF = TA::HALFS + TB::HALFS;
    static constexpr size_t LOOP = (size_t)BUFFERS * BUF * 2, LDS = S::EPI > LOOP ? S::EPI : LOOP;
};

// E consecutive results of row m from column n on.  LOOSE: rows that start anywhere (the hardware takes 16 bytes at any address, in two requests).
template <typename T, int E, bool LOOSE>
__device__ __forceinline__ void put(T* to, const papr_pack<T, E>& t) {
    if (LOOSE) __builtin_memcpy(to, &t, sizeof(t));
    else *reinterpret_cast<papr_pack<T, E>*>(to) = t;
}
// z as 16-bit rows hold it: beyond their largest number that number (the slopes there are the activations' limits, 0 and 1, where those of an infinity are 0 times
// infinity); NaN stays
template <typename T>
__device__ __forceinline__ float kept_finite(float z) {
    if (sizeof(T) == 4) return z;
    const float most = largest<T>();
    return z == z ? __builtin_amdgcn_fmed3f(z, -most, most) : z;
}
template <typename Z, int E, bool LOOSE>
__device__ __forceinline__ void put_z(const float (&v)[E], void* z, int64_t at) {
    papr_pack<Z, E> t;
#pragma unroll
    for (int i = 0; i < E; ++i) t.v[i] = (Z)kept_finite<Z>(v[i]);
    put<Z, E, LOOSE>(reinterpret_cast<Z*>(z) + at, t);
}
template <typename T, int OUT, int E, bool LOOSE>
__device__ __forceinline__ void finish(float (&v)[E], int64_t m, int64_t n, int64_t N, const float (&bias)[E], const papr_pack<T, E>& res, const Epilogue& ep) {
    if (OUT == OUT_FORWARD) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] += bias[i];
        if (ep.z) {
            if (__is_same(T, bf16) && z_in_f16(ep.act)) put_z<f16, E, LOOSE>(v, ep.z, m * N + n);
            else put_z<T, E, LOOSE>(v, ep.z, m * N + n);
        }
        act_values<sizeof(T) == 4>(v, ep.act);
        if (ep.res)
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] += (float)res.v[i];
    }
    papr_pack<T, E> t;
#pragma unroll
    for (int i = 0; i < E; ++i) t.v[i] = (T)v[i];
    put<T, E, LOOSE>(reinterpret_cast<T*>(ep.out) + m * N + n, t);
}
template <typename T>
__device__ __forceinline__ void finish_one(float value, int64_t m, int64_t n, int64_t N, const Epilogue& ep) {
    float v[1] = {value}, bias[1] = {ep.bias ? (float)reinterpret_cast<const T*>(ep.bias)[n] : 0.f};
    papr_pack<T, 1> res;
    if (ep.res) res.v[0] = reinterpret_cast<const T*>(ep.res)[m * ep.ld_res + n];
    finish<T, OUT_FORWARD, 1, false>(v, m, n, N, bias, res, ep);
}
// 32 rows of a wave's part, from its LDS: 16 bytes of a row a lane
template <typename T, int OUT, typename S, bool LOOSE>
__device__ __forceinline__ void write_block(const float* epi, int64_t mw, int64_t n, int64_t M, int64_t N, const float (&bias)[16 / sizeof(T)], const Epilogue& ep) {
    constexpr int COLS = S::IN * 32, E = 16 / sizeof(T), LPR = COLS / E, RPP = 64 / LPR;
    const int lane = threadIdx.x & 63;
    const bool whole = LOOSE ? n + E <= N : n < N, with_res = OUT == OUT_FORWARD && ep.res;
    papr_pack<T, E> res[32 / RPP];
    if (with_res)
#pragma unroll
        for (int r = 0; r < 32 / RPP; ++r) {
            const int64_t m = mw + r * RPP + lane / LPR;
            if (m >= M || !whole) continue;
            const T* src = reinterpret_cast<const T*>(ep.res) + m * ep.ld_res + n;
            if (LOOSE) __builtin_memcpy(&res[r], src, sizeof(res[r]));
            else res[r] = *reinterpret_cast<const papr_pack<T, E>*>(src);
        }
#pragma unroll
    for (int r = 0; r < 32 / RPP; ++r) {
        const int64_t m = mw + r * RPP + lane / LPR;
        const float* at = epi + (r * RPP + lane / LPR) * S::EPI_STRIDE + lane % LPR * E;
        float v[E];
#pragma unroll
        for (int c = 0; c < E; c += 4) {
            const float4 t = *reinterpret_cast<const float4*>(at + c);
            v[c] = t.x; v[c + 1] = t.y; v[c + 2] = t.z; v[c + 3] = t.w;
        }
        if (m < M && whole) finish<T, OUT, E, LOOSE>(v, m, n, N, bias, res[r], ep);
    }
    if (LOOSE && !whole)                           // (the last columns of the rows)
#pragma unroll 1
        for (int r = 0; r < 32 / RPP; ++r) {
            const int64_t m = mw + r * RPP + lane / LPR;
            const float* at = epi + (r * RPP + lane / LPR) * S::EPI_STRIDE + lane % LPR * E;
#pragma unroll 1
            for (int i = 0; m < M && n + i < N; ++i) {
                if (OUT == OUT_FORWARD) finish_one<T>(at[i], m, n + i, N, ep);
                else reinterpret_cast<T*>(ep.out)[m * N + n + i] = (T)at[i];
            }
        }
}

// The results of a workgroup's tile, from the accumulators of its waves.  smem: Shape::EPI bytes, free of earlier readers.
template <typename T, int OUT, typename S>
__device__ __forceinline__ void write_tile(const f32x16 (&acc)[S::IM][S::IN], short* smem, int64_t m0, int64_t n0, int64_t M, int64_t N, int part, const Epilogue& ep) {
    constexpr int IM = S::IM, IN = S::IN, EPI_STRIDE = S::EPI_STRIDE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
    if (OUT == OUT_SLAB) {
        // float32, as it lies: a lane holds column lane & 31 of a 32 x 32 block, rows (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
        float* out = reinterpret_cast<float*>(ep.out) + (int64_t)part * M * N;
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
    // Through LDS, 32 rows of the wave's own at a time (no barrier), so that a lane takes 16 bytes of a row: whole lines in and out.
    float* epi = reinterpret_cast<float*>(smem) + wave * 32 * EPI_STRIDE;
    constexpr int COLS = IN * 32, E = 16 / sizeof(T);
    constexpr bool FORWARD = OUT == OUT_FORWARD || OUT == OUT_FORWARD_LOOSE;
    const int64_t n = n0 + wn * COLS + lane % (COLS / E) * E;
    float bias[E];
#pragma unroll
    for (int i = 0; i < E; ++i) bias[i] = FORWARD && ep.bias && n + i < N ? (float)reinterpret_cast<const T*>(ep.bias)[n + i] : 0.f;
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int64_t mw = m0 + (wm * IM + i) * 32;
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) epi[((e & 3) + 8 * (e >> 2) + 4 * (lane >> 5)) * EPI_STRIDE + j * 32 + (lane & 31)] = acc[i][j][e];
        // (the forward pass's two forms are kernels of their own: an activation's five forms times a tile's passes, twice, do not fit the instruction cache -- with both
        // in one kernel 65,536 x 1024 -> 1024 took 345 us for 235)
        if constexpr (FORWARD) write_block<T, OUT_FORWARD, S, OUT == OUT_FORWARD_LOOSE>(epi, mw, n, M, N, bias, ep);
        else if (ep.wide) write_block<T, OUT, S, false>(epi, mw, n, M, N, bias, ep);
        else write_block<T, OUT, S, true>(epi, mw, n, M, N, bias, ep);
    }
}

// A float32 result that is NaN because an operand is (then it is found at once) or is infinite: the sum of its terms as the definition has them.
template <typename T, int LAYOUT, int FMT>
__device__ __forceinline__ float term(const Operand& o, int64_t r, int64_t k) {
    const int64_t at = LAYOUT == K_RUNS ? r * o.ld + k : k * o.ld + r;
    if (FMT == 0) return (float)reinterpret_cast<const T*>(o.p)[at];
    float v[4];
    papr_codes_to_float<FMT>((unsigned)reinterpret_cast<const uint8_t*>(o.p)[at], __uint_as_float((unsigned)o.exps[at >> 5] << 23), v);
    return v[0];
}
template <typename T, int LA, int LB, int FMT>
__device__ __forceinline__ float sum_again(const Operand& A, const Operand& B, int64_t m, int64_t n, int64_t kb, int64_t ke) {
    float s = 0.f;
    for (int64_t k = kb; k < ke && s == s; ++k) s = __builtin_fmaf(term<T, LA, 0>(A, m, k), term<T, LB, FMT>(B, n, k), s);
    return s;
}

// Operands through registers: what the streaming kernel cannot take -- float32 (512,000 x 256 -> 256 forward 501 us, d_x 419, d_W 375: 134 - 179 TFLOP/s for the card's 154 of a
// float32 library product; 8192 x 1024 -> 4096 200), 8-bit rows (d_W of 65,536 x 1024 -> 1024 from a pair and codes 293 us, 940 TFLOP/s of its two products, the matrix pipe 42 %
// busy) and short odd rows.  Bound by one stage of loads being on its way and, in float32, by cutting the values apart.
template <typename T, int LA, int LB, int FA, int FMT, bool VEC, int OUT, typename S>
__global__ __launch_bounds__(S::THREADS, 2) void product_kernel(Operand A, Operand B, int64_t K, int64_t k_per_part, unsigned tiles_m, unsigned tiles_n, Epilogue ep) {
    typedef Plan<T, LA, LB, FA, FMT, VEC, S> P;
    typedef typename P::TA TA;
    typedef typename P::TB TB;
    constexpr int IM = S::IM, IN = S::IN, BK = P::BK;
    extern __shared__ __attribute__((aligned(16))) short smem[];
    __shared__ int nan_seen;                       // (float32 only)
    constexpr bool SPLIT = TA::SPLIT || TB::SPLIT;
    if (SPLIT && threadIdx.x == 0) nan_seen = 0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
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
    // The next tile is on its way in registers while one is multiplied.  float32 (three parts of every value: three times the LDS and six times the matrix instructions of
    // a step) has one buffer and two barriers a step of 32 terms instead of two buffers of 16: half as many steps shorter than the way to memory.
    typename TA::Held ha;
    typename TB::Held hb;
    auto load = [&](int64_t k) __attribute__((always_inline)) {
        if (k >= ke) return;
        a.load(ha, A, m0, k, K);
        b.load(hb, B, n0, k, K);
    };
    auto store = [&](int64_t k, int buf) __attribute__((always_inline)) {
        if (k >= ke) return;
        a.store(ha, smem + buf * P::BUF);
        b.store(hb, smem + buf * P::BUF + TA::HALFS);
    };
    auto multiply = [&](int buf) __attribute__((always_inline)) {
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
            for (int w = 2; w >= 0; --w)          // (the parts' products in order of weight, smallest first; those of weight 2^-25 are left out)
#pragma unroll
                for (int p = 0; p < TA::PLANES; ++p)
#pragma unroll
                    for (int q = 0; q < TB::PLANES; ++q)
                        if (p + q == w)
#pragma unroll
                            for (int i = 0; i < IM; ++i)
#pragma unroll
                                for (int j = 0; j < IN; ++j) acc[i][j] = mfma(fa[p][i], fb[q][j], acc[i][j]);
        }
    };
    load(kb);
    if constexpr (P::BUFFERS == 1) {
        for (int64_t k = kb; k < ke; k += BK) {
            store(k, 0);
            __syncthreads();
            load(k + BK);
            multiply(0);
            __syncthreads();
        }
    } else {
        store(kb, 0);
        __syncthreads();
        int buf = 0;
        for (int64_t k = kb; k < ke; k += BK, buf ^= 1) {
            load(k + BK);
            multiply(buf);
            store(k + BK, buf ^ 1);
            __syncthreads();
        }
    }
    bool again = false;
    if constexpr (SPLIT) {                         // (looking at every value on its way into LDS instead cost 4 to 8 % of a product)
        bool nan = false;
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j)
#pragma unroll
                for (int e = 0; e < 16; e += 2) nan |= __builtin_isunordered(acc[i][j][e], acc[i][j][e + 1]);
        if (nan) nan_seen = 1;
        __syncthreads();
        again = nan_seen != 0;
    }
    write_tile<T, OUT, S>(acc, smem, m0, n0, A.rows, B.rows, at.part, ep);
    if constexpr (SPLIT) {
        if (!again) return;
        __syncthreads();
        float* out = reinterpret_cast<float*>(ep.out) + (OUT == OUT_SLAB ? at.part * A.rows * B.rows : 0);
        for (int i = threadIdx.x; i < S::TM * S::TN; i += S::THREADS) {
            const int64_t m = m0 + i / S::TN, n = n0 + i % S::TN;
            if (m >= A.rows || n >= B.rows) continue;
            float& to = out[m * B.rows + n];
            if (to == to) continue;
            float v[1] = {sum_again<T, LA, LB, FMT>(A, B, m, n, kb, ke)};
            if constexpr (OUT == OUT_SLAB || OUT == OUT_ROWS) to = v[0];
            else finish_one<T>(v[0], m, n, B.rows, ep);
        }
    }
}

// The same product for 16-bit rows that start on 16 bytes: operands go straight from memory into LDS (global_load_lds, 16 bytes a lane), DEPTH stages of 32 terms, three
// of them on their way while one is multiplied (product_kernel: one, in registers).  In d_x and d_W of 8192 x 1024 -> 4096 waves wait 31 to 38 % of their time and the matrix pipe
// is half busy, as at 8192^3.  An instruction fills 1 KB in lane order, so the images are made by which address a lane asks for:
//   K_RUNS:   16 rows of 32 halfs, pieces exchanged by the row number as in Tile;
//   ROWS_RUN: one "line" = the k rows q, q + LINES, q + 2 LINES, ... of R halfs one behind the other (1 KB), lines 1,088 bytes apart: the four consecutive k that a
//             16-lane group of a transposing read wants lie on different quarters of the banks.
// Rows past the operand's end: some row of it (never stored); terms past the part's end: a block of zeros.
// The fragments of a 16-term step are read under the matrix instructions of the step before, and the stage's one barrier stands between its two steps: in front of
// it a wave has read all of its stage (whose buffer the requests behind the barrier overwrite), behind it the next stage, requested three stages earlier, is there.
// What bounds it: the matrix pipe and, for short sums, filling the pipeline and writing the results (the forward product of 65,536 x 1024 -> 1024: 234 us, a quarter busy).  8192^3 in
// bf16 0.86 - 0.96 ms (1150 - 1280 TFLOP/s; the card's library product 1281), d_x and d_W of 65,536 x 1024 -> 1024 from a pair 258 and 245 us (1060, 1120 of their two products).
__device__ const uint4 zero_block[4] = {};

__device__ __forceinline__ void request16(const void* src, unsigned lds) {         // 64 lanes x 16 bytes -> LDS [lds, +1 KB) in lane order
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(src), "s"(lds) : "memory");
}

template <typename T, int LAYOUT, int R, int WAVES>
struct Stage {
    static constexpr int BK = 32, LINE = LAYOUT == K_RUNS ? 1024 : 1088, LINES = R * BK * 2 / 1024, BYTES = LINES * LINE, N = LINES / WAVES;
    static_assert(LINES % WAVES == 0 && R * 2 <= 1024, "whole requests per wave");
    typedef typename Matrix<T>::frag frag;
    const char* src[N];                                                            // this lane's address of the next stage's requests
    int k[N];                                                                      // its term inside the stage
    int64_t step;

    __device__ __forceinline__ void start(const Operand& o, int64_t r0, int64_t k0, int wave) {
        const int lane = threadIdx.x & 63;
        const int64_t left = o.rows - r0;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int line = wave * N + q;
            int r;
            if (LAYOUT == K_RUNS) {
                r = line * 16 + lane / 4;
                k[q] = 8 * ((lane & 3) ^ ((r >> 2) & 3));
                if (r >= left) r = (int)left - 1;
                src[q] = reinterpret_cast<const char*>(o.p) + ((r0 + r) * o.ld + k0 + k[q]) * 2;
            } else {
                r = 8 * (lane % (R / 8));
                k[q] = line + lane / (R / 8) * LINES;
                if (r >= left) r = 0;
                src[q] = reinterpret_cast<const char*>(o.p) + ((k0 + k[q]) * o.ld + r0 + r) * 2;
            }
        }
        step = (LAYOUT == K_RUNS ? (int64_t)BK : BK * o.ld) * 2;
    }
    // requests of the next stage; `left`: terms from its first on; `low`: bytes to the rows that are asked for; `last`: the stage behind it takes the next terms
    __device__ __forceinline__ void request(unsigned lds, int64_t left, int wave, int64_t low, bool last) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const void* p = k[q] < left ? (const void*)(src[q] + low) : (const void*)zero_block;
            request16(p, lds + (unsigned)(wave * N + q) * LINE);
            if (last) src[q] += step;
        }
    }
    // this lane's corner of the fragments (bytes): rows `row` .. + 31, step 0
    static __device__ __forceinline__ unsigned corner(int row) {
        const int lane = threadIdx.x & 63;
        if (LAYOUT == K_RUNS) { const int r = row + (lane & 31); return (unsigned)(r * 64 + (((lane >> 5) ^ ((r >> 2) & 3)) << 4)); }
        const int c = 8 * (lane >> 5) + ((lane & 15) >> 2);
        return (unsigned)(c % LINES * LINE + c / LINES * R * 2 + (row + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2);
    }
    // LINES is 16 (R = 256) or 8 (R = 128): the second step's k + 16 is one half of a line on, or two quarters; four k on is four lines (LINES > 4, c < 12)
    static __device__ __forceinline__ frag read(unsigned stage, unsigned corner, int ks) {
        s16x8 v;
        if (LAYOUT == K_RUNS) {
            // (piece c of step 1 is piece c + 2: the exchange turns + 2 into ^ 2)
            v = *reinterpret_cast<const __attribute__((address_space(3))) s16x8*>(stage + (corner ^ (unsigned)(ks * 32)));
        } else {
            const unsigned a = stage + corner + (unsigned)(ks * 16 / LINES * R * 2);
            const s16x4 lo = read_tr4(a), hi = read_tr4(a + 4 * LINE);
            v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return __builtin_bit_cast(frag, v);
    }
};

template <typename T, int LA, int LB, typename S>
struct Stream {
    static constexpr int DEPTH = S::DEPTH;
    typedef Stage<T, LA, S::TM, S::WM * S::WN> SA;
    typedef Stage<T, LB, S::TN, S::WM * S::WN> SB;
    static constexpr unsigned BYTES = SA::BYTES + SB::BYTES;
    static constexpr size_t LOOP = (size_t)DEPTH * BYTES, LDS = S::EPI > LOOP ? S::EPI : LOOP;
};

template <typename T, int LA, int LB, int FA, int OUT, typename S>
__global__ __launch_bounds__(S::THREADS, 2) void stream_kernel(Operand A, Operand B, int64_t K, int64_t k_per_part, unsigned tiles_m, unsigned tiles_n, Epilogue ep) {
    typedef Stream<T, LA, LB, S> P;
    typedef typename P::SA SA;
    typedef typename P::SB SB;
    constexpr int IM = S::IM, IN = S::IN, WAITING = (P::DEPTH - 2) * (SA::N + SB::N);          // requests of the stages behind the next one
    extern __shared__ __attribute__((aligned(16))) short smem[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / S::WN, wn = wave % S::WN;
    const Place at = place_of(blockIdx.x, gridDim.x, tiles_m, tiles_n);
    const int64_t m0 = (int64_t)at.m * S::TM, n0 = (int64_t)at.n * S::TN;
    const int64_t kb = at.part * k_per_part, ke = kb + k_per_part < K ? kb + k_per_part : K;
    constexpr int SETS = FA == PAIR ? 2 : 1;        // (a pair's high and low rows: two stages with the same terms of B)
    const int stages = (int)((ke - kb + 31) / 32) * SETS;
    const unsigned lds = (unsigned)(size_t)smem;
    f32x16 acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    SA a;
    SB b;
    a.start(A, m0, kb, wave);
    b.start(B, n0, kb, wave);
    int64_t left = ke - kb;
    auto request = [&](int st) {
        const unsigned to = lds + (unsigned)(st % P::DEPTH) * P::BYTES;
        const int set = SETS == 2 ? st & 1 : 0;
        a.request(to, left, wave, set ? A.low : 0, set == SETS - 1);
        b.request(to + SA::BYTES, left, wave, 0, set == SETS - 1);
        if (set == SETS - 1) left -= 32;
    };
    unsigned ca[IM], cb[IN];
#pragma unroll
    for (int i = 0; i < IM; ++i) ca[i] = SA::corner((wm * IM + i) * 32);
#pragma unroll
    for (int j = 0; j < IN; ++j) cb[j] = SA::BYTES + SB::corner((wn * IN + j) * 32);
    struct Frags { typename SA::frag a[IM]; typename SB::frag b[IN]; } f0, f1;
    auto read = [&](Frags& f, int st, int ks) {
        const unsigned from = lds + (unsigned)(st % P::DEPTH) * P::BYTES;
#pragma unroll
        for (int j = 0; j < IN; ++j) f.b[j] = SB::read(from, cb[j], ks);
#pragma unroll
        for (int i = 0; i < IM; ++i) f.a[i] = SA::read(from, ca[i], ks);
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int j = 0; j < IN; ++j) acc[i][j] = mfma(f.a[i], f.b[j], acc[i][j]);
    };
#pragma unroll
    for (int st = 0; st < P::DEPTH - 1; ++st) request(st);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(WAITING) : "memory");     // stage 0 is there (every wave's part of it)
    request(P::DEPTH - 1);
    read(f0, 0, 0);
    for (int st = 0; st < stages; ++st) {
        read(f1, st, 1);
        multiply(f0);
        // stage st is read (its reads are waited for), stage st + 1 is there: the two stages behind it may be on their way
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(WAITING) : "memory");
        request(st + P::DEPTH);
        read(f0, st + 1, 0);                       // (behind the last stage: a stage of zeros, not multiplied)
        multiply(f1);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    write_tile<T, OUT, S>(acc, smem, m0, n0, A.rows, B.rows, at.part, ep);
}

// Few rows (one token, a handful): the weight is read once and that is the time.  A workgroup takes 16 columns of the result, its waves a part of the sum each,
// straight from memory into the operands of 16 x 16 x 32 matrix instructions (rows of x come from the caches); the parts meet in LDS, in wave order.
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(Operand A, Operand B, int64_t K, bool aligned, Epilogue ep) {
    constexpr int PARTS = sizeof(T) == 4 ? 3 : 1, AHEAD = 8 / MT / (sizeof(T) / 2);
    typedef typename Matrix<T>::frag frag;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    __shared__ float lds[WAVES][MT * 16][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, k8 = lane >> 4 << 3;
    const int64_t M = A.rows, N = B.rows, n0 = (int64_t)blockIdx.x * 16;
    const int steps = (int)((K + 31) / 32), per = (steps + WAVES - 1) / WAVES, beg = wave * per, end = beg + per < steps ? beg + per : steps;
    struct Eight { papr_pack<T, 8> t; };
    auto fetch = [&](Eight& v, const Operand& o, int64_t row, int step) __attribute__((always_inline)) {
        row = row < o.rows ? row : o.rows - 1;
        const int64_t k = (int64_t)step * 32 + k8;
        const T* src = reinterpret_cast<const T*>(o.p) + row * o.ld + k;
        if ((int64_t)step * 32 + 32 <= K) {
            if (aligned) {
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(&v.t)[i] = reinterpret_cast<const uint4*>(src)[i];
            } else __builtin_memcpy(&v.t, src, sizeof(v.t));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v.t.v[i] = k + i < K ? src[i] : (T)0.f;
        }
    };
    auto parts = [&](frag (&f)[PARTS], const Eight& v) __attribute__((always_inline)) {
        if constexpr (PARTS == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[0][i] = v.t.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                bf16 cut[3];
                cut_float(v.t.v[i], cut);
                f[0][i] = cut[0]; f[1][i] = cut[1]; f[2][i] = cut[2];
            }
        }
    };
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int s0 = beg; s0 < end; s0 += AHEAD) {
        Eight wv[AHEAD], xv[AHEAD][MT];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (s0 + a >= end) break;
            fetch(wv[a], B, n0 + r, s0 + a);
#pragma unroll
            for (int t = 0; t < MT; ++t) fetch(xv[a][t], A, t * 16 + r, s0 + a);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (s0 + a >= end) break;
            frag wf[PARTS];
            parts(wf, wv[a]);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                frag xf[PARTS];
                parts(xf, xv[a][t]);
#pragma unroll
                for (int w = 2; w >= 0; --w)
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        const int q = w - p;
                        if (q >= 0 && q < PARTS) {
                            if constexpr (__is_same(T, f16)) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[p], wf[q], acc[t], 0, 0, 0);
                            else acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[p], wf[q], acc[t], 0, 0, 0);
                        }
                    }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) lds[wave][t * 16 + 4 * (lane >> 4) + e][r] = acc[t][e];
    __syncthreads();
    for (int i = threadIdx.x; i < MT * 256; i += 64 * WAVES) {
        const int64_t m = i >> 4, n = n0 + (i & 15);
        if (m >= M || n >= N) continue;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += lds[w][m][i & 15];
        if constexpr (sizeof(T) == 4)
            if (v != v) v = sum_again<T, K_RUNS, K_RUNS, 0>(A, B, m, n, 0, K);
        finish_one<T>(v, m, n, N, ep);
    }
}

// papr_profile_collect: one record a product (its slabs' joining included)
struct Timed {
    hipStream_t s;
    bool on;
    Timed(int kernel, int64_t M, int64_t N, int64_t K, hipStream_t stream) : s(stream), on(papr_prof_on()) {
        if (on) papr_prof_begin2(kernel, (long)M, (int)N, (int)K, 0, 2LL * M * N * K, s);
    }
    ~Timed() { if (on) papr_prof_end(s); }
};

// Up to here the few-rows kernel is the faster one: 1 x 1024 -> 4096 bf16 3.8 us against 10.1 of 64 x 64 tiles, 32 x 4096 -> 1024 26.8 against 29.6, 64 x 4096 -> 1024 48 against 30.
constexpr int FEW_ROWS = 32;

template <typename T>
int launch_few_rows(const Operand& A, const Operand& B, int64_t K, bool vec, const Epilogue& ep, hipStream_t s) {
    // (sixteen waves where there are fewer workgroups than compute units and steps enough: 16 x 4096 -> 1024 in bf16 16.6 us with eight)
    const dim3 grid((unsigned)((B.rows + 15) / 16));
    const bool many = B.rows <= 16 * papr_cu_count() / 2 && K >= 1024;
    if (A.rows <= 16) {
        if (many) few_rows_kernel<T, 1, 16><<<grid, 1024, 0, s>>>(A, B, K, vec, ep);
        else few_rows_kernel<T, 1, 8><<<grid, 512, 0, s>>>(A, B, K, vec, ep);
    } else {
        if (many) few_rows_kernel<T, 2, 16><<<grid, 1024, 0, s>>>(A, B, K, vec, ep);
        else few_rows_kernel<T, 2, 8><<<grid, 512, 0, s>>>(A, B, K, vec, ep);
    }
    PAPR_CHECK_LAUNCH("papr_linear_fwd");
    return 0;
}

// The slabs of a sum in parts, V results a lane.  SPREAD: the four waves of a workgroup take a quarter of the parts each (many parts: their loads are a chain), quarters
// added in order; otherwise a lane adds all parts of its results.  Bound by reading the slabs, which mostly still lie in the caches: 8192 x 4096 -> 1024 12 us with its launch.
template <typename T, int V, bool SPREAD>
__global__ __launch_bounds__(256) void join_slabs_kernel(const float* __restrict__ slab, int64_t n, int parts, T* __restrict__ out) {
    __shared__ float lds[SPREAD ? 4 : 1][SPREAD ? 64 * V : 1];
    const int lane = SPREAD ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6, per = SPREAD ? (parts + 3) / 4 : parts;
    constexpr int SPAN = (SPREAD ? 64 : 256) * V;
    const int beg = SPREAD ? wave * per : 0, end = beg + per < parts ? beg + per : parts;
    for (int64_t i0 = (int64_t)blockIdx.x * SPAN; i0 < n; i0 += (int64_t)gridDim.x * SPAN) {
        const int64_t at = i0 + lane * V, i = at < n ? at : 0;
        papr_pack<float, V> s;
#pragma unroll
        for (int v = 0; v < V; ++v) s.v[v] = 0.f;
#pragma unroll 8
        for (int k = beg; k < end; ++k) {
            const auto t = *reinterpret_cast<const papr_pack<float, V>*>(slab + k * n + i);
#pragma unroll
            for (int v = 0; v < V; ++v) s.v[v] += t.v[v];
        }
        if constexpr (SPREAD) {
#pragma unroll
            for (int v = 0; v < V; ++v) lds[wave][lane * V + v] = s.v[v];
            __syncthreads();
            if (wave == 0)
#pragma unroll
                for (int v = 0; v < V; ++v) s.v[v] = (s.v[v] + lds[1][lane * V + v]) + (lds[2][lane * V + v] + lds[3][lane * V + v]);
        }
        if (at < n && (!SPREAD || wave == 0)) {
            papr_pack<T, V> t;
#pragma unroll
            for (int v = 0; v < V; ++v) t.v[v] = (T)s.v[v];
            *reinterpret_cast<papr_pack<T, V>*>(out + at) = t;
        }
        if constexpr (SPREAD) __syncthreads();
    }
}
template <typename T>
int join_slabs(const float* slab, int64_t n, int parts, T* out, hipStream_t s) {
    const bool spread = parts >= 16, wide = n % 4 == 0 && ((uintptr_t)out & 15) == 0;
    const int64_t span = (spread ? 64 : 256) * (wide ? 4 : 1), need = (n + span - 1) / span, cap = (int64_t)papr_cu_count() * 16;
    const dim3 grid((unsigned)(need < cap ? need : cap));
    if (spread) {
        if (wide) join_slabs_kernel<T, 4, true><<<grid, 256, 0, s>>>(slab, n, parts, out);
        else join_slabs_kernel<T, 1, true><<<grid, 256, 0, s>>>(slab, n, parts, out);
    } else {
        if (wide) join_slabs_kernel<T, 4, false><<<grid, 256, 0, s>>>(slab, n, parts, out);
        else join_slabs_kernel<T, 1, false><<<grid, 256, 0, s>>>(slab, n, parts, out);
    }
    PAPR_CHECK_LAUNCH("papr_linear slabs");
    return 0;
}

// d_z = d_y act'(z) (none: d_y as it is, nothing is written) and the column sums of it in float32, one partial row per workgroup.  In the rows' type where that is exact
// (float32; relu: d_y or zero), else SPLIT in two values of it: high = d_z rounded and kept finite, low = what is left, rounded (so an infinity stays one in their sum).  Bound by
// HBM: 512,000 x 256 float32 320 us (4.9 TB/s), 8192 x 4096 bfloat16 in two values 55 (4.9).
// A thread holds whole vectors of columns; the threads of a workgroup beyond one row's take further rows.
template <typename T, typename Z, bool SPLIT, bool VEC>
__global__ __launch_bounds__(256) void slope_kernel(const T* __restrict__ d_y, int64_t ld, const Z* __restrict__ z, int64_t M, int N, int act, int lanes, T* __restrict__ d_z,
                                                    T* __restrict__ low, int64_t ldz, float* __restrict__ part, int64_t rows_per_block) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    __shared__ float fold[256 * V];
    const int per = 256 / lanes, cg = threadIdx.x % lanes, rl = threadIdx.x / lanes;
    const int c = (blockIdx.y * lanes + cg) * V;
    const int64_t beg = (int64_t)blockIdx.x * rows_per_block, end = beg + rows_per_block < M ? beg + rows_per_block : M;
    const float most = largest<T>();
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.f;
    if (d_z && !VEC && c >= N && c < ldz)           // (zeros up to whole vectors)
        for (int64_t m = beg + rl; m < end; m += per) {
            d_z[m * ldz + c] = (T)0.f;
            if (SPLIT) low[m * ldz + c] = (T)0.f;
        }
    if (c < N)
#pragma unroll 4
        for (int64_t m = beg + rl; m < end; m += per) {
            const auto g = *reinterpret_cast<const papr_pack<T, V>*>(d_y + m * ld + c);
            if (d_z) {
                const auto t = *reinterpret_cast<const papr_pack<Z, V>*>(z + m * N + c);
                float v[V], zv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) { v[i] = (float)g.v[i]; zv[i] = (float)t.v[i]; }
                act_slopes<sizeof(T) == 4>(v, zv, act);
                papr_pack<T, V> to, rest;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sum[i] += v[i];
                    to.v[i] = (T)(SPLIT ? __builtin_amdgcn_fmed3f(v[i], -most, most) : v[i]);
                    if (SPLIT) rest.v[i] = (T)(v[i] - (float)to.v[i]);
                }
                *reinterpret_cast<papr_pack<T, V>*>(d_z + m * ldz + c) = to;
                if (SPLIT) *reinterpret_cast<papr_pack<T, V>*>(low + m * ldz + c) = rest;
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

typedef Shape<2, 4, 4, 2, 4> Large;                // 256 x 256, eight waves
typedef Shape<2, 2, 2, 2, 4> Middle;               // 128 x 128, four waves
typedef Shape<2, 2, 1, 1, 4> Small;                // 64 x 64, four waves

template <auto KERNEL, size_t LDS, typename S>
int launch_kernel(const Operand& A, const Operand& B, int64_t K, const Choice& c, const Epilogue& ep, hipStream_t s) {
    static_assert(LDS <= 160 * 1024, "a compute unit's LDS");
    const int64_t tm = (A.rows + S::TM - 1) / S::TM, tn = (B.rows + S::TN - 1) / S::TN, grid = tm * tn * c.parts;
    PAPR_REQUIRE(grid < (int64_t)1 << 31, "papr_linear: %lld tiles", (long long)grid);
    if (LDS > 65536) {
        static std::atomic<uint64_t> ready{0};        // (devices on which this kernel may already use more than 64 KB of LDS)
        int dev = 0;
        (void)hipGetDevice(&dev);
        const uint64_t bit = 1ull << (dev & 63);
        if (dev > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
            (void)hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS);
            ready.fetch_or(bit, std::memory_order_relaxed);
        }
    }
    KERNEL<<<dim3((unsigned)grid), dim3(S::THREADS), LDS, s>>>(A, B, K, c.per, (unsigned)tm, (unsigned)tn, ep);
    PAPR_CHECK_LAUNCH("papr_linear product");
    return 0;
}

template <typename T, int LA, int LB, int FA, int FMT, bool VEC, int OUT, typename S>
int launch_shape(const Operand& A, const Operand& B, int64_t K, const Choice& c, const Epilogue& ep, hipStream_t s) {
    if constexpr (sizeof(T) == 2 && FMT == 0 && VEC && S::TM >= 128)
        return launch_kernel<stream_kernel<T, LA, LB, FA, OUT, S>, Stream<T, LA, LB, S>::LDS, S>(A, B, K, c, ep, s);
    else
        return launch_kernel<product_kernel<T, LA, LB, FA, FMT, VEC, OUT, S>, Plan<T, LA, LB, FA, FMT, VEC, S>::LDS, S>(A, B, K, c, ep, s);
}

template <typename T, int LA, int LB, int FA, int FMT, bool VEC, int OUT>
int launch_choice(const Choice& c, const Operand& A, const Operand& B, int64_t K, const Epilogue& ep, hipStream_t s) {
    if constexpr (FMT == 0 && VEC)
        if (c.shape == 0) return launch_shape<T, LA, LB, FA, FMT, VEC, OUT, Large>(A, B, K, c, ep, s);
    if (c.shape <= 1) return launch_shape<T, LA, LB, FA, FMT, VEC, OUT, Middle>(A, B, K, c, ep, s);
    return launch_shape<T, LA, LB, FA, FMT, VEC, OUT, Small>(A, B, K, c, ep, s);
}
template <typename T, int LA, int LB, int FA, int FMT, int OUT>
int launch_product(const Choice& c, bool vec, const Operand& A, const Operand& B, int64_t K, const Epilogue& ep, hipStream_t s) {
    return vec ? launch_choice<T, LA, LB, FA, FMT, true, OUT>(c, A, B, K, ep, s) : launch_choice<T, LA, LB, FA, FMT, false, OUT>(c, A, B, K, ep, s);
}

// C = A B^T into contiguous rows of type T, the sum in parts where the tiles alone do not fill the chip
template <typename T, int LA, int LB, int FA, int FMT>
int rows_product(bool vec, const Operand& A, const Operand& B, int64_t K, void* out, float* slab, hipStream_t s) {
    const Choice c = choose(A.rows, B.rows, K, path_of(sizeof(T) == 4 ? PAPR_TYPE_F32 : PAPR_TYPE_F16, vec, FMT, FA == PAIR), true);
    Epilogue ep = {};
    if (c.parts == 1) {
        ep.out = out;
        ep.wide = ((uintptr_t)out & 15) == 0 && (B.rows * sizeof(T)) % 16 == 0;
        return launch_product<T, LA, LB, FA, FMT, OUT_ROWS>(c, vec, A, B, K, ep, s);
    }
    ep.out = slab;
    if (int rc = launch_product<T, LA, LB, FA, FMT, OUT_SLAB>(c, vec, A, B, K, ep, s)) return rc;
    return join_slabs<T>(slab, A.rows * B.rows, (int)c.parts, (T*)out, s);
}

template <typename T, int FA>
int weight_product(int keep, bool vec, const Operand& A, const Operand& B, int64_t M, void* d_w, float* slab, hipStream_t s) {
    if (keep == PAPR_KEEP_E4M3) return rows_product<T, ROWS_RUN, ROWS_RUN, FA, PAPR_KEEP_E4M3>(vec, A, B, M, d_w, slab, s);
    if (keep == PAPR_KEEP_INT8) return rows_product<T, ROWS_RUN, ROWS_RUN, FA, PAPR_KEEP_INT8>(vec, A, B, M, d_w, slab, s);
    return rows_product<T, ROWS_RUN, ROWS_RUN, FA, 0>(vec, A, B, M, d_w, slab, s);
}

template <typename T>
int forward(const Operand& x, const Operand& w, int64_t K, bool vec, const Epilogue& ep, hipStream_t s) {
    Timed timed(13, x.rows, w.rows, K, s);
    if (x.rows <= FEW_ROWS) return launch_few_rows<T>(x, w, K, vec, ep, s);
    const Choice c = choose(x.rows, w.rows, K, path_of(sizeof(T) == 4 ? PAPR_TYPE_F32 : PAPR_TYPE_F16, vec, 0, false), false, aside_of(ep.res, ep.z, sizeof(T)));
    return ep.wide ? launch_product<T, K_RUNS, K_RUNS, 0, 0, OUT_FORWARD>(c, vec, x, w, K, ep, s) : launch_product<T, K_RUNS, K_RUNS, 0, 0, OUT_FORWARD_LOOSE>(c, vec, x, w, K, ep, s);
}

template <typename T>
int grad_rows(bool vec, const Operand& d_z, const Operand& w, int64_t N, void* d_x, float* slab, hipStream_t s) {
    Timed timed(14, d_z.rows, N, w.rows, s);
    if constexpr (sizeof(T) == 2)
        if (d_z.low) return rows_product<T, K_RUNS, ROWS_RUN, PAIR, 0>(vec, d_z, w, N, d_x, slab, s);
    return rows_product<T, K_RUNS, ROWS_RUN, 0, 0>(vec, d_z, w, N, d_x, slab, s);
}

template <typename T>
int grad_weight(int keep, bool vec, const Operand& d_z, const Operand& x, int64_t M, void* d_w, float* slab, hipStream_t s) {
    Timed timed(15, M, d_z.rows, x.rows, s);
    if constexpr (sizeof(T) == 2)
        if (d_z.low) return weight_product<T, PAIR>(keep, vec, d_z, x, M, d_w, slab, s);
    return weight_product<T, 0>(keep, vec, d_z, x, M, d_w, slab, s);
}

template <typename T>
int slopes(bool vec, const SlopeGrid& g, const void* d_y, int64_t ld, const void* z, int64_t M, int N, int act, void* d_z, int64_t low, int64_t ldz, float* part, hipStream_t s) {
    const dim3 grid((unsigned)g.blocks, g.cols);
    T *high = (T*)d_z, *rest = low ? (T*)((char*)d_z + low) : nullptr;
    auto launch = [&](auto of, auto split) {
        typedef decltype(of) Z;
        constexpr bool SPLIT = decltype(split)::value;
        if (vec) slope_kernel<T, Z, SPLIT, true><<<grid, 256, 0, s>>>((const T*)d_y, ld, (const Z*)z, M, N, act, g.lanes, high, rest, ldz, part, g.rows_per_block);
        else slope_kernel<T, Z, SPLIT, false><<<grid, 256, 0, s>>>((const T*)d_y, ld, (const Z*)z, M, N, act, g.lanes, high, rest, ldz, part, g.rows_per_block);
    };
    if constexpr (sizeof(T) == 4) launch(T(), std::false_type());
    else if (!low) launch(T(), std::false_type());
    else if (__is_same(T, bf16) && z_in_f16(act)) launch(f16(), std::true_type());
    else launch(T(), std::true_type());
    PAPR_CHECK_LAUNCH("papr_linear_bwd");
    return 0;
}

}  // namespace papr_linear

// one of linear_f32.hip, linear_f16.hip, linear_bf16.hip
#define PAPR_LINEAR_INSTANCES(T)                                                                                                                                    \
    namespace papr_linear {                                                                                                                                         \
    template int forward<T>(const Operand&, const Operand&, int64_t, bool, const Epilogue&, hipStream_t);                                                           \
    template int grad_rows<T>(bool, const Operand&, const Operand&, int64_t, void*, float*, hipStream_t);                                                           \
    template int grad_weight<T>(int, bool, const Operand&, const Operand&, int64_t, void*, float*, hipStream_t);                                                    \
    template int slopes<T>(bool, const SlopeGrid&, const void*, int64_t, const void*, int64_t, int, int, void*, int64_t, int64_t, float*, hipStream_t);              \
    }
