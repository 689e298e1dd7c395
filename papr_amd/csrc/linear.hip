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

__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case PAPR_ACT_RELU: return z > 0.f ? z : 0.f;
        case PAPR_ACT_LEAKY_RELU: return z > 0.f ? z : 0.2f * z;
        case PAPR_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
        case PAPR_ACT_SILU: return z / (1.f + expf(-z));
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case PAPR_ACT_RELU: return z > 0.f ? 1.f : 0.f;
        case PAPR_ACT_LEAKY_RELU: return z > 0.f ? 1.f : 0.2f;
        case PAPR_ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
        case PAPR_ACT_SILU: { const float p = 1.f / (1.f + expf(-z)); return p * (1.f + z * (1.f - p)); }
        default: return 1.f;
    }
}

enum { K_RUNS = 0, ROWS_RUN = 1 };                // which index of an operand is contiguous in memory
enum { OUT_FORWARD = 0, OUT_ROWS = 1, OUT_SLAB = 2 };

struct Operand { const void* p; int64_t ld; int64_t rows; const uint8_t* exps; };       // exps: 8-bit rows only (ld in codes)
struct Epilogue {
    void* out; int64_t ld_out;
    const void* bias; const void* res; int64_t ld_res; void* z;
    int act;
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
//   K_RUNS:   image [R][BK] halfs, 16-byte pieces exchanged by the row number so that 8 rows' reads of one piece cover all banks.
//   ROWS_RUN: image [BK][R + pad] halfs as it lies in memory; the transposing LDS read hands a lane 8 consecutive k of its row.  The row stride is
//             64 bytes modulo 256: the four k a 16-lane group reads lie on different quarters of the banks.
// FMT: 0 rows of type T, else 8-bit rows (ROWS_RUN only).
template <typename T, int LAYOUT, int FMT, bool VEC, int R, int BK, int THREADS>
struct Tile {
    static constexpr bool SPLIT = sizeof(T) == 4 && FMT == 0;
    static constexpr int PLANES = SPLIT ? 3 : 1;
    static constexpr int PIECE = SPLIT ? 4 : 8;                                   // elements of one load
    static constexpr int N = R * BK / PIECE / THREADS;
    static constexpr int STRIDE = LAYOUT == K_RUNS ? BK : (R * 2 % 256 == 64 ? R : R + 32);
    static constexpr int PLANE = (LAYOUT == K_RUNS ? R : BK) * STRIDE;            // halfs
    static constexpr int HALFS = PLANES * PLANE;
    static_assert(R * BK % (PIECE * THREADS) == 0, "whole pieces per thread");
    typedef typename Matrix<T>::frag frag;

    uint4 reg[N];
    uint8_t ex[FMT ? N : 1];

    // piece q of this thread: (row, k) of its first element inside the tile
    static __device__ __forceinline__ void where(int q, int& r, int& k) {
        const int id = q * THREADS + threadIdx.x;
        if (LAYOUT == K_RUNS) { r = id / (BK / PIECE); k = id % (BK / PIECE) * PIECE; }
        else { k = id / (R / PIECE); r = id % (R / PIECE) * PIECE; }
    }

    // the tile at rows r0 .., k0 .. of an operand with K terms; `inside`: every piece that starts inside the operand may be read whole and no k is past K
    __device__ __forceinline__ void load(const Operand& o, int64_t r0, int64_t k0, int64_t K) {
        bool inside = k0 + BK <= K;
        // (a piece that crosses the end of a contiguous row of rows reads the start of the next one; those rows of the product are never stored, but
        // behind the last k there is no next one)
        if (LAYOUT == ROWS_RUN && !VEC && FMT == 0) inside = k0 + BK < K && o.rows >= PIECE;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            const int64_t kk = k0 + k;
            int64_t rr = r0 + r;
            if (FMT) {                                                            // 8-bit rows: padded to whole blocks of 32 codes, aligned
                rr = rr < o.ld ? rr : 0;
                const bool in = kk < K;
                const int64_t ks = in ? kk : 0;
                const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(o.p) + ks * o.ld + rr);
                ex[q] = o.exps[ks * (o.ld >> 5) + (rr >> 5)];
                reg[q].x = in ? c.x : 0u;
                reg[q].y = in ? c.y : 0u;
                continue;
            }
            rr = rr < o.rows ? rr : (LAYOUT == K_RUNS ? o.rows - 1 : 0);
            const T* src = reinterpret_cast<const T*>(o.p) + (LAYOUT == K_RUNS ? rr * o.ld + kk : kk * o.ld + rr);
            if (inside) {
                if (VEC) reg[q] = *reinterpret_cast<const uint4*>(src);
                else __builtin_memcpy(&reg[q], src, 16);
            } else if (VEC) {
                const bool in = kk < K;
                if (!in) src = reinterpret_cast<const T*>(o.p);
                const uint4 t = *reinterpret_cast<const uint4*>(src);
                reg[q].x = in ? t.x : 0u; reg[q].y = in ? t.y : 0u; reg[q].z = in ? t.z : 0u; reg[q].w = in ? t.w : 0u;
            } else {
                papr_pack<T, PIECE> t;
#pragma unroll
                for (int i = 0; i < PIECE; ++i) {
                    const bool in = LAYOUT == K_RUNS ? kk + i < K : kk < K && rr + i < o.rows;
                    t.v[i] = in ? src[i] : (T)0.f;
                }
                __builtin_memcpy(&reg[q], &t, 16);
            }
        }
    }

    __device__ __forceinline__ void store(short* lds) const {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int r, k;
            where(q, r, k);
            int at;
            if (LAYOUT == K_RUNS) {
                const int sw = BK == 64 ? r & 7 : (r >> 1) & 3;
                at = r * STRIDE + (((k >> 3) ^ sw) << 3) + (k & 7);
            } else at = k * STRIDE + r;
            if (FMT) {
                float v[8];
                const float scale = __uint_as_float((unsigned)ex[q] << 23);
                papr_codes_to_float<FMT>(reg[q].x, scale, v);
                papr_codes_to_float<FMT>(reg[q].y, scale, v + 4);
                frag h;
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] = v[i];                          // (exact: at most 8 significant bits)
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
    static __device__ __forceinline__ frag read(const short* lds, int plane, int base, int ks) {
        const int lane = threadIdx.x & 63;
        s16x8 v;
        if (LAYOUT == K_RUNS) {
            const int r = base + (lane & 31), sw = BK == 64 ? r & 7 : (r >> 1) & 3;
            v = *reinterpret_cast<const s16x8*>(lds + plane * PLANE + r * STRIDE + (((ks * 2 + (lane >> 5)) ^ sw) << 3));
        } else {
            const unsigned a = (unsigned)(size_t)(lds + plane * PLANE) +
                               2u * (unsigned)((ks * 16 + 8 * (lane >> 5) + ((lane & 15) >> 2)) * STRIDE + base + 16 * ((lane >> 4) & 1) + 4 * (lane & 3));
            const s16x4 lo = read_tr4(a), hi = read_tr4(a + 8 * STRIDE);
            v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return __builtin_bit_cast(frag, v);
    }
};

template <typename T, int LA, int LB, int FMT, bool VEC, int OUT, int WM, int WN, int IM, int IN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(Operand A, Operand B, int64_t K, int64_t k_per_split, Epilogue ep) {
    constexpr int THREADS = 64 * WM * WN, TM = WM * IM * 32, TN = WN * IN * 32, BK = sizeof(T) == 4 ? 32 : 64;
    typedef Tile<T, LA, 0, VEC, TM, BK, THREADS> TA;
    typedef Tile<T, LB, FMT, VEC, TN, BK, THREADS> TB;
    constexpr int BUF = TA::HALFS + TB::HALFS;
    extern __shared__ __attribute__((aligned(16))) short smem[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    const int64_t m0 = (int64_t)blockIdx.x * TM, n0 = (int64_t)blockIdx.y * TN;
    const int64_t kb = (int64_t)blockIdx.z * k_per_split, ke = kb + k_per_split < K ? kb + k_per_split : K;
    f32x16 acc[IM][IN];
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    TA a;
    TB b;
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
        const short *la = smem + buf * BUF, *lb = la + TA::HALFS;
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
            a.store(smem + (buf ^ 1) * BUF);
            b.store(smem + (buf ^ 1) * BUF + TA::HALFS);
        }
        __syncthreads();
    }
    // a lane holds column lane & 31 of a 32 x 32 block, rows (e & 3) + 8 (e >> 2) + 4 (lane >> 5)
#pragma unroll
    for (int j = 0; j < IN; ++j) {
        const int64_t n = n0 + (wn * IN + j) * 32 + (lane & 31);
        if (n >= B.rows) continue;
        const float bias = OUT == OUT_FORWARD && ep.bias ? (float)reinterpret_cast<const T*>(ep.bias)[n] : 0.f;
#pragma unroll
        for (int i = 0; i < IM; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int64_t m = m0 + (wm * IM + i) * 32 + (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5);
                if (m >= A.rows) continue;
                float v = acc[i][j][e];
                if (OUT == OUT_SLAB) {
                    reinterpret_cast<float*>(ep.out)[((int64_t)blockIdx.z * A.rows + m) * B.rows + n] = v;
                    continue;
                }
                if (OUT == OUT_FORWARD) {
                    v += bias;
                    if (ep.z) reinterpret_cast<T*>(ep.z)[m * B.rows + n] = (T)v;
                    v = act_value(v, ep.act);
                    if (ep.res) v += (float)reinterpret_cast<const T*>(ep.res)[m * ep.ld_res + n];
                }
                reinterpret_cast<T*>(ep.out)[m * ep.ld_out + n] = (T)v;
            }
    }
}

// the slabs of a split sum, added in split order
template <typename T>
__global__ __launch_bounds__(256) void join_slabs_kernel(const float* __restrict__ slab, int64_t n, int splits, T* __restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < splits; ++k) s += slab[k * n + i];
        out[i] = (T)s;
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
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float v = (float)g.v[i] * act_slope((float)t.v[i], act);
                    sum[i] += v;
                    g.v[i] = (T)v;
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

constexpr int TILE = 128;

int64_t splits_for(int64_t M, int64_t N, int64_t K, int bk) {
    // enough workgroups for two on every compute unit, at least eight steps of the sum in each
    const int64_t tiles = ((M + TILE - 1) / TILE) * ((N + TILE - 1) / TILE), steps = (K + bk - 1) / bk;
    int64_t s = 2 * (int64_t)papr_cu_count() / tiles;
    if (s > steps / 8) s = steps / 8;
    if (s > 1024) s = 1024;
    return s < 1 ? 1 : s;
}

template <typename T, int LA, int LB, int FMT, bool VEC, int OUT>
int launch_product(const Operand& A, const Operand& B, int64_t K, int64_t splits, const Epilogue& ep, hipStream_t s) {
    constexpr int WM = 2, WN = 2, IM = 2, IN = 2, BK = sizeof(T) == 4 ? 32 : 64;
    typedef Tile<T, LA, 0, VEC, TILE, BK, 256> TA;
    typedef Tile<T, LB, FMT, VEC, TILE, BK, 256> TB;
    constexpr size_t lds = 2 * (TA::HALFS + TB::HALFS) * 2;
    auto kernel = product_kernel<T, LA, LB, FMT, VEC, OUT, WM, WN, IM, IN>;
    const int64_t steps = (K + BK - 1) / BK, per = (steps + splits - 1) / splits * BK;
    const dim3 grid((unsigned)((A.rows + TILE - 1) / TILE), (unsigned)((B.rows + TILE - 1) / TILE), (unsigned)((K + per - 1) / per));
    static std::atomic<uint64_t> ready{0};            // (devices on which this kernel may already use more than 64 KB of LDS)
    int dev = 0;
    (void)hipGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (lds > 65536 && !(ready.load(std::memory_order_relaxed) & bit)) {
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    kernel<<<grid, dim3(256), lds, s>>>(A, B, K, per, ep);
    PAPR_CHECK_LAUNCH("papr_linear product");
    return 0;
}

template <typename T, int LA, int LB, int FMT, int OUT>
int launch_aligned(bool vec, const Operand& A, const Operand& B, int64_t K, int64_t splits, const Epilogue& ep, hipStream_t s) {
    return vec ? launch_product<T, LA, LB, FMT, true, OUT>(A, B, K, splits, ep, s) : launch_product<T, LA, LB, FMT, false, OUT>(A, B, K, splits, ep, s);
}

// C = A B^T into rows of type T, the sum split where the tiles alone do not fill the chip
template <typename T, int LA, int LB, int FMT>
int rows_product(bool vec, const Operand& A, const Operand& B, int64_t K, void* out, float* slab, hipStream_t s) {
    constexpr int BK = sizeof(T) == 4 ? 32 : 64;
    const int64_t steps = (K + BK - 1) / BK;
    int64_t splits = slab ? splits_for(A.rows, B.rows, K, BK) : 1;
    const int64_t per = (steps + splits - 1) / splits;
    splits = (steps + per - 1) / per;
    Epilogue ep = {};
    if (splits == 1) {
        ep.out = out;
        ep.ld_out = B.rows;
        return launch_aligned<T, LA, LB, FMT, OUT_ROWS>(vec, A, B, K, 1, ep, s);
    }
    ep.out = slab;
    if (int rc = launch_aligned<T, LA, LB, FMT, OUT_SLAB>(vec, A, B, K, splits, ep, s)) return rc;
    const int64_t n = A.rows * B.rows, need = (n + 255) / 256, cap = (int64_t)papr_cu_count() * 16;
    join_slabs_kernel<T><<<dim3((unsigned)(need < cap ? need : cap)), dim3(256), 0, s>>>(slab, n, (int)splits, (T*)out);
    PAPR_CHECK_LAUNCH("papr_linear slabs");
    return 0;
}

// float32 slabs of a weight gradient (N, K) summed over M rows
size_t slab_floats(int type, int64_t M, int64_t N, int64_t K) {
    const int64_t s = splits_for(N, K, M, type == PAPR_TYPE_F32 ? 32 : 64);
    return s > 1 ? (size_t)(s * N * K) : 0;
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
    const Epilogue ep = {y, d->N, bias, res, ld_res, z, d->act};
    PAPR_TYPE_SWITCH(d->type, return launch_aligned<T, K_RUNS, K_RUNS, 0, OUT_FORWARD>(vec, A, B, d->K, 1, ep, as_stream(stream)));
}

extern "C" size_t papr_linear_bwd_workspace_bytes(const papr_linear_desc* d) {
    if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0 || !papr_type_ok(d->type)) return 0;
    const size_t dz = d->act == PAPR_ACT_NONE ? 0 : up16((size_t)d->M * d->N * papr_type_bytes(d->type));
    size_t part = 0;
    for (int piece = 1; piece <= 8; piece *= 2) {
        const size_t p = (size_t)slope_grid(d->M, (int)d->N, piece).blocks * d->N * sizeof(float);
        part = p > part ? p : part;
    }
    return dz + up16(part) + slab_floats(d->type, d->M, d->N, d->K) * sizeof(float);
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
        PAPR_TYPE_SWITCH(d->type, rc = (rows_product<T, K_RUNS, ROWS_RUN, 0>(vec, A, B, N, d_x, nullptr, s)));
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
