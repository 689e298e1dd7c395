// Element types of the row-block operators (linear.hip, join.hip, rows8.hip): rows in float32, float16 or bfloat16, arithmetic in float32.
#pragma once
#include "papr_common.h"

typedef _Float16 f16;
typedef __bf16 bf16;

template <typename T, int N>
struct alignas(sizeof(T) * N) papr_pack { T v[N]; };

// the row types behind the PAPR_TYPE_* codes: the statement sees the type as T
#define PAPR_TYPE_SWITCH(code, ...)                                                   \
    do {                                                                              \
        if ((code) == PAPR_TYPE_F32) { typedef float T; __VA_ARGS__; }                \
        else if ((code) == PAPR_TYPE_F16) { typedef f16 T; __VA_ARGS__; }             \
        else { typedef bf16 T; __VA_ARGS__; }                                         \
    } while (0)

static inline bool papr_type_ok(int t) { return t == PAPR_TYPE_F32 || t == PAPR_TYPE_F16 || t == PAPR_TYPE_BF16; }
static inline int papr_type_bytes(int t) { return t == PAPR_TYPE_F32 ? 4 : 2; }
// whole 16-byte vectors: base, row stride (elements) and width
static inline bool papr_rows_aligned(const void* p, int64_t ld, int64_t width, int bytes) {
    return ((uintptr_t)p & 15) == 0 && (ld * bytes) % 16 == 0 && (width * bytes) % 16 == 0;
}

// N elements of a row of which `left` are there (the others zero, or not written).  LOOSE: rows that start anywhere and end inside a vector -- the hardware takes 16 bytes
// at any address, and the one lane with the row's end takes its elements one by one; otherwise left >= N and the address is the vector's own.
template <bool LOOSE, typename T, int N>
__device__ __forceinline__ void papr_get(papr_pack<T, N>& t, const T* p, int left) {
    if (!LOOSE) t = *reinterpret_cast<const papr_pack<T, N>*>(p);
    else if (left >= N) __builtin_memcpy(&t, __builtin_assume_aligned(p, sizeof(T)), sizeof(t));
    else
#pragma unroll
        for (int i = 0; i < N; ++i) t.v[i] = i < left ? p[i] : (T)0.f;
}
template <bool LOOSE, typename T, int N>
__device__ __forceinline__ void papr_put(T* p, const papr_pack<T, N>& t, int left) {
    if (!LOOSE) *reinterpret_cast<papr_pack<T, N>*>(p) = t;
    else if (left >= N) __builtin_memcpy(__builtin_assume_aligned(p, sizeof(T)), &t, sizeof(t));
    else
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = t.v[i];
}

// 1 / (1 + exp(-z)), hardware exp2 and reciprocal.  EXACT (float32 rows): the exponent's product with log2(e) in two parts, a relative error of a few ulp for every z.
// Otherwise one product: |z| 2^-24 relative, far below a 16-bit type's rounding, and half the instructions (they are what an epilogue of short sums waits for).
template <bool EXACT>
__device__ __forceinline__ float papr_sigmoid(float z) {
    const float a = z * -1.44269504f;
    if (!EXACT) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a));
    const float rest = fabsf(a) < 126.f ? __builtin_fmaf(z, -1.44269504f, -a) + z * -1.92596299e-8f : 0.f;
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(a) * __builtin_fmaf(rest, 0.693147181f, 1.f));
}

// Parameters (norm gains and shifts, column scales) may be held in another type than the rows: N values from element `at` on, the type uniform.
template <int N>
__device__ __forceinline__ void load_param(float (&v)[N], const void* p, int type, int64_t at) {
    if (type == PAPR_TYPE_F32) {
        const auto t = *reinterpret_cast<const papr_pack<float, N>*>(reinterpret_cast<const float*>(p) + at);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = t.v[i];
    } else if (type == PAPR_TYPE_F16) {
        const auto t = *reinterpret_cast<const papr_pack<f16, N>*>(reinterpret_cast<const f16*>(p) + at);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t.v[i];
    } else {
        const auto t = *reinterpret_cast<const papr_pack<bf16, N>*>(reinterpret_cast<const bf16*>(p) + at);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t.v[i];
    }
}
__device__ __forceinline__ void store_param(void* p, int type, int64_t at, float v) {
    if (type == PAPR_TYPE_F32) reinterpret_cast<float*>(p)[at] = v;
    else if (type == PAPR_TYPE_F16) reinterpret_cast<f16*>(p)[at] = (f16)v;
    else reinterpret_cast<bf16*>(p)[at] = (bf16)v;
}

// Column sums left as one partial row per workgroup, part (blocks, n), added up in block order (the same bits on every run).  One workgroup takes 64
// columns; its 16 waves take strips of the blocks.
struct papr_colsum_out { void* p[5]; int32_t type[5]; };
int papr_colsum_reduce(const float* part, int64_t n_blocks, int32_t width, int32_t n_arrays, const papr_colsum_out& out, hipStream_t s);      // join.hip

// Four 8-bit codes (rows8.hip) times their block's power-of-two scale.
template <int FMT>
__device__ __forceinline__ void papr_codes_to_float(unsigned w, float scale, float* v) {
    if (FMT == PAPR_KEEP_E4M3) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        v[0] = a[0] * scale; v[1] = a[1] * scale; v[2] = b[0] * scale; v[3] = b[1] * scale;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = (int)(w << (24 - 8 * i)) >> 24;
            v[i] = c == -128 ? __uint_as_float(0x7FC00000u) : (float)c * scale;
        }
    }
}
