// Rows kept in 8 bits: every 32 columns of a row share a power-of-two scale, 2^e = the smallest with max|x| <= top 2^e, and hold codes x / 2^e rounded
// to nearest (ties to even) -- e4m3 (top 448: four significant bits, exponents down to 2^-6) or int8 (top 127).  A power of two, so that the division is
// exact and a code times its scale has at most 8 significant bits: exact in every row type and a matrix operand as it is.
//   * e >= -120; magnitudes beyond the largest value the row type can hold with the format's significant bits (1.875 / 1.984375 times 2^15 in float16,
//     times 2^127 in the others) are kept as that value -- rounding up would give infinity;  NaN and infinities are kept as NaN (int8: code -128).
//   * layout: codes (rows, ceil(width / 32) * 32) bytes, the padding zero; exponents (rows, ceil(width / 32)) bytes, e + 127.
// Bound by HBM (one read of the rows, one write of 33/32 bytes an element, and back).  Four lanes hold a block, eight columns each: the maximum over a block is
// two DPP steps, a lane writes eight codes at once.  512,000 x 256 bf16 to e4m3 86 us, back 64 (together 5.2 TB/s); odd rows, 16 bytes at any address: 320,000 x 117
// float32 28 us to e4m3 (67 value by value), back 68 (91).
#include "block_types.h"

namespace {

template <int FMT, typename T>
__device__ __forceinline__ float keep_limit() {
    const float top = FMT == PAPR_KEEP_E4M3 ? 1.875f : 1.984375f;
    return __is_same(T, f16) ? top * 0x1p15f : top * 0x1p127f;
}

template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void pack_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows, int width, int blocks, uint8_t* __restrict__ codes,
                                                        uint8_t* __restrict__ exps) {
    const int64_t n = rows * blocks * 4;
    const float limit = keep_limit<FMT, T>();
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < n; u += (int64_t)gridDim.x * 256) {      // (n is a multiple of 4: a block's lanes stay together)
        const int64_t blk = u >> 2, row = blk / blocks;
        const int b = (int)(blk - row * blocks), col = b * 32 + (int)(u & 3) * 8;
        const T* src = x + row * ldx + col;
        float v[8];
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int c = 0; c < 8 / V; ++c) {
            papr_pack<T, V> t;
            const int left = width - (col + c * V);
            if (left > 0) papr_get<!VEC>(t, src + c * V, left);
#pragma unroll
            for (int i = 0; i < V; ++i) v[c * V + i] = left > 0 ? (float)t.v[i] : 0.f;
        }
        float peak = 0.f;
        unsigned bad = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!(fabsf(v[i]) <= 3.402823466e38f)) { bad |= 1u << i; v[i] = 0.f; }
            v[i] = fminf(fmaxf(v[i], -limit), limit);
            peak = fmaxf(peak, fabsf(v[i]));
        }
        peak = fmaxf(peak, PAPR_DPP_F(peak, 0xB1));
        peak = fmaxf(peak, PAPR_DPP_F(peak, 0x4E));
        const unsigned bits = __float_as_uint(peak);
        constexpr int TOP_E = FMT == PAPR_KEEP_E4M3 ? 8 : 6;
        constexpr unsigned TOP_F = FMT == PAPR_KEEP_E4M3 ? 0x600000u : 0x7E0000u;
        int e = (int)(bits >> 23) - 127 - TOP_E + ((bits & 0x7FFFFFu) > TOP_F ? 1 : 0);
        e = e < -120 ? -120 : e;
        const float inv = __uint_as_float((unsigned)(127 - e) << 23);
        unsigned w[2];
        if (FMT == PAPR_KEEP_E4M3) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * inv, v[4 * h + 1] * inv, 0, false);
                p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * inv, v[4 * h + 3] * inv, p, true);
                w[h] = (unsigned)p;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[h] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) w[h] |= ((unsigned)(int)rintf(v[4 * h + i] * inv) & 255u) << (8 * i);
            }
        }
        if (bad) {
            const unsigned nan = FMT == PAPR_KEEP_E4M3 ? 0x7Fu : 0x80u;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (bad >> i & 1) w[i >> 2] = (w[i >> 2] & ~(255u << (8 * (i & 3)))) | nan << (8 * (i & 3));
        }
        *reinterpret_cast<uint2*>(codes + blk * 32 + (u & 3) * 8) = make_uint2(w[0], w[1]);
        if ((u & 3) == 0) exps[blk] = (uint8_t)(e + 127);
    }
}

template <typename T, int FMT, bool VEC>
__global__ __launch_bounds__(256) void unpack_rows_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, int64_t rows, int width, int blocks,
                                                          T* __restrict__ x) {
    const int64_t n = rows * blocks * 4;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < n; u += (int64_t)gridDim.x * 256) {
        const int64_t blk = u >> 2, row = blk / blocks;
        const int b = (int)(blk - row * blocks), col = b * 32 + (int)(u & 3) * 8;
        const uint2 w = *reinterpret_cast<const uint2*>(codes + blk * 32 + (u & 3) * 8);
        const float scale = __uint_as_float((unsigned)exps[blk] << 23);
        float v[8];
        papr_codes_to_float<FMT>(w.x, scale, v);
        papr_codes_to_float<FMT>(w.y, scale, v + 4);
        T* dst = x + row * width + col;
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int c = 0; c < 8 / V; ++c) {
            papr_pack<T, V> t;
            const int left = width - (col + c * V);
#pragma unroll
            for (int i = 0; i < V; ++i) t.v[i] = (T)v[c * V + i];
            if (left > 0) papr_put<!VEC>(dst + c * V, t, left);
        }
    }
}

unsigned rows8_grid(int64_t rows, int blocks) {
    const int64_t need = (rows * blocks * 4 + 255) / 256, cap = (int64_t)papr_cu_count() * 32;
    return (unsigned)(need < cap ? need : cap);
}

}  // namespace

extern "C" int papr_rows8_pack(int32_t type, int32_t fmt, const void* x, int64_t ldx, int64_t rows, int32_t width, void* codes, void* exps, papr_stream_t stream) {
    PAPR_REQUIRE(papr_type_ok(type) && (fmt == PAPR_KEEP_E4M3 || fmt == PAPR_KEEP_INT8), "papr_rows8_pack: unknown type %d or format %d", type, fmt);
    PAPR_REQUIRE(rows >= 0 && width >= 1 && width <= PAPR_ROWS8_MAX_WIDTH, "papr_rows8_pack: rows %lld, width %d (1 .. %d)", (long long)rows, width, PAPR_ROWS8_MAX_WIDTH);
    PAPR_REQUIRE(rows <= 1 || ldx >= width, "papr_rows8_pack: row stride %lld does not cover %d columns", (long long)ldx, width);
    if (rows == 0) return 0;
    PAPR_REQUIRE(x && codes && exps, "papr_rows8_pack: a pointer is missing");
    PAPR_REQUIRE(((uintptr_t)codes & 7) == 0, "papr_rows8_pack: the codes start on 8 bytes");
    const int blocks = (width + 31) / 32;
    const unsigned grid = rows8_grid(rows, blocks);
    hipStream_t s = as_stream(stream);
    const bool vec = papr_rows_aligned(x, ldx, width, papr_type_bytes(type));
    PAPR_TYPE_SWITCH(type, {
        if (fmt == PAPR_KEEP_E4M3) {
            if (vec) pack_rows_kernel<T, PAPR_KEEP_E4M3, true><<<grid, 256, 0, s>>>((const T*)x, ldx, rows, width, blocks, (uint8_t*)codes, (uint8_t*)exps);
            else pack_rows_kernel<T, PAPR_KEEP_E4M3, false><<<grid, 256, 0, s>>>((const T*)x, ldx, rows, width, blocks, (uint8_t*)codes, (uint8_t*)exps);
        } else {
            if (vec) pack_rows_kernel<T, PAPR_KEEP_INT8, true><<<grid, 256, 0, s>>>((const T*)x, ldx, rows, width, blocks, (uint8_t*)codes, (uint8_t*)exps);
            else pack_rows_kernel<T, PAPR_KEEP_INT8, false><<<grid, 256, 0, s>>>((const T*)x, ldx, rows, width, blocks, (uint8_t*)codes, (uint8_t*)exps);
        }
    });
    PAPR_CHECK_LAUNCH("papr_rows8_pack");
    return 0;
}

extern "C" int papr_rows8_unpack(int32_t type, int32_t fmt, const void* codes, const void* exps, int64_t rows, int32_t width, void* x, papr_stream_t stream) {
    PAPR_REQUIRE(papr_type_ok(type) && (fmt == PAPR_KEEP_E4M3 || fmt == PAPR_KEEP_INT8), "papr_rows8_unpack: unknown type %d or format %d", type, fmt);
    PAPR_REQUIRE(rows >= 0 && width >= 1 && width <= PAPR_ROWS8_MAX_WIDTH, "papr_rows8_unpack: rows %lld, width %d (1 .. %d)", (long long)rows, width, PAPR_ROWS8_MAX_WIDTH);
    if (rows == 0) return 0;
    PAPR_REQUIRE(x && codes && exps, "papr_rows8_unpack: a pointer is missing");
    PAPR_REQUIRE(((uintptr_t)codes & 7) == 0, "papr_rows8_unpack: the codes start on 8 bytes");
    const int blocks = (width + 31) / 32;
    const unsigned grid = rows8_grid(rows, blocks);
    hipStream_t s = as_stream(stream);
    const bool vec = papr_rows_aligned(x, width, width, papr_type_bytes(type));
    PAPR_TYPE_SWITCH(type, {
        if (fmt == PAPR_KEEP_E4M3) {
            if (vec) unpack_rows_kernel<T, PAPR_KEEP_E4M3, true><<<grid, 256, 0, s>>>((const uint8_t*)codes, (const uint8_t*)exps, rows, width, blocks, (T*)x);
            else unpack_rows_kernel<T, PAPR_KEEP_E4M3, false><<<grid, 256, 0, s>>>((const uint8_t*)codes, (const uint8_t*)exps, rows, width, blocks, (T*)x);
        } else {
            if (vec) unpack_rows_kernel<T, PAPR_KEEP_INT8, true><<<grid, 256, 0, s>>>((const uint8_t*)codes, (const uint8_t*)exps, rows, width, blocks, (T*)x);
            else unpack_rows_kernel<T, PAPR_KEEP_INT8, false><<<grid, 256, 0, s>>>((const uint8_t*)codes, (const uint8_t*)exps, rows, width, blocks, (T*)x);
        }
    });
    PAPR_CHECK_LAUNCH("papr_rows8_unpack");
    return 0;
}
