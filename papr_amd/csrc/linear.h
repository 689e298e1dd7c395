// Linear layers over rows: what linear.hip (the C entry points) asks of linear_kernels.h, compiled type by type (linear_f32.hip, linear_f16.hip, linear_bf16.hip).
#pragma once
#include "block_types.h"

namespace papr_linear {

__host__ __device__ inline bool z_in_f16(int act) { return act == PAPR_ACT_GELU || act == PAPR_ACT_SILU; }       // of bfloat16 rows

struct Operand { const void* p; int64_t ld; int64_t rows; const uint8_t* exps; int64_t low = 0; };       // exps: 8-bit rows only (ld in codes); low: bytes to the second half of a pair
struct Epilogue {                                  // out and z (M, N) contiguous
    void* out;
    const void* bias; const void* res; int64_t ld_res; void* z;
    int act;
    int wide;                                      // whole 16-byte vectors in every row of out, z and res
};

// Which tile shape, and into how many parts the sum is cut: the least estimated time.  A compute unit gets q = ceil(tiles x parts / compute units) tiles; a tile costs
// its 64-term steps and a fixed part (filling the pipeline, writing the results), both measured per shape with the unit's resident workgroups sharing it; fewer
// tiles than that leave a unit waiting more (`lone`: a single tile against a full unit).  aside: bytes moved beside each result (residual, z).  Parts cost their slabs' way to memory and back and one more launch.
//                                                                                              256 x 256      128 x 128      64 x 64
//   streaming 16-bit (8192 x 4096 x 1024 and 65,536 x 1024 x 1024), us a step                    1.5            0.55          0.24
//   16-bit through registers (8191 x 1001 x 1003, 8-bit rows)                                    (slower)       1.6           0.55
//   float32 (512,000 x 256 x 256, 8192 x 4096 x 1024; 8-bit rows 1.8 / 0.9)                      10.6           2.9           1.1
//   a pair (d_z of a 16-bit layer): streaming                                                    3.0            1.1           0.5
//   a pair through registers                                                                     (slower)       2.6           0.8
enum { PATH_STREAM, PATH_REGISTERS, PATH_F32, PATH_F32_ODD, PATH_F32_KEPT, PATH_PAIR, PATH_PAIR_REGISTERS, PATHS };
struct Choice { int shape; int64_t parts, per; double us; };      // per: terms of a part
inline Choice choose(int64_t M, int64_t N, int64_t K, int path, bool may_split, int aside = 0) {
    static const int side[3] = {256, 128, 64}, resident[3] = {1, 2, 4}, first[PATHS] = {0, 1, 0, 1, 1, 0, 1};
    static const double step_us[PATHS][3] = {{1.5, 0.55, 0.24}, {0, 1.6, 0.55}, {10.6, 2.9, 1.1}, {0, 2.9, 1.1}, {0, 1.8, 0.9}, {3.0, 1.1, 0.5}, {0, 2.6, 0.8}};
    static const double fixed_us[PATHS][3] = {{9.0, 1.7, 0.5}, {0, 2.5, 1.0}, {10.0, 2.2, 1.5}, {0, 2.2, 1.5}, {0, 2.2, 1.5}, {9.0, 1.7, 0.5}, {0, 2.5, 1.0}};
    static const double lone[PATHS][3] = {{1.0, 1.3, 2.0}, {1.0, 1.8, 1.5}, {1.0, 1.5, 1.4}, {1.0, 1.5, 1.4}, {1.0, 1.5, 1.9}, {1.0, 1.3, 2.0}, {1.0, 1.8, 1.2}}, lone_fixed = 2.5;
    const int64_t cus = papr_cu_count(), steps = (K + 63) / 64;
    Choice best = {0, 1, 0, 0};
    double least = 0;
    for (int s = first[path]; s < 3; ++s) {
        const int64_t tiles = ((M + side[s] - 1) / side[s]) * ((N + side[s] - 1) / side[s]);
        const int64_t tried[4] = {1, cus / tiles, 2 * cus / tiles, 4 * cus / tiles};
        for (int64_t parts : tried) {
            if (parts > 1 && !may_split) continue;
            if (parts > steps / 2) parts = steps / 2;
            if (parts > 1024) parts = 1024;
            if (parts < 1) parts = 1;
            const int64_t per = (steps + parts - 1) / parts;
            parts = (steps + per - 1) / per;
            const int64_t q = (tiles * parts + cus - 1) / cus;
            const double alone = q < resident[s] ? (double)(resident[s] - q) / (resident[s] - 1) : 0, share = 1 + (lone[path][s] - 1) * alone;
            double t = (double)q * (step_us[path][s] * per * share + fixed_us[path][s] * (1 + (lone_fixed - 1) * alone));
            // (a tile's rows of the residual and of z: a compute unit's share of the memory is 20 KB a microsecond, and other tiles cover all of it, half of it, a fifth)
            t += (double)q * side[s] * side[s] * aside / 20e3 * (s == 0 ? 1.0 : s == 1 ? 0.5 : 0.2);
            if (parts > 1) t += (double)parts * M * N * 8 / 5e6 + 3;
            if (least == 0 || t < least) { least = t; best = {s, parts, per * 64, t}; }
        }
    }
    return best;
}
inline int aside_of(const void* res, const void* z, size_t bytes) { return ((res ? 1 : 0) + (z ? 1 : 0)) * (int)bytes; }
inline int path_of(int type, bool vec, int keep, bool pair) {
    if (type == PAPR_TYPE_F32) return keep ? PATH_F32_KEPT : vec ? PATH_F32 : PATH_F32_ODD;
    return vec && !keep ? (pair ? PATH_PAIR : PATH_STREAM) : pair ? PATH_PAIR_REGISTERS : PATH_REGISTERS;
}

// vec: every operand row starts on 16 bytes and may be read in whole vectors (what a vector holds behind the row's end is zero where the sum runs along the row).  d_z.low: d_z is a pair.
template <typename T> int forward(const Operand& x, const Operand& w, int64_t K, bool vec, const Epilogue& ep, hipStream_t s);
template <typename T> int grad_rows(bool vec, const Operand& d_z, const Operand& w, int64_t N, void* d_x, float* slab, hipStream_t s);
template <typename T> int grad_weight(int keep, bool vec, const Operand& d_z, const Operand& x, int64_t M, void* d_w, float* slab, hipStream_t s);
struct SlopeGrid { int lanes; int64_t blocks, rows_per_block; unsigned cols; };
template <typename T> int slopes(bool vec, const SlopeGrid& g, const void* d_y, int64_t ld, const void* z, int64_t M, int N, int act, void* d_z, int64_t low, int64_t ldz, float* part, hipStream_t s);

}  // namespace papr_linear
