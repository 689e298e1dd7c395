// The C entry points of the linear layers (the mathematics and the kernels: linear_kernels.h).
#include "linear.h"

using namespace papr_linear;

namespace {

// float32 slabs of one product
size_t slab_floats(int type, int64_t M, int64_t N, int64_t K) {
    size_t most = 0;                                  // (the path, and with it the choice, depends on alignments that the workspace's size does not know)
    for (int path = 0; path < PATHS; ++path) {
        if ((type == PAPR_TYPE_F32) != (path == PATH_F32 || path == PATH_F32_ODD || path == PATH_F32_KEPT)) continue;
        const int64_t parts = choose(M, N, K, path, true).parts;
        if (parts > 1 && (size_t)(parts * M * N) > most) most = (size_t)(parts * M * N);
    }
    return most;
}

SlopeGrid slope_grid(int64_t M, int N, int piece) {
    SlopeGrid g;
    const int groups = (N + piece - 1) / piece;
    g.lanes = 1;
    while (g.lanes < groups && g.lanes < 256) g.lanes *= 2;
    g.cols = (unsigned)((groups + g.lanes - 1) / g.lanes);
    const int64_t per = 256 / g.lanes;
    int64_t blocks = (M + 8 * per - 1) / (8 * per), cap = (int64_t)papr_cu_count() * 4 / g.cols;
    if (cap < 1) cap = 1;
    if (blocks > cap) blocks = cap;
    g.rows_per_block = (M + blocks - 1) / blocks;
    g.blocks = (M + g.rows_per_block - 1) / g.rows_per_block;
    return g;
}

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// d_z of 16-bit rows is rounded to their type in front of its two products, an error of the gradients' own rounding's size (together 1.4 times it).  Where the products
// are over in a few microseconds whatever they multiply (2^28 terms: 5 us at a fifth of the matrix pipe's rate) that is not paid for: d_z stays in float32 and the
// products take it as the sum of two 16-bit values.  (none and relu: d_z is d_y or zero and needs no rounding.)
bool keeps_wide(const papr_linear_desc* d) {
    return d->type != PAPR_TYPE_F32 && d->act != PAPR_ACT_NONE && d->act != PAPR_ACT_RELU && (double)d->M * (double)d->N * (double)d->K <= 268435456.0;
}

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
    PAPR_TYPE_SWITCH(d->type, return forward<T>(A, B, d->K, vec, ep, as_stream(stream)));
}

extern "C" size_t papr_linear_bwd_workspace_bytes(const papr_linear_desc* d) {
    if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0 || !papr_type_ok(d->type)) return 0;
    const size_t dz = d->act == PAPR_ACT_NONE ? 0 : up16((size_t)d->M * d->N * (keeps_wide(d) ? 4 : papr_type_bytes(d->type)));
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
    const bool slope = d->act != PAPR_ACT_NONE, wide = keeps_wide(d);
    char* ws = reinterpret_cast<char*>(workspace);
    void* dz = slope ? ws : nullptr;
    if (slope) ws += up16((size_t)M * N * (wide ? 4 : b));
    float* part = reinterpret_cast<float*>(ws);
    if (slope || d_b) {
        const bool vec = papr_rows_aligned(d_y, ld_dy, N, b) && ((uintptr_t)z & 15) == 0;
        const SlopeGrid g = slope_grid(M, (int)N, vec ? 16 / b : 1);
        int rc = 0;
        PAPR_TYPE_SWITCH(d->type, rc = slopes<T>(wide, vec, g, d_y, ld_dy, z, M, (int)N, d->act, dz, d_b ? part : nullptr, s));
        if (rc) return rc;
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
    const bool vg = papr_rows_aligned(g, ldg, N, wide ? 4 : b);
    if (d_x) {
        const Operand A = {g, ldg, M, nullptr}, B = {w, ldw, K, nullptr};
        const bool vec = vg && papr_rows_aligned(w, ldw, K, b);
        int rc = 0;
        PAPR_TYPE_SWITCH(d->type, rc = grad_rows<T>(wide, vec, A, B, N, d_x, slab, s));
        if (rc) return rc;
    }
    if (d_w) {
        const Operand A = {g, ldg, N, nullptr}, B = {x, ldx, K, (const uint8_t*)exps};
        const bool vec = vg && (d->keep || papr_rows_aligned(x, ldx, K, b));
        int rc = 0;
        PAPR_TYPE_SWITCH(d->type, rc = grad_weight<T>(wide, d->keep, vec, A, B, M, d_w, slab, s));
        if (rc) return rc;
    }
    return 0;
}
