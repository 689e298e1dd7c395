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

// d_z of 16-bit rows is two values of their type (linear_kernels.h says why), but for none and relu, whose d_z is d_y or zero: exact in one.
bool is_pair(const papr_linear_desc* d) { return d->type != PAPR_TYPE_F32 && d->act != PAPR_ACT_NONE && d->act != PAPR_ACT_RELU; }

// Rows of 16-bit values whose width is no multiple of eight start anywhere, and the streaming kernels want them on 16 bytes: where a product is long enough, its operands
// are copied into rows of whole vectors first (zeros behind the end).  20,000 x 701 -> 500 forward: 94 us through registers, 39 streaming, the copies 14.
int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
double copy_us(int64_t rows, int64_t width) { return 3.0 + (double)rows * width * 4 / 4e6; }
bool pads_forward(const papr_linear_desc* d) {
    if (d->type == PAPR_TYPE_F32 || d->K % 8 == 0 || d->M <= 256) return false;
    return choose(d->M, d->N, d->K, PATH_STREAM, false).us + copy_us(d->M, d->K) + copy_us(d->N, d->K) < choose(d->M, d->N, d->K, PATH_REGISTERS, false).us;
}
// the backward pass's two products: what each gains by it, its own copies counted (d_z leaves the slope kernel padded; where there is none, d_y is copied)
bool pads_rows(const papr_linear_desc* d) {
    if (d->type == PAPR_TYPE_F32 || (d->K % 8 == 0 && d->N % 8 == 0)) return false;
    const double copies = (d->K % 8 ? copy_us(d->N, d->K) : 0) + (d->act == PAPR_ACT_NONE && d->N % 8 ? copy_us(d->M, d->N) : 0);
    return choose(d->M, d->K, d->N, path_of(d->type, true, 0, is_pair(d)), true).us + copies < choose(d->M, d->K, d->N, path_of(d->type, false, 0, is_pair(d)), true).us;
}
bool pads_weight(const papr_linear_desc* d) {
    if (d->type == PAPR_TYPE_F32 || d->keep || (d->K % 8 == 0 && d->N % 8 == 0)) return false;
    const double copies = (d->K % 8 ? copy_us(d->M, d->K) : 0) + (d->act == PAPR_ACT_NONE && d->N % 8 ? copy_us(d->M, d->N) : 0);
    return choose(d->N, d->K, d->M, path_of(d->type, true, 0, is_pair(d)), true).us + copies < choose(d->N, d->K, d->M, path_of(d->type, false, 0, is_pair(d)), true).us;
}

// rows of `width` 16-bit values to rows of up8(width): eight a lane, one or two sets of rows of one width in a launch
struct Rows { const uint16_t* x; int64_t ld, rows; uint16_t* out; };
__global__ __launch_bounds__(256) void pad_rows_kernel(Rows a, Rows b, int width, int pieces) {
    const Rows p = blockIdx.y ? b : a;
    const int lanes = pieces < 256 ? pieces : 256, per = 256 / lanes;
    const int r = threadIdx.x / lanes, c0 = threadIdx.x % lanes;
    if (r >= per) return;
    for (int64_t m = (int64_t)blockIdx.x * per + r; m < p.rows; m += (int64_t)gridDim.x * per)
        for (int c = c0; c < pieces; c += lanes) {
            const uint16_t* src = p.x + m * p.ld + c * 8;
            papr_pack<uint16_t, 8> t;
            if (c * 8 + 8 <= width) __builtin_memcpy(&t, src, 16);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) t.v[i] = c * 8 + i < width ? src[i] : (uint16_t)0;
            *reinterpret_cast<papr_pack<uint16_t, 8>*>(p.out + (m * pieces + c) * 8) = t;
        }
}
int pad_rows(const Rows& a, const Rows* b, int64_t width, hipStream_t s) {
    const int64_t pieces = up8(width) / 8, per = pieces < 256 ? 256 / pieces : 1, most = b && b->rows > a.rows ? b->rows : a.rows, need = (most + per - 1) / per,
                  cap = (int64_t)papr_cu_count() * 16;
    pad_rows_kernel<<<dim3((unsigned)(need < cap ? need : cap), b ? 2 : 1), 256, 0, s>>>(a, b ? *b : a, (int)width, (int)pieces);
    PAPR_CHECK_LAUNCH("papr_linear rows");
    return 0;
}

int linear_check(const char* who, int type, int64_t M, int64_t N, int64_t K, int act) {
    PAPR_REQUIRE(papr_type_ok(type), "%s: unknown row type %d", who, type);
    PAPR_REQUIRE(M >= 0 && N >= 1 && K >= 1 && N <= (1 << 20) && K <= (1 << 20), "%s: M %lld, N %lld, K %lld", who, (long long)M, (long long)N, (long long)K);
    PAPR_REQUIRE(M < (int64_t)1 << 31, "%s: %lld rows", who, (long long)M);
    PAPR_REQUIRE(act >= PAPR_ACT_NONE && act <= PAPR_ACT_SILU, "%s: unknown activation %d", who, act);
    return 0;
}
// (a tile's rows lie at 32-bit offsets from its first: 256 rows of float32)
bool stride_ok(int64_t ld, int64_t width) { return ld >= width && ld <= PAPR_LINEAR_MAX_STRIDE; }

}  // namespace

extern "C" size_t papr_linear_fwd_workspace_bytes(const papr_linear_desc* d) {
    if (!d || d->M <= 0 || d->N <= 0 || d->K <= 0 || !papr_type_ok(d->type) || !pads_forward(d)) return 0;
    return (size_t)(d->M + d->N) * up8(d->K) * 2;
}

extern "C" int papr_linear_fwd(const papr_linear_desc* d, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* res, int64_t ld_res,
                               void* y, void* z, void* workspace, papr_stream_t stream) {
    PAPR_REQUIRE(d, "papr_linear_fwd: no descriptor");
    if (int rc = linear_check("papr_linear_fwd", d->type, d->M, d->N, d->K, d->act)) return rc;
    if (d->M == 0) return 0;
    PAPR_REQUIRE(x && w && y, "papr_linear_fwd: a pointer is missing");
    PAPR_REQUIRE(stride_ok(ldx, d->K) && stride_ok(ldw, d->K), "papr_linear_fwd: row strides %lld, %lld (%lld .. %d)", (long long)ldx, (long long)ldw, (long long)d->K,
                 PAPR_LINEAR_MAX_STRIDE);
    PAPR_REQUIRE(!res || d->M == 1 || ld_res >= d->N, "papr_linear_fwd: the residual's row stride %lld does not cover %lld columns", (long long)ld_res, (long long)d->N);
    const int b = papr_type_bytes(d->type);
    bool vec = papr_rows_aligned(x, ldx, d->K, b) && papr_rows_aligned(w, ldw, d->K, b);
    Operand A = {x, ldx, d->M, nullptr}, B = {w, ldw, d->N, nullptr};
    if (pads_forward(d)) {
        PAPR_REQUIRE(workspace && ((uintptr_t)workspace & 15) == 0, "papr_linear_fwd: the workspace is missing or does not start on 16 bytes");
        const int64_t ld = up8(d->K);
        char* wide_w = (char*)workspace + (size_t)d->M * ld * 2;
        const Rows rows = {(const uint16_t*)x, ldx, d->M, (uint16_t*)workspace}, weight = {(const uint16_t*)w, ldw, d->N, (uint16_t*)wide_w};
        if (int rc = pad_rows(rows, &weight, d->K, as_stream(stream))) return rc;
        A = {workspace, ld, d->M, nullptr};
        B = {wide_w, ld, d->N, nullptr};
        vec = true;
    }
    const Epilogue ep = {y, bias, res, ld_res, z, d->act,
                         papr_rows_aligned(y, d->N, d->N, b) && (!z || ((uintptr_t)z & 15) == 0) && (!res || papr_rows_aligned(res, ld_res, d->N, b))};
    PAPR_TYPE_SWITCH(d->type, return forward<T>(A, B, d->K, vec, ep, as_stream(stream)));
}

namespace {

// what the backward pass keeps in its workspace, in this order
struct Layout { size_t d_z, part, d_y, x, w, slab, total; int64_t ldz, low; };
Layout layout_of(const papr_linear_desc* d) {
    Layout l = {};
    const bool slope = d->act != PAPR_ACT_NONE, rows = pads_rows(d), weight = pads_weight(d);
    l.ldz = rows || weight ? up8(d->N) : d->N;
    l.d_z = slope ? up16((size_t)d->M * l.ldz * papr_type_bytes(d->type)) : 0;
    if (is_pair(d)) { l.low = (int64_t)l.d_z; l.d_z *= 2; }
    for (int piece = 1; piece <= 8; piece *= 2) {
        const size_t p = up16((size_t)slope_grid(d->M, (int)up8(d->N), piece).blocks * d->N * sizeof(float));
        l.part = p > l.part ? p : l.part;
    }
    l.d_y = !slope && (rows || weight) && d->N % 8 ? up16((size_t)d->M * l.ldz * 2) : 0;
    l.x = weight && d->K % 8 ? up16((size_t)d->M * up8(d->K) * 2) : 0;
    l.w = rows && d->K % 8 ? up16((size_t)d->N * up8(d->K) * 2) : 0;
    const size_t sx = slab_floats(d->type, d->M, d->K, d->N), sw = slab_floats(d->type, d->N, d->K, d->M);
    l.slab = up16((sx > sw ? sx : sw) * sizeof(float));
    l.total = l.d_z + l.part + l.d_y + l.x + l.w + l.slab;
    return l;
}

}  // namespace

extern "C" size_t papr_linear_bwd_workspace_bytes(const papr_linear_desc* d) {
    return !d || d->M <= 0 || d->N <= 0 || d->K <= 0 || !papr_type_ok(d->type) ? 0 : layout_of(d).total;
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
    PAPR_REQUIRE(stride_ok(ld_dy, N) && (!d_x || stride_ok(ldw, K)) && (!d_w || d->keep || stride_ok(ldx, K)), "papr_linear_bwd: row strides (at most %d)", PAPR_LINEAR_MAX_STRIDE);
    PAPR_REQUIRE(!d_w || !d->keep || (ldx == (K + 31) / 32 * 32 && ((uintptr_t)x & 7) == 0), "papr_linear_bwd: kept rows are whole blocks of 32 codes on 8 bytes");
    PAPR_REQUIRE(((uintptr_t)workspace & 15) == 0, "papr_linear_bwd: the workspace starts on 16 bytes");
    const int b = papr_type_bytes(d->type);
    const bool slope = d->act != PAPR_ACT_NONE;
    const Layout l = layout_of(d);
    char* at = reinterpret_cast<char*>(workspace);
    auto take = [&](size_t bytes) { char* p = at; at += bytes; return (void*)p; };
    void* dz = take(l.d_z);
    float* part = (float*)take(l.part);
    void *y8 = take(l.d_y), *x8 = take(l.x), *w8 = take(l.w);
    float* slab = (float*)take(l.slab);
    int rc = 0;
    if (slope || d_b) {
        const bool vec = papr_rows_aligned(d_y, ld_dy, N, b) && ((uintptr_t)z & 15) == 0;
        const SlopeGrid g = slope_grid(M, (int)(vec ? N : up8(N)), vec ? 16 / b : 1);
        PAPR_TYPE_SWITCH(d->type, rc = slopes<T>(vec, g, d_y, ld_dy, z, M, (int)N, d->act, slope ? dz : nullptr, l.low, l.ldz, d_b ? part : nullptr, s));
        if (rc) return rc;
        if (d_b) {
            papr_colsum_out out = {};
            out.p[0] = d_b;
            out.type[0] = d->type;
            if ((rc = papr_colsum_reduce(part, g.blocks, (int)N, 1, out, s))) return rc;
        }
    }
    // d_z as the products take it: from the slope kernel, or d_y itself, copied where its rows have to start on 16 bytes
    Operand G = {slope ? dz : d_y, slope ? l.ldz : ld_dy, 0, nullptr, l.low};
    if (l.d_y && (d_x || d_w)) {
        if ((rc = pad_rows({(const uint16_t*)d_y, ld_dy, M, (uint16_t*)y8}, nullptr, N, s))) return rc;
        G = {y8, l.ldz, 0, nullptr};
    }
    // the weight and the rows, where their products want them copied too
    const Rows weight = {(const uint16_t*)w, ldw, N, (uint16_t*)w8}, rows = {(const uint16_t*)x, ldx, M, (uint16_t*)x8};
    const bool copy_w = d_x && l.w, copy_x = d_w && l.x;
    if (copy_w || copy_x)
        if ((rc = pad_rows(copy_x ? rows : weight, copy_x && copy_w ? &weight : nullptr, K, s))) return rc;
    const bool vg = papr_rows_aligned(G.p, G.ld, G.ld == l.ldz ? l.ldz : N, b);
    if (d_x) {
        Operand A = G, B = {w, ldw, K, nullptr};
        A.rows = M;
        bool vec = vg && papr_rows_aligned(w, ldw, K, b);
        if (l.w) {
            B = {w8, up8(K), K, nullptr};
            vec = vg;
        }
        PAPR_TYPE_SWITCH(d->type, rc = grad_rows<T>(vec, A, B, N, d_x, slab, s));
        if (rc) return rc;
    }
    if (d_w) {
        Operand A = G, B = {x, ldx, K, (const uint8_t*)exps};
        A.rows = N;
        bool vec = vg && (d->keep || papr_rows_aligned(x, ldx, K, b));
        if (l.x) {
            B = {x8, up8(K), K, nullptr};
            vec = vg;
        }
        PAPR_TYPE_SWITCH(d->type, rc = grad_weight<T>(d->keep, vec, A, B, M, d_w, slab, s));
        if (rc) return rc;
    }
    return 0;
}
