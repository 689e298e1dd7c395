// Host side of papr_amd/blocks.py: operands as the C ABI takes them, outputs from torch's allocator, the autograd nodes.  Native because these calls are made one at a
// time -- a token's layer is a few microseconds of device work, and a training call's way through an interpreted forward and backward was longer than most of its
// kernels (25,600 x 117 float32 rows through a joint and back: 190 us of host time around 47 us of device time).  The library's entry points arrive as addresses
// (bind), so that there is one loaded library in the process.  Arguments that do not fit are answered with None; papr_amd/blocks.py says what is wrong with them.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>

#include "../../include/papr_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

namespace {

#define PAPR_ENTRY(name) decltype(&name) name##_ = nullptr
PAPR_ENTRY(papr_last_error);
PAPR_ENTRY(papr_linear_fwd);
PAPR_ENTRY(papr_linear_bwd);
PAPR_ENTRY(papr_linear_fwd_workspace_bytes);
PAPR_ENTRY(papr_linear_bwd_workspace_bytes);
PAPR_ENTRY(papr_rows8_pack);
PAPR_ENTRY(papr_rows8_unpack);
PAPR_ENTRY(papr_join_fwd);
PAPR_ENTRY(papr_join_bwd);
PAPR_ENTRY(papr_join_bwd_workspace_bytes);
#undef PAPR_ENTRY

PyObject *hip_names = nullptr, *debug_name = nullptr;      // papr_amd.hip's namespace (never released: autograd threads may outlive the interpreter's modules)

void bind(const py::dict& at, const py::object& hip) {
    if (!hip_names) {
        hip_names = py::object(hip.attr("__dict__")).release().ptr();
        debug_name = PyUnicode_InternFromString("DEBUG_SYNC");
    }
    auto take = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at[name].cast<uintptr_t>()); };
    take(papr_last_error_, "papr_last_error");
    take(papr_linear_fwd_, "papr_linear_fwd");
    take(papr_linear_bwd_, "papr_linear_bwd");
    take(papr_linear_fwd_workspace_bytes_, "papr_linear_fwd_workspace_bytes");
    take(papr_linear_bwd_workspace_bytes_, "papr_linear_bwd_workspace_bytes");
    take(papr_rows8_pack_, "papr_rows8_pack");
    take(papr_rows8_unpack_, "papr_rows8_unpack");
    take(papr_join_fwd_, "papr_join_fwd");
    take(papr_join_bwd_, "papr_join_bwd");
    take(papr_join_bwd_workspace_bytes_, "papr_join_bwd_workspace_bytes");
}

void check(int code, const char* what) {
    if (code) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(code) + "): " + papr_last_error_());
    // hip.DEBUG_SYNC: every library call named and waited for, those of the backward pass's threads too
    struct Held { PyGILState_STATE state = PyGILState_Ensure(); ~Held() { PyGILState_Release(state); } } held;
    PyObject* debug = PyDict_GetItem(hip_names, debug_name);
    if (debug && debug != Py_False && PyObject_IsTrue(debug)) py::reinterpret_borrow<py::dict>(hip_names)["check"](0, what);
}

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return PAPR_TYPE_F32;
        case at::kHalf: return PAPR_TYPE_F16;
        case at::kBFloat16: return PAPR_TYPE_BF16;
        default: return -1;
    }
}

// the library launches on the current device: the rows' own, and its current stream
struct On {
    c10::DeviceGuard guard;
    void* stream;
    explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

// These calls work on the operands' memory, once, and know the backward pass alone.  What goes another way would get the wrong answer without a word: a tangent lost, a
// recorded program without the call in it, an operand without memory taken for one that is not there.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level*/ 0).defined(); }
bool has_tangent(const Maybe& t) { return t && has_tangent(*t); }
bool stands_for(const Tensor& t) {                  // another tensor, or none: subclasses with a dispatch of their own (fake, distributed), operands of torch.func transforms
    return t.defined() && t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                                                   c10::DispatchKey::Functionalize}));
}
bool stands_for(const Maybe& t) { return t && stands_for(*t); }
bool recording() {
    using Modes = c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing()) return true;
    if (!Modes::any_modes_set()) return false;
    for (auto key : {c10::impl::TorchDispatchModeKey::PROXY, c10::impl::TorchDispatchModeKey::FAKE, c10::impl::TorchDispatchModeKey::FUNCTIONAL})
        if (Modes::get_mode(key)) return true;
    return false;
}
template <typename... Operands>
void refuse_recording(const char* who, const Operands&... operands) {
    TORCH_CHECK_NOT_IMPLEMENTED(!recording(), "papr_amd: ", who, " cannot be traced (torch.jit.trace, make_fx, torch.export): its call is not a torch operator");
    TORCH_CHECK_NOT_IMPLEMENTED(!(stands_for(operands) || ...), "papr_amd: ", who, " takes plain tensors, not a torch.func transform's or a subclass with a dispatch of its own");
}
template <typename... Operands>
void refuse_tangents(const char* who, const Operands&... operands) {
    TORCH_CHECK_NOT_IMPLEMENTED(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !(has_tangent(operands) || ...), "papr_amd: ", who,
                                " has no forward-mode derivative (an operand carries a tangent)");
}

// the values in memory (a view that torch negates lazily -- the imaginary part of a conjugate -- holds them with the other sign), outside the graph
Tensor untracked(const Tensor& t) { return (t.requires_grad() ? t.detach() : t).resolve_neg(); }

// t as (rows, width) with unit column stride and rows that do not overlap; a copy only where its strides ask for one
Tensor rows_of(const Tensor& given, int64_t width) {
    Tensor t = untracked(given);
    if (t.dim() != 2) t = t.reshape({-1, width});
    if ((width > 1 && t.stride(1) != 1) || (t.size(0) > 1 && (t.stride(0) < width || t.stride(0) > PAPR_LINEAR_MAX_STRIDE))) t = t.contiguous();
    return t;
}
int64_t ld_of(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int64_t ld_of(const Maybe& t) { return t ? ld_of(*t) : 0; }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Maybe& t) { return t ? t->data_ptr() : nullptr; }
Tensor fresh(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().requires_grad(false)); }
Tensor bytes_like(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kByte).requires_grad(false)); }
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const Maybe& t) { return t && t->requires_grad(); }
Tensor or_none(const Maybe& t) { return t ? *t : Tensor(); }

// A tensor kept for the backward pass.  Hooks of saved tensors (moved to host memory and back, recomputed) may bring back another tensor: it has to be of the same
// sizes, type and device, and its strides are seen to again.
class Kept {
    SavedVariable saved;
    at::DimVector sizes;
    at::ScalarType type = at::kByte;
    at::Device device = at::kCPU;

    Tensor checked() const {
        Tensor t = saved.unpack();
        TORCH_CHECK(!t.defined() || (t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.device() == device), "papr_amd: a saved tensor came back as ",
                    t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", was ", type, " ", at::IntArrayRef(sizes), " on ", device);
        return t.defined() ? untracked(t) : t;
    }

   public:
    void hold(const Tensor& t) {
        if (!t.defined()) return;
        saved = SavedVariable(t, false);
        sizes.assign(t.sizes().begin(), t.sizes().end());
        type = t.scalar_type();
        device = t.device();
    }
    void hold(const Maybe& t) { if (t) hold(*t); }
    void release() { saved.reset_data(); }
    Tensor rows() const { Tensor t = checked(); return t.defined() ? rows_of(t, sizes.back()) : t; }
    Tensor dense() const { Tensor t = checked(); return t.defined() ? t.contiguous() : t; }
};

// gradients of which no derivative exists: using one in a graph raises there
variable_list last_of_their_kind(variable_list grads, const char* who) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) {
            g = g.detach();
            g.set_requires_grad(true);
        }
    const size_t n = grads.size();
    return torch::autograd::DelayedError(std::string("papr_amd: ") + who + " has no second derivative", (int64_t)n).apply(std::move(grads));
}

// ------------------------------------------------------------------------------------------ rows in 8 bits
std::pair<Tensor, Tensor> pack_of(const Tensor& rows, int fmt) {
    const int64_t n = rows.size(0), width = rows.size(1), blocks = (width + 31) / 32;
    Tensor codes = bytes_like(rows, {n, blocks * 32}), exps = bytes_like(rows, {n, blocks});
    On on(rows);
    check(papr_rows8_pack_(type_of(rows), fmt, ptr(rows), ld_of(rows), n, (int32_t)width, ptr(codes), ptr(exps), on.stream), "papr_rows8_pack");
    return {codes, exps};
}

py::object pack(const Tensor& x, int fmt) {
    refuse_recording("pack_rows", x);
    if (!x.is_cuda() || type_of(x) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > PAPR_ROWS8_MAX_WIDTH) return py::none();
    auto p = pack_of(rows_of(x, x.size(-1)), fmt);
    return py::make_tuple(p.first, p.second);
}

py::object unpack(const Tensor& codes, const Tensor& exps, int fmt, int type, std::vector<int64_t> shape) {
    refuse_recording("PackedRows.rows", codes, exps);
    const at::ScalarType types[3] = {at::kFloat, at::kHalf, at::kBFloat16};
    if (fmt < 1 || type < 0 || type > 2 || shape.empty() || shape.back() < 1 || shape.back() > PAPR_ROWS8_MAX_WIDTH) return py::none();
    int64_t n = 1;
    for (size_t i = 0; i + 1 < shape.size(); ++i) n *= shape[i];
    const int64_t blocks = (shape.back() + 31) / 32;
    if (!codes.is_cuda() || exps.device() != codes.device() || codes.scalar_type() != at::kByte || exps.scalar_type() != at::kByte) return py::none();
    if (codes.sizes() != at::IntArrayRef({n, blocks * 32}) || exps.sizes() != at::IntArrayRef({n, blocks})) return py::none();
    Tensor c = codes.contiguous(), e = exps.contiguous();
    if ((uintptr_t)ptr(c) & 7) c = c.clone();
    Tensor out = at::empty(shape, c.options().dtype(types[type]));
    On on(out);
    check(papr_rows8_unpack_(type, fmt, ptr(c), ptr(e), n, (int32_t)shape.back(), ptr(out), on.stream), "papr_rows8_unpack");
    return py::cast(out);
}

// ------------------------------------------------------------------------------------------ linear layers
struct LinearBackward : Node {
    papr_linear_desc d{};
    Kept held, exps, weight, z;
    std::vector<int64_t> x_shape;

    std::string name() const override { return "PaprLinearBackward"; }
    void release_variables() override {
        held.release();
        exps.release();
        weight.release();
        z.release();
    }
    variable_list apply(variable_list&& grads) override {
        const Tensor& d_y = grads[0];
        variable_list out(4);
        if (!d_y.defined()) return out;
        refuse_recording("linear_rows", d_y);
        refuse_tangents("linear_rows", d_y);
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
        if (task_should_compute_output(3)) out[3] = d_y;
        if (need_x || need_w || need_b) {
            Tensor h = d.keep ? held.dense() : held.rows(), e = exps.dense(), w = weight.rows(), zz = z.dense(), g = rows_of(d_y, d.N);
            On on(g);
            if (need_x) out[0] = fresh(g, x_shape);
            if (need_w) out[1] = fresh(g, {d.N, d.K});
            if (need_b) out[2] = fresh(g, {d.N});
            if (d.M == 0) {
                for (int i = 0; i < 3; ++i)
                    if (out[i].defined()) out[i].zero_();
            } else {
                Tensor ws = bytes_like(g, {(int64_t)papr_linear_bwd_workspace_bytes_(&d) + 16});
                check(papr_linear_bwd_(&d, ptr(g), ld_of(g), ptr(zz), need_w ? ptr(h) : nullptr, h.defined() ? ld_of(h) : 0, ptr(e), need_x ? ptr(w) : nullptr,
                                       w.defined() ? ld_of(w) : 0, ptr(out[0]), ptr(out[1]), ptr(out[2]), ptr(ws), on.stream), "papr_linear_bwd");
            }
        }
        return last_of_their_kind(std::move(out), "linear_rows");
    }
};

bool linear_fits(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int act, int keep_fmt) {
    if (!x.is_cuda() || type_of(x) < 0 || x.dim() < 1 || w.dim() != 2 || w.scalar_type() != x.scalar_type() || w.device() != x.device() || act < 0 || keep_fmt < 0) return false;
    const int64_t K = w.size(1), N = w.size(0);
    if (K < 1 || N < 1 || x.size(-1) != K || K > (1 << 20) || N > (1 << 20)) return false;
    if (b && (b->scalar_type() != x.scalar_type() || b->device() != x.device() || b->dim() != 1 || b->size(0) != N)) return false;
    if (!r) return true;
    if (r->scalar_type() != x.scalar_type() || r->device() != x.device() || r->dim() != x.dim() || r->size(-1) != N) return false;
    return r->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1);
}

py::object linear(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int act, int keep_fmt) {
    refuse_recording("linear_rows", x, w, b, r);
    refuse_tangents("linear_rows", x, w, b, r);
    if (!linear_fits(x, w, b, r, act, keep_fmt)) return py::none();
    const int64_t K = w.size(1), N = w.size(0);
    const bool tracked = at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b) || wants_grad(r));
    Tensor rows = rows_of(x, K), w2 = rows_of(w, K);
    Maybe b1 = b ? Maybe(untracked(*b).contiguous()) : Maybe(), r2 = r ? Maybe(rows_of(*r, N)) : Maybe();
    papr_linear_desc d{};
    d.type = type_of(x);
    d.act = act;
    d.M = rows.size(0);
    d.N = N;
    d.K = K;
    const bool slopes = tracked && act != PAPR_ACT_NONE && (wants_grad(x) || wants_grad(w) || wants_grad(b));
    auto shape = x.sizes().vec();                  // (outputs in their final shape: contiguous, so the same rows)
    shape.back() = N;
    Tensor y = fresh(rows, shape), z;
    if (slopes) z = at::empty({d.M, N}, rows.options().requires_grad(false).dtype(d.type == PAPR_TYPE_BF16 && (act == PAPR_ACT_GELU || act == PAPR_ACT_SILU) ? at::kHalf : rows.scalar_type()));
    {
        On on(rows);                               // (the workspace's size is the device's)
        const size_t aside = papr_linear_fwd_workspace_bytes_(&d);
        Tensor ws = aside ? bytes_like(rows, {(int64_t)aside}) : Tensor();
        check(papr_linear_fwd_(&d, ptr(rows), ld_of(rows), ptr(w2), ld_of(w2), ptr(b1), ptr(r2), ld_of(r2), ptr(y), ptr(z), ptr(ws), on.stream), "papr_linear_fwd");
    }
    if (tracked) {
        auto node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, or_none(b), or_none(r)));
        if (wants_grad(w)) {
            if (keep_fmt) {
                auto p = pack_of(rows, keep_fmt);
                node->held.hold(p.first);
                node->exps.hold(p.second);
                d.keep = keep_fmt;
            } else node->held.hold(rows);
        }
        if (wants_grad(x)) node->weight.hold(w2);
        node->z.hold(z);
        node->d = d;
        node->x_shape = x.sizes().vec();
        torch::autograd::set_history(y, node);
    }
    return py::cast(y);
}

// ------------------------------------------------------------------------------------------ the joint of a block
struct Joint {                                     // operands as the library takes them: the descriptor points into the tensors
    Tensor x;
    Maybe f, gate, params[5];                      // scale, post gain, post shift, pre gain, pre shift
    papr_join_desc d{};

    void describe() {
        auto norm = [&](papr_block_norm& n, int at) {
            n.gain = ptr(params[at]);
            n.shift = ptr(params[at + 1]);
            n.type = params[at] ? type_of(*params[at]) : params[at + 1] ? type_of(*params[at + 1]) : 0;
        };
        d.rows = x.size(0);
        d.width = (int32_t)x.size(1);
        d.type = type_of(x);
        d.x = ptr(x);
        d.ldx = ld_of(x);
        d.f = ptr(f);
        d.ldf = ld_of(f);
        d.gate = ptr(gate);
        d.ldg = ld_of(gate);
        d.gate_form = !gate ? PAPR_GATE_ABSENT : gate->size(1) == x.size(1) ? PAPR_GATE_FULL : PAPR_GATE_ROW;
        d.scale_cols = ptr(params[0]);
        d.scale_type = params[0] ? type_of(*params[0]) : 0;
        norm(d.post, 1);
        norm(d.pre, 3);
    }
};

struct JoinBackward : Node {
    papr_join_desc d{};                            // numbers only: the pointers are set when the saved tensors are back
    bool has_h = false;
    Kept x, f, gate, stats, params[5];
    std::vector<int64_t> shape, gate_shape;

    std::string name() const override { return "PaprJoinBackward"; }
    void release_variables() override {
        x.release();
        f.release();
        gate.release();
        stats.release();
        for (auto& p : params) p.release();
    }
    variable_list apply(variable_list&& grads) override {
        variable_list out(8);
        Joint j;
        auto maybe = [](const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); };
        j.x = x.rows();
        j.f = maybe(f.rows());
        j.gate = maybe(gate.rows());
        for (int i = 0; i < 5; ++i) j.params[i] = maybe(params[i].dense());
        Tensor st = stats.dense();
        On on(j.x);
        j.d = d;
        j.describe();
        const int64_t rows = j.d.rows, width = j.d.width;
        Tensor d_y = j.f ? grads[0] : Tensor(), d_h = has_h ? grads.back() : Tensor();
        if (!d_y.defined() && !d_h.defined()) return out;
        refuse_recording("join_rows", d_y, d_h);
        refuse_tangents("join_rows", d_y, d_h);
        auto full = [&](const Tensor& t) { return t.defined() ? untracked(t).reshape({rows, width}).contiguous() : t; };
        d_y = full(d_y);
        d_h = full(d_h);
        if (task_should_compute_output(0)) out[0] = fresh(j.x, shape);
        if (j.f && task_should_compute_output(1)) out[1] = fresh(j.x, shape);
        if (j.gate && task_should_compute_output(2)) out[2] = fresh(j.x, gate_shape);
        bool sums = false;
        for (int i = 0; i < 5; ++i)                // (without d_h the next norm's are zero)
            if (j.params[i] && task_should_compute_output(3 + i)) {
                out[3 + i] = fresh(*j.params[i], {width});
                sums = true;
            }
        papr_join_grads g = {ptr(out[6]), ptr(out[7]), ptr(out[4]), ptr(out[5]), ptr(out[3])};
        Tensor ws = sums ? bytes_like(j.x, {(int64_t)papr_join_bwd_workspace_bytes_(rows, (int32_t)width) + 16}) : Tensor();
        check(papr_join_bwd_(&j.d, (const float*)ptr(st), ptr(d_y), ptr(d_h), ptr(out[0]), ptr(out[1]), ptr(out[2]), &g, ptr(ws), on.stream), "papr_join_bwd");
        return last_of_their_kind(std::move(out), "join_rows");
    }
};

bool param_fits(const Maybe& p, const Tensor& x) { return !p || (type_of(*p) >= 0 && p->device() == x.device() && p->dim() == 1 && p->size(0) == x.size(-1)); }

// pre_kind < 0: no next norm
py::object join(const Tensor& x, const Maybe& f, const Maybe& gate, double scale, const Maybe& scale_cols, int post_kind, double post_eps, const Maybe& post_gain,
                const Maybe& post_shift, int pre_kind, double pre_eps, const Maybe& pre_gain, const Maybe& pre_shift, int gate_act) {
    const char* who = f ? "join_rows" : "norm_rows";
    refuse_recording(who, x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift);
    refuse_tangents(who, x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift);
    if (!x.is_cuda() || type_of(x) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) > PAPR_JOIN_MAX_WIDTH || post_kind < 0 || gate_act < 0 || pre_kind < -1) return py::none();
    const int64_t width = x.size(-1);
    if (width < 2 && (post_kind == PAPR_NORM_LAYER || pre_kind == PAPR_NORM_LAYER)) return py::none();
    auto rows_fit = [&](const Maybe& t) { return !t || (t->scalar_type() == x.scalar_type() && t->device() == x.device()); };
    if (!rows_fit(f) || !rows_fit(gate) || (f && f->sizes() != x.sizes())) return py::none();
    if (gate && gate->sizes() != x.sizes()) {
        auto want = x.sizes().vec();
        want.back() = 1;
        if (gate->sizes() != at::IntArrayRef(want)) return py::none();
    }
    const Maybe* given[5] = {&scale_cols, &post_gain, &post_shift, &pre_gain, &pre_shift};
    bool tracked = wants_grad(x) || wants_grad(f) || wants_grad(gate);
    for (auto p : given) {
        if (!param_fits(*p, x)) return py::none();
        tracked = tracked || wants_grad(*p);
    }
    if ((post_gain && post_shift && post_gain->scalar_type() != post_shift->scalar_type()) || (pre_gain && pre_shift && pre_gain->scalar_type() != pre_shift->scalar_type())) return py::none();
    tracked = tracked && at::GradMode::is_enabled();
    Joint j;
    j.x = rows_of(x, width);
    if (f) j.f = rows_of(*f, width);
    if (gate) j.gate = rows_of(*gate, gate->size(-1));
    for (int i = 0; i < 5; ++i)
        if (*given[i]) j.params[i] = untracked(**given[i]).contiguous();
    j.d.gate_act = gate_act;
    j.d.scale = (float)scale;
    j.d.post.kind = post_kind;
    j.d.post.eps = (float)post_eps;
    j.d.pre.kind = pre_kind < 0 ? PAPR_NORM_NONE : pre_kind;
    j.d.pre.eps = (float)pre_eps;
    j.describe();
    Tensor y = f ? fresh(j.x, x.sizes()) : Tensor(), h = pre_kind >= 0 ? fresh(j.x, x.sizes()) : Tensor();
    Tensor stats = tracked ? at::empty({j.d.rows, 6}, j.x.options().dtype(at::kFloat)) : Tensor();
    {
        On on(j.x);
        check(papr_join_fwd_(&j.d, ptr(y), ptr(h), (float*)ptr(stats), on.stream), "papr_join_fwd");
    }
    if (tracked) {
        auto node = std::shared_ptr<JoinBackward>(new JoinBackward(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, or_none(f), or_none(gate), or_none(scale_cols), or_none(post_gain), or_none(post_shift), or_none(pre_gain),
                                                                 or_none(pre_shift)));
        node->d = j.d;
        node->has_h = pre_kind >= 0;
        node->x.hold(j.x);
        node->f.hold(j.f);
        node->gate.hold(j.gate);
        node->stats.hold(stats);
        for (int i = 0; i < 5; ++i) node->params[i].hold(j.params[i]);
        node->shape = x.sizes().vec();
        if (gate) node->gate_shape = gate->sizes().vec();
        if (y.defined()) torch::autograd::set_history(y, node);
        if (h.defined()) torch::autograd::set_history(h, node);
    }
    if (!y.defined()) return py::cast(h);
    if (!h.defined()) return py::cast(y);
    return py::make_tuple(y, h);
}

}  // namespace

PYBIND11_MODULE(_blocks, m) {
    m.def("bind", &bind);
    m.def("pack", &pack);
    m.def("unpack", &unpack);
    m.def("linear", &linear);
    m.def("join", &join);
}
