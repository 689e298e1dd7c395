"""Row blocks: the parts of a residual feed-forward block over rows of float32, float16 or bfloat16, each with its backward pass.

    norm_rows    h = N(x)                                                  the norm in front of a block
    linear_rows  y = act(x W^T + b) + r                                    a Linear layer with its epilogue
    join_rows    y = x + s * a(g) * N_post(f),  h = N_pre(y)               the block's end and the next block's norm in one pass
    pack_rows    rows in 8 bits, PackedRows.rows() back                    what linear_rows(keep=...) holds for its backward pass

They are what `FeedForward.forward` of the reference does around its MLP (models/attn.py:111-117: innorm, mlp, outnorm, the residual branch), for rows that are not
the render path's own: `papr_amd.ops` runs the embedding MLPs as whole chains instead.  All work goes through libpapr_hip.so (include/papr_hip.h: papr_linear_*,
papr_join_*, papr_rows8_*) on the current stream of the rows' device; there is no CPU form.  Workspaces come from torch's allocator call by call, so calls on
several streams and in several captured graphs do not share any.  Second derivatives are not defined.
"""
import collections
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import hip

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
ACTS = {"none": 0, "relu": 1, "leakyrelu": 2, "gelu": 3, "silu": 4}
KEEPS = {"e4m3": 1, "int8": 2}
NORMS = {"none": 0, "layernorm": 1, "rmsnorm": 2}
GATE_ACTS = {"none": 0, "sigmoid": 1, "silu": 2}
BLOCK = 32                                             # columns that share a scale in packed rows

# A norm over the last dimension: "layernorm" (v - mean) / (std + eps) * gain + shift with the unbiased deviation (models/attn.py:39-42), "rmsnorm"
# v / sqrt(mean(v^2) + eps) * gain (+ shift), "none" v * gain + shift.  gain and shift: (width,) tensors of one type, or None.
Norm = collections.namedtuple("Norm", ["kind", "gain", "shift", "eps"], defaults=["layernorm", None, None, 1e-6])


def _fail(who, what):
    raise ValueError("papr_amd: %s: %s" % (who, what))


def _check_rows(who, name, t, operand=False):
    if not torch.is_tensor(t):
        _fail(who, "%s is not a tensor" % name)
    if t.dtype not in TYPES:
        _fail(who, "%s has type %s (float32, float16, bfloat16)" % (name, t.dtype))
    if not operand and (t.dim() < 1 or t.shape[-1] < 1):
        _fail(who, "%s has shape %s: rows of at least one column" % (name, tuple(t.shape)))


def _check_device(who, x, *others):
    if not x.is_cuda:
        raise RuntimeError("papr_amd: %s runs only on a ROCm device (HIP); there is no CPU fallback (the rows are on %s)" % (who, x.device))
    for t in others:
        if t is not None and t.device != x.device:
            _fail(who, "a tensor is on %s, the rows on %s" % (t.device, x.device))


def _rows(t, width):
    """t as (rows, width) with unit column stride and rows that do not overlap; a copy only where its strides ask for one."""
    if t.requires_grad:
        t = t.detach()
    if t.dim() != 2:
        t = t.reshape(-1, width)
    down, across = t.stride()
    if (across != 1 and width > 1) or (down < width and t.shape[0] > 1):
        t = t.contiguous()
    return t


def _ld(t):
    return max(t.stride(0), t.shape[1])


def _p(t):
    return None if t is None else t.data_ptr()


_stream = torch._C._cuda_getCurrentRawStream


def _launch(what, dev, fn, *args):
    """fn(*args, stream) on the rows' device (the library launches on the current one) and its current stream."""
    i = dev.index
    if torch._C._cuda_getDevice() == i:
        code = fn(*args, _stream(i))
    else:
        with torch.cuda.device(i):
            code = fn(*args, _stream(i))
    if code or hip.DEBUG_SYNC:
        hip.check(code, what)


def _wants_grad(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


# ---------------------------------------------------------------------------------------------- rows in 8 bits
class PackedRows:
    """Rows in 8 bits: `codes` (rows, 32 ceil(width / 32)) uint8, `exps` (rows, ceil(width / 32)) uint8 -- columns 32 j .. 32 j + 31 of a row stand for
    code * 2^(exps[row, j] - 127) --, `fmt` "e4m3" or "int8", and the `shape` and `dtype` of what was packed."""

    def __init__(self, codes, exps, fmt, shape, dtype):
        self.codes, self.exps, self.fmt, self.shape, self.dtype = codes, exps, fmt, shape, dtype

    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def rows(self):
        """The values they stand for, in the type and shape that was packed."""
        out = torch.empty(self.shape, device=self.codes.device, dtype=self.dtype)
        _launch("papr_rows8_unpack", out.device, hip.lib().papr_rows8_unpack, TYPES[self.dtype], KEEPS[self.fmt], self.codes.data_ptr(), self.exps.data_ptr(),
                self.codes.shape[0], self.shape[-1], out.data_ptr())
        return out


def pack_rows(x, fmt="e4m3"):
    """x (..., width) -> PackedRows: 8 bits a value and one power-of-two scale for every 32 columns of a row (33/32 bytes a value).  "e4m3" keeps four significant
    bits of every value down to 2^-14 of its block's largest, "int8" seven bits below the block's largest.  NaN and infinities come back as NaN.  No gradient: this
    is how an activation is kept, not a part of the model."""
    _check_rows("pack_rows", "x", x)
    if fmt not in KEEPS:
        _fail("pack_rows", "unknown format %r (%s)" % (fmt, ", ".join(KEEPS)))
    _check_device("pack_rows", x)
    return _pack(_rows(x, x.shape[-1]), fmt, x.shape)


def _pack(rows, fmt, shape):
    n, width = rows.shape
    blocks = (width + BLOCK - 1) // BLOCK
    codes = torch.empty((n, blocks * BLOCK), device=rows.device, dtype=torch.uint8)
    exps = torch.empty((n, blocks), device=rows.device, dtype=torch.uint8)
    _launch("papr_rows8_pack", rows.device, hip.lib().papr_rows8_pack, TYPES[rows.dtype], KEEPS[fmt], rows.data_ptr(), _ld(rows), n, width, codes.data_ptr(), exps.data_ptr())
    return PackedRows(codes, exps, fmt, shape, rows.dtype)


# ---------------------------------------------------------------------------------------------- linear layers
def _linear_call(x, weight, bias, residual, act, want_z):
    """(y, z or None, descriptor) of 2-D rows"""
    M, K = x.shape
    N = weight.shape[0]
    dt, dev = x.dtype, x.device
    y = torch.empty((M, N), device=dev, dtype=dt)
    z = torch.empty((M, N), device=dev, dtype=dt) if want_z else None
    d = hip.LinearDesc(TYPES[dt], act, 0, 0, M, N, K)
    _launch("papr_linear_fwd", dev, hip.lib().papr_linear_fwd, d, x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight), _p(bias), _p(residual),
            0 if residual is None else _ld(residual), y.data_ptr(), _p(z))
    return y, z, d


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, keep):
        K, N = weight.shape[1], weight.shape[0]
        need = ctx.needs_input_grad
        rows, w2 = _rows(x, K), _rows(weight, K)
        y, z, d = _linear_call(rows, w2, None if bias is None else bias.detach().contiguous(), None if residual is None else _rows(residual, N), act,
                               act != 0 and (need[0] or need[1] or need[2]))
        packed = _pack(rows, keep, rows.shape) if keep is not None and need[1] else None
        held = None if not need[1] else rows if packed is None else packed.codes
        ctx.save_for_backward(held, None if packed is None else packed.exps, w2 if need[0] else None, z)
        if packed is not None:
            d.keep = KEEPS[keep]
        ctx.desc, ctx.shapes = d, (x.shape, weight.shape)
        return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (N,))

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        held, exps, w2, z = ctx.saved_tensors
        d = ctx.desc
        M, N, K = d.M, d.N, d.K
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        d_res = d_y if need_r else None
        if not (need_x or need_w or need_b):
            return None, None, None, d_res, None, None
        dev, dt = d_y.device, d_y.dtype
        x_shape, w_shape = ctx.shapes
        if M == 0:
            return (d_y.new_zeros(x_shape) if need_x else None, d_y.new_zeros(w_shape) if need_w else None, d_y.new_zeros(N) if need_b else None, d_res, None, None)
        g = _rows(d_y, N)
        d_x = torch.empty((M, K), device=dev, dtype=dt) if need_x else None
        d_w = torch.empty((N, K), device=dev, dtype=dt) if need_w else None
        d_b = torch.empty((N,), device=dev, dtype=dt) if need_b else None
        lib = hip.lib()
        ws = torch.empty(lib.papr_linear_bwd_workspace_bytes(d) + 16, device=dev, dtype=torch.uint8)
        _launch("papr_linear_bwd", dev, lib.papr_linear_bwd, d, g.data_ptr(), _ld(g), _p(z), _p(held), 0 if held is None else _ld(held), _p(exps), _p(w2),
                0 if w2 is None else _ld(w2), _p(d_x), _p(d_w), _p(d_b), ws.data_ptr())
        return d_x if d_x is None or len(x_shape) == 2 else d_x.reshape(x_shape), d_w, d_b, d_res, None, None


def linear_rows(x, weight, bias=None, residual=None, act="none", keep=None):
    """act(x @ weight.T + bias) + residual over the last dimension: x (..., K), weight (N, K), bias (N,), residual (..., N), all of one type (float32, float16,
    bfloat16; sums in float32, the result rounded once).  act: none, relu, leakyrelu (slope 0.2), gelu (erf form), silu.

    keep = "e4m3" / "int8": in training the rows x are held for the weight's gradient as pack_rows keeps them -- a quarter (float32) or half of the memory -- and that
    gradient is d_z^T times the values they stand for; y and every other gradient are those of keep=None.  An activation's argument is held in the rows' type.  float32
    rows with infinities give NaN."""
    if not _linear_fits(x, weight, bias, residual, act, keep):
        _explain_linear(x, weight, bias, residual, act, keep)
    if _wants_grad(x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, residual, ACTS[act], keep)
    K = x.shape[-1]
    y = _linear_call(_rows(x, K), _rows(weight, K), None if bias is None else bias.contiguous(), None if residual is None else _rows(residual, weight.shape[0]),
                     ACTS[act], False)[0]
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (weight.shape[0],))


def _linear_fits(x, weight, bias, residual, act, keep):
    """Everything in order?  (One pass of cheap comparisons: a serving call is over in microseconds; what is wrong is _explain_linear's to say.)"""
    if not (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor) and x.is_cuda and x.dim() and weight.dim() == 2):
        return False
    dt, dev, (N, K) = x.dtype, x.device, weight.shape
    if dt not in TYPES or weight.dtype != dt or weight.device != dev or x.shape[-1] != K or K < 1 or N < 1 or act not in ACTS or not (keep is None or keep in KEEPS):
        return False
    if bias is not None and not (isinstance(bias, torch.Tensor) and bias.dtype == dt and bias.shape == (N,) and bias.device == dev):
        return False
    return residual is None or (isinstance(residual, torch.Tensor) and residual.dtype == dt and residual.device == dev and residual.shape == x.shape[:-1] + (N,))


def _explain_linear(x, weight, bias, residual, act, keep):
    who = "linear_rows"
    _check_rows(who, "x", x)
    if act not in ACTS:
        _fail(who, "unknown activation %r (%s)" % (act, ", ".join(ACTS)))
    if keep is not None and keep not in KEEPS:
        _fail(who, "unknown format %r of the kept rows (%s)" % (keep, ", ".join(KEEPS)))
    _check_rows(who, "weight", weight, True)
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        _fail(who, "weight has shape %s, x %s" % (tuple(weight.shape), tuple(x.shape)))
    N = weight.shape[0]
    for name, t, shape in (("bias", bias, (N,)), ("residual", residual, tuple(x.shape[:-1]) + (N,))):
        if t is None:
            continue
        _check_rows(who, name, t, True)
        if tuple(t.shape) != shape:
            _fail(who, "%s has shape %s, not %s" % (name, tuple(t.shape), shape))
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            _fail(who, "%s is %s, x %s" % (name, t.dtype, x.dtype))
    _check_device(who, x, weight, bias, residual)
    _fail(who, "arguments that do not fit")


# ---------------------------------------------------------------------------------------------- the joint of a block
def _flat(t):
    if t is None:
        return None
    return (t.detach() if t.requires_grad else t).contiguous()


class _Joint:
    """One call's operands as the library takes them: 2-D rows, contiguous parameters, the descriptor over them."""
    __slots__ = ("x", "f", "gate", "params", "desc", "has_h")

    def __init__(self, x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift, meta):
        scale, post_kind, post_eps, pre_kind, pre_eps, gate_act = meta
        width = x.shape[-1]
        self.x = x = _rows(x, width)
        self.f = f = None if f is None else _rows(f, width)
        form = 0
        if gate is not None:
            form = 2 if gate.shape[-1] == width else 1
            gate = _rows(gate, gate.shape[-1])
        self.gate = gate
        self.params = p = (_flat(scale_cols), _flat(post_gain), _flat(post_shift), _flat(pre_gain), _flat(pre_shift))
        self.has_h = pre_kind is not None
        norm = lambda kind, eps, gain, shift: hip.BlockNorm(kind, 0 if gain is None and shift is None else TYPES[(shift if gain is None else gain).dtype], eps, 0,
                                                            _p(gain), _p(shift))
        self.desc = hip.JoinDesc(x.shape[0], width, TYPES[x.dtype], x.data_ptr(), _ld(x), _p(f), 0 if f is None else _ld(f), _p(gate), 0 if gate is None else _ld(gate),
                                 form, gate_act, _p(p[0]), 0 if p[0] is None else TYPES[p[0].dtype], scale, norm(post_kind, post_eps, p[1], p[2]),
                                 norm(pre_kind or 0, pre_eps, p[3], p[4]))

    def run(self, want_stats):
        x = self.x
        shape, dt, dev = x.shape, x.dtype, x.device
        y = None if self.f is None else torch.empty(shape, device=dev, dtype=dt)
        h = torch.empty(shape, device=dev, dtype=dt) if self.has_h else None
        stats = torch.empty((shape[0], 6), device=dev, dtype=torch.float32) if want_stats else None
        _launch("papr_join_fwd", dev, hip.lib().papr_join_fwd, self.desc, _p(y), _p(h), _p(stats))
        return y, h, stats


class _JoinFn(torch.autograd.Function):
    """(y, h) of join_rows, h alone without f (norm_rows), y alone without a next norm."""

    @staticmethod
    def forward(ctx, x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift, meta):
        j = _Joint(x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift, meta)
        y, h, stats = j.run(True)
        ctx.save_for_backward(j.x, j.f, j.gate, stats, *j.params)
        ctx.desc, ctx.has_h, ctx.shapes = j.desc, j.has_h, (x.shape, None if gate is None else gate.shape)      # (the descriptor points at the saved tensors)
        ctx.set_materialize_grads(False)
        if x.dim() != 2:
            y, h = (None if t is None else t.reshape(x.shape) for t in (y, h))
        return h if y is None else y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, *d_out):
        saved = ctx.saved_tensors                      # (refuses operands that were written to in between)
        xr, fr, gr, stats = saved[:4]
        params = saved[4:]
        need = ctx.needs_input_grad
        rows, width = xr.shape
        dev, dt = xr.device, xr.dtype
        d_y = d_out[0] if fr is not None else None
        d_h = d_out[-1] if ctx.has_h else None
        if d_y is None and d_h is None:
            return (None,) * 9
        if d_y is not None:
            d_y = d_y.reshape(rows, width).contiguous()
        if d_h is not None:
            d_h = d_h.reshape(rows, width).contiguous()
        d_x = torch.empty((rows, width), device=dev, dtype=dt) if need[0] else None
        d_f = torch.empty((rows, width), device=dev, dtype=dt) if need[1] else None
        d_g = torch.empty((rows, gr.shape[1]), device=dev, dtype=dt) if need[2] else None
        # scale, post gain, post shift, pre gain, pre shift (without d_h the last two are zero)
        d_p = [torch.empty((width,), device=dev, dtype=p.dtype) if need[3 + i] and p is not None else None for i, p in enumerate(params)]
        s, pg, ps, qg, qs = [_p(t) for t in d_p]
        lib = hip.lib()
        ws = torch.empty(lib.papr_join_bwd_workspace_bytes(rows, width) + 16, device=dev, dtype=torch.uint8) if any(need[3:8]) else None
        _launch("papr_join_bwd", dev, lib.papr_join_bwd, ctx.desc, stats.data_ptr(), _p(d_y), _p(d_h), _p(d_x), _p(d_f), _p(d_g), hip.JoinGrads(qg, qs, pg, ps, s), _p(ws))
        shape, g_shape = ctx.shapes
        if len(shape) != 2:
            d_x, d_f = (None if t is None else t.reshape(shape) for t in (d_x, d_f))
            d_g = None if d_g is None else d_g.reshape(g_shape)
        return (d_x, d_f, d_g, *d_p, None)


def _check_norm(who, name, norm, x):
    if not isinstance(norm, Norm):
        _fail(who, "%s is not a Norm" % name)
    if norm.kind not in NORMS:
        _fail(who, "unknown norm %r (%s)" % (norm.kind, ", ".join(NORMS)))
    width = x.shape[-1]
    if norm.kind == "layernorm" and width < 2:
        _fail(who, "layernorm's unbiased deviation needs two columns")
    for part, t in (("gain", norm.gain), ("shift", norm.shift)):
        if t is None:
            continue
        _check_rows(who, "%s.%s" % (name, part), t, True)
        if tuple(t.shape) != (width,):
            _fail(who, "%s.%s has shape %s, not (%d,)" % (name, part, tuple(t.shape), width))
    if norm.gain is not None and norm.shift is not None and norm.gain.dtype != norm.shift.dtype:
        _fail(who, "%s: gain is %s, shift %s" % (name, norm.gain.dtype, norm.shift.dtype))


def _check_width(who, x):
    if x.shape[-1] > hip.JOIN_MAX_WIDTH:
        _fail(who, "rows of %d columns (at most %d)" % (x.shape[-1], hip.JOIN_MAX_WIDTH))


def _join(x, f, gate, scale, scale_cols, post, pre, gate_act):
    tensors = (x, f, gate, scale_cols, post.gain, post.shift) + ((pre.gain, pre.shift) if pre else (None, None))
    meta = (scale, NORMS[post.kind], float(post.eps), NORMS[pre.kind] if pre else None, float(pre.eps) if pre else 0.0, gate_act)
    if _wants_grad(*tensors):
        return _JoinFn.apply(*tensors, meta)
    y, h, _ = _Joint(*tensors, meta).run(False)
    if x.dim() != 2:
        y, h = (None if t is None else t.reshape(x.shape) for t in (y, h))
    return h if y is None else y if h is None else (y, h)


def norm_rows(x, norm):
    """The norm in front of a block: N(x) over the last dimension, norm = Norm(kind, gain, shift, eps); statistics in float32."""
    _check_rows("norm_rows", "x", x)
    _check_width("norm_rows", x)
    _check_norm("norm_rows", "norm", norm, x)
    _check_device("norm_rows", x, norm.gain, norm.shift)
    return _join(x, None, None, 1.0, None, Norm("none"), norm, 0)


def join_rows(x, f, gate=None, scale=1.0, post=None, pre=None, gate_act="sigmoid"):
    """The end of a residual block and the start of the next in one pass over the rows:

        y = x + scale * gate_act(gate) * N_post(f),    h = N_pre(y)

    x, f (..., width) of one type; gate (..., width) or one per row (..., 1), of that type, or None; scale a number or a (width,) tensor; post, pre: Norm or None
    (post: f as it is; pre: no h).  gate_act: none, sigmoid, silu.  Returns (y, h), or y alone without pre.  h is the norm of y before y's rounding.  Parameters
    (scale, gains, shifts) may be float32 beside 16-bit rows; their gradients are sums in float32, returned in their own type."""
    who = "join_rows"
    _check_rows(who, "x", x)
    _check_width(who, x)
    _check_rows(who, "f", f, True)
    if f.shape != x.shape or f.dtype != x.dtype:
        _fail(who, "f is %s %s, x %s %s" % (f.dtype, tuple(f.shape), x.dtype, tuple(x.shape)))
    if gate_act not in GATE_ACTS:
        _fail(who, "unknown gate activation %r (%s)" % (gate_act, ", ".join(GATE_ACTS)))
    width = x.shape[-1]
    if gate is not None:
        _check_rows(who, "gate", gate, True)
        if gate.dtype != x.dtype or (gate.shape != x.shape and tuple(gate.shape) != tuple(x.shape[:-1]) + (1,)):
            _fail(who, "gate is %s %s, x %s %s" % (gate.dtype, tuple(gate.shape), x.dtype, tuple(x.shape)))
    scale_cols = None
    if torch.is_tensor(scale):
        _check_rows(who, "scale", scale, True)
        if tuple(scale.shape) != (width,):
            _fail(who, "scale has shape %s, not (%d,)" % (tuple(scale.shape), width))
        scale, scale_cols = 1.0, scale
    for name, norm in (("post", post), ("pre", pre)):
        if norm is not None:
            _check_norm(who, name, norm, x)
    _check_device(who, x, f, gate, scale_cols, *(t for norm in (post, pre) if norm is not None for t in (norm.gain, norm.shift)))
    return _join(x, f, gate, float(scale), scale_cols, post if post is not None else Norm("none"), pre, GATE_ACTS[gate_act])
