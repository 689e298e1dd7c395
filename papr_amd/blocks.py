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
    t = t.detach()
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if t.numel() and ((width > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < width)):
        t = t.contiguous()
    return t


def _ld(t):
    return max(t.stride(0), t.shape[1])


def _p(t):
    return None if t is None else t.data_ptr()


class _on:
    """The rows' device as the current one, and its stream (the library launches on the current device)."""

    def __init__(self, dev):
        self.guard = torch.cuda.device(dev) if torch.cuda.current_device() != dev.index else None
        self.index = dev.index

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in ts)


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
        with _on(out.device) as s:
            hip.check(hip.lib().papr_rows8_unpack(TYPES[self.dtype], KEEPS[self.fmt], _p(self.codes), _p(self.exps), self.codes.shape[0], self.shape[-1], _p(out), s),
                      "papr_rows8_unpack")
        return out


def pack_rows(x, fmt="e4m3"):
    """x (..., width) -> PackedRows: 8 bits a value and one power-of-two scale for every 32 columns of a row (33/32 bytes a value).  "e4m3" keeps four significant
    bits of every value down to 2^-14 of its block's largest, "int8" seven bits below the block's largest.  NaN and infinities come back as NaN.  No gradient: this
    is how an activation is kept, not a part of the model."""
    _check_rows("pack_rows", "x", x)
    if fmt not in KEEPS:
        _fail("pack_rows", "unknown format %r (%s)" % (fmt, ", ".join(KEEPS)))
    _check_device("pack_rows", x)
    width = x.shape[-1]
    rows = _rows(x, width)
    n, blocks = rows.shape[0], (width + BLOCK - 1) // BLOCK
    codes = torch.empty((n, blocks * BLOCK), device=x.device, dtype=torch.uint8)
    exps = torch.empty((n, blocks), device=x.device, dtype=torch.uint8)
    with _on(x.device) as s:
        hip.check(hip.lib().papr_rows8_pack(TYPES[x.dtype], KEEPS[fmt], _p(rows), _ld(rows), n, width, _p(codes), _p(exps), s), "papr_rows8_pack")
    return PackedRows(codes, exps, fmt, tuple(x.shape), x.dtype)


# ---------------------------------------------------------------------------------------------- linear layers
def _linear_call(x, weight, bias, residual, act, want_z):
    """(y, z or None) of 2-D rows"""
    M, K = x.shape
    N = weight.shape[0]
    y = torch.empty((M, N), device=x.device, dtype=x.dtype)
    z = torch.empty_like(y) if want_z else None
    d = hip.LinearDesc(TYPES[x.dtype], act, 0, 0, M, N, K)
    with _on(x.device) as s:
        hip.check(hip.lib().papr_linear_fwd(d, _p(x), _ld(x), _p(weight), _ld(weight), _p(bias), _p(residual), 0 if residual is None else _ld(residual), _p(y), _p(z), s),
                  "papr_linear_fwd")
    return y, z


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, keep):
        K, N = weight.shape[1], weight.shape[0]
        need = ctx.needs_input_grad
        rows, w2 = _rows(x, K), _rows(weight, K)
        y, z = _linear_call(rows, w2, None if bias is None else bias.detach().contiguous(), None if residual is None else _rows(residual, N), act,
                            act != 0 and any(need[:3]))
        packed = pack_rows(rows, keep) if keep is not None and need[1] else None
        held = None if not need[1] else rows if packed is None else packed.codes
        ctx.save_for_backward(held, None if packed is None else packed.exps, w2 if need[0] else None, z)
        ctx.act, ctx.keep, ctx.dims, ctx.shapes = act, keep if packed is not None else None, (rows.shape[0], N, K), (x.shape, weight.shape)
        return y.reshape(x.shape[:-1] + (N,))

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        held, exps, w2, z = ctx.saved_tensors
        M, N, K = ctx.dims
        need = ctx.needs_input_grad
        d_res = d_y if need[3] else None
        if not any(need[:3]):
            return None, None, None, d_res, None, None
        dev, dt = d_y.device, d_y.dtype
        if M == 0:
            return (d_y.new_zeros(ctx.shapes[0]) if need[0] else None, d_y.new_zeros(ctx.shapes[1]) if need[1] else None, d_y.new_zeros(N) if need[2] else None,
                    d_res, None, None)
        g = _rows(d_y, N)
        new = lambda *shape: torch.empty(shape, device=dev, dtype=dt)
        d_x, d_w, d_b = new(M, K) if need[0] else None, new(N, K) if need[1] else None, new(N) if need[2] else None
        d = hip.LinearDesc(TYPES[dt], ctx.act, KEEPS.get(ctx.keep, 0), 0, M, N, K)
        lib = hip.lib()
        with _on(dev) as s:
            ws = torch.empty(max(int(lib.papr_linear_bwd_workspace_bytes(d)), 16), device=dev, dtype=torch.uint8)
            hip.check(lib.papr_linear_bwd(d, _p(g), _ld(g), _p(z), _p(held), 0 if held is None else _ld(held), _p(exps), _p(w2), 0 if w2 is None else _ld(w2),
                                          _p(d_x), _p(d_w), _p(d_b), _p(ws), s), "papr_linear_bwd")
        return None if d_x is None else d_x.reshape(ctx.shapes[0]), d_w, d_b, d_res, None, None


def linear_rows(x, weight, bias=None, residual=None, act="none", keep=None):
    """act(x @ weight.T + bias) + residual over the last dimension: x (..., K), weight (N, K), bias (N,), residual (..., N), all of one type (float32, float16,
    bfloat16; sums in float32, the result rounded once).  act: none, relu, leakyrelu (slope 0.2), gelu (erf form), silu.

    keep = "e4m3" / "int8": in training the rows x are held for the weight's gradient as pack_rows keeps them -- a quarter (float32) or half of the memory -- and that
    gradient is d_z^T times the values they stand for; y and every other gradient are those of keep=None.  An activation's argument is held in the rows' type.  float32
    rows with infinities give NaN."""
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
    if _wants_grad(x, weight, bias, residual):
        return _LinearFn.apply(x, weight, bias, residual, ACTS[act], keep)
    K = x.shape[-1]
    y, _ = _linear_call(_rows(x, K), _rows(weight, K), None if bias is None else bias.detach().contiguous(), None if residual is None else _rows(residual, N), ACTS[act], False)
    return y if x.dim() == 2 else y.reshape(x.shape[:-1] + (N,))


# ---------------------------------------------------------------------------------------------- the joint of a block
def _join_desc(x, f, gate, scale, scale_cols, norms, gate_act):
    """The descriptor of a call over 2-D rows; norms = ((kind, gain, shift, eps) of the block's output, of the next block)."""
    rows, width = x.shape
    form = 0 if gate is None else 2 if gate.shape[1] == width else 1
    ns = [hip.BlockNorm(kind, TYPES[gain.dtype] if gain is not None else TYPES[shift.dtype] if shift is not None else 0, eps, 0, _p(gain), _p(shift))
          for kind, gain, shift, eps in norms]
    return hip.JoinDesc(rows, width, TYPES[x.dtype], _p(x), _ld(x), _p(f), 0 if f is None else _ld(f), _p(gate), 0 if gate is None else _ld(gate), form, gate_act,
                        _p(scale_cols), 0 if scale_cols is None else TYPES[scale_cols.dtype], scale, ns[0], ns[1])


def _join_call(d, like, want_y, want_h, want_stats):
    rows, width = like.shape
    y = torch.empty((rows, width), device=like.device, dtype=like.dtype) if want_y else None
    h = torch.empty((rows, width), device=like.device, dtype=like.dtype) if want_h else None
    stats = torch.empty((rows, 6), device=like.device, dtype=torch.float32) if want_stats else None
    with _on(like.device) as s:
        hip.check(hip.lib().papr_join_fwd(d, _p(y), _p(h), _p(stats), s), "papr_join_fwd")
    return y, h, stats


class _JoinFn(torch.autograd.Function):
    """(y, h) of join_rows, h alone without f (norm_rows), y alone without a next norm."""

    @staticmethod
    def forward(ctx, x, f, gate, scale_cols, post_gain, post_shift, pre_gain, pre_shift, meta):
        scale, post, pre, gate_act = meta
        width = x.shape[-1]
        two = lambda t, w=width: None if t is None else _rows(t, w)
        flat = lambda t: None if t is None else t.detach().contiguous()
        xr, fr, gr = two(x), two(f), two(gate, None if gate is None else gate.shape[-1])
        params = [flat(t) for t in (scale_cols, post_gain, post_shift, pre_gain, pre_shift)]
        d = _join_desc(xr, fr, gr, scale, params[0], ((post[0], params[1], params[2], post[1]), (pre[0], params[3], params[4], pre[1]) if pre else (0, None, None, 0.0)), gate_act)
        y, h, stats = _join_call(d, xr, f is not None, pre is not None, True)
        ctx.save_for_backward(xr, fr, gr, stats, *params)
        ctx.meta, ctx.shapes = meta, (x.shape, None if gate is None else gate.shape)
        ctx.set_materialize_grads(False)
        out = [t.reshape(x.shape) for t in (y, h) if t is not None]
        return tuple(out) if len(out) > 1 else out[0]

    @staticmethod
    @once_differentiable
    def backward(ctx, *d_out):
        xr, fr, gr, stats = ctx.saved_tensors[:4]
        params = ctx.saved_tensors[4:]
        scale, post, pre, gate_act = ctx.meta
        need = ctx.needs_input_grad
        rows, width = xr.shape
        dev, dt = xr.device, xr.dtype
        d_out = list(d_out)
        d_y = d_out.pop(0) if fr is not None else None
        d_h = d_out.pop(0) if pre else None
        none = (None,) * 9
        if d_y is None and d_h is None:
            return none
        full = lambda t: None if t is None else t.reshape(rows, width).contiguous()
        d_y, d_h = full(d_y), full(d_h)
        new = lambda *shape: torch.empty(shape, device=dev, dtype=dt)
        d_x = new(rows, width) if need[0] else None
        d_f = new(rows, width) if need[1] else None
        d_g = new(rows, gr.shape[1]) if need[2] else None
        # scale, post gain, post shift, pre gain, pre shift (the last two have none without d_h)
        d_p = [torch.empty_like(p) if need[3 + i] and p is not None else None for i, p in enumerate(params)]
        d = _join_desc(xr, fr, gr, scale, params[0], ((post[0], params[1], params[2], post[1]), (pre[0], params[3], params[4], pre[1]) if pre else (0, None, None, 0.0)), gate_act)
        grads = hip.JoinGrads(_p(d_p[3]), _p(d_p[4]), _p(d_p[1]), _p(d_p[2]), _p(d_p[0]))
        lib = hip.lib()
        with _on(dev) as s:
            ws = None
            if any(t is not None for t in d_p):
                ws = torch.empty(max(int(lib.papr_join_bwd_workspace_bytes(rows, width)), 16), device=dev, dtype=torch.uint8)
            hip.check(lib.papr_join_bwd(d, _p(stats), _p(d_y), _p(d_h), _p(d_x), _p(d_f), _p(d_g), grads, _p(ws), s), "papr_join_bwd")
        back = lambda t, shape: None if t is None else t.reshape(shape)
        return (back(d_x, ctx.shapes[0]), back(d_f, ctx.shapes[0]), back(d_g, ctx.shapes[1])) + tuple(d_p) + (None,)


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
    meta = (scale, (NORMS[post.kind], float(post.eps)), (NORMS[pre.kind], float(pre.eps)) if pre else None, gate_act)
    if _wants_grad(*tensors):
        return _JoinFn.apply(*tensors, meta)
    width = x.shape[-1]
    two = lambda t, w=width: None if t is None else _rows(t, w)
    flat = lambda t: None if t is None else t.detach().contiguous()
    xr, fr, gr, sc = two(x), two(f), two(gate, None if gate is None else gate.shape[-1]), flat(scale_cols)
    held = [flat(t) for t in tensors[4:]]
    d = _join_desc(xr, fr, gr, scale, sc, ((meta[1][0], held[0], held[1], meta[1][1]), (meta[2][0], held[2], held[3], meta[2][1]) if pre else (0, None, None, 0.0)), gate_act)
    out = [t if x.dim() == 2 else t.reshape(x.shape) for t in _join_call(d, xr, f is not None, pre is not None, False)[:2] if t is not None]
    return tuple(out) if len(out) > 1 else out[0]


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
