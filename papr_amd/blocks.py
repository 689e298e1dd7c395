"""Row blocks: the parts of a residual feed-forward block over rows of float32, float16 or bfloat16, each with its backward pass.

    norm_rows    h = N(x)                                                  the norm in front of a block
    linear_rows  y = act(x W^T + b) + r                                    a Linear layer with its epilogue
    join_rows    y = x + s * a(g) * N_post(f),  h = N_pre(y)               the block's end and the next block's norm in one pass
    pack_rows    rows in 8 bits, PackedRows.rows() back                    what linear_rows(keep=...) holds for its backward pass

They are what `FeedForward.forward` of the reference does around its MLP (models/attn.py:111-117: innorm, mlp, outnorm, the residual branch), for rows that are not
the render path's own: `papr_amd.ops` runs the embedding MLPs as whole chains instead.  All work goes through libpapr_hip.so (include/papr_hip.h: papr_linear_*,
papr_join_*, papr_rows8_*) on the current stream of the rows' device; there is no CPU form.  The calls and their autograd nodes are native (csrc/blocks_glue.cpp).  Workspaces come from torch's allocator call by call, so calls on
several streams and in several captured graphs do not share any.  Second derivatives and forward-mode derivatives are not defined and refused,
and so are traces (torch.jit.trace, make_fx) and torch.func transforms: the calls are not torch operators.
"""
import collections
import ctypes as C
import math

import torch

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


_native = None


def _load():
    """The native host side over the loaded library (raises if either has not been built)."""
    global _native
    L = hip.lib()
    try:
        from . import _blocks as m
    except ImportError as e:
        raise RuntimeError("papr_amd: papr_amd/_blocks.so is missing or does not load (%s) -- run `python -c 'import __graft_entry__ as g; g.build()'`" % e)
    m.bind({name: C.cast(getattr(L, name), C.c_void_p).value for name in hip.EXPORTS if name.startswith(("papr_linear_", "papr_join_", "papr_rows8_", "papr_last_error"))}, hip)
    _native = m
    return m


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
        try:
            x = (_native or _load()).unpack(self.codes, self.exps, KEEPS.get(self.fmt, 0), TYPES.get(self.dtype, -1), self.shape)
        except TypeError:
            x = None
        if x is None:
            self._explain()
        return x

    def _explain(self):
        who, shape = "PackedRows.rows", tuple(self.shape)
        if self.fmt not in KEEPS:
            _fail(who, "unknown format %r (%s)" % (self.fmt, ", ".join(KEEPS)))
        if self.dtype not in TYPES:
            _fail(who, "type %s (float32, float16, bfloat16)" % (self.dtype,))
        if not shape or shape[-1] < 1:
            _fail(who, "shape %s: rows of at least one column" % (shape,))
        if shape[-1] > hip.ROWS8_MAX_WIDTH:
            _fail(who, "rows of %d columns (at most %d)" % (shape[-1], hip.ROWS8_MAX_WIDTH))
        rows, blocks = math.prod(shape[:-1]), (shape[-1] + BLOCK - 1) // BLOCK
        for name, t, want in (("codes", self.codes, (rows, blocks * BLOCK)), ("exps", self.exps, (rows, blocks))):
            if not torch.is_tensor(t) or t.dtype != torch.uint8 or tuple(t.shape) != want:
                _fail(who, "%s of rows %s are uint8 %s" % (name, shape, want))
        _check_device(who, self.codes, self.exps)
        _fail(who, "arguments that do not fit")


def pack_rows(x, fmt="e4m3"):
    """x (..., width) -> PackedRows: 8 bits a value and one power-of-two scale for every 32 columns of a row (33/32 bytes a value).  "e4m3" keeps four significant
    bits of every value down to 2^-14 of its block's largest, "int8" seven bits below the block's largest.  NaN and infinities come back as NaN.  No gradient: this
    is how an activation is kept, not a part of the model."""
    packed = (_native or _load()).pack(x, KEEPS.get(fmt, 0)) if isinstance(x, torch.Tensor) and fmt in KEEPS else None
    if packed is None:
        _check_rows("pack_rows", "x", x)
        if fmt not in KEEPS:
            _fail("pack_rows", "unknown format %r (%s)" % (fmt, ", ".join(KEEPS)))
        if x.shape[-1] > hip.ROWS8_MAX_WIDTH:
            _fail("pack_rows", "rows of %d columns (at most %d)" % (x.shape[-1], hip.ROWS8_MAX_WIDTH))
        _check_device("pack_rows", x)
    return PackedRows(packed[0], packed[1], fmt, x.shape, x.dtype)


# ---------------------------------------------------------------------------------------------- linear layers
def linear_rows(x, weight, bias=None, residual=None, act="none", keep=None):
    """act(x @ weight.T + bias) + residual over the last dimension: x (..., K), weight (N, K), bias (N,), residual (..., N), all of one type (float32, float16,
    bfloat16; sums in float32, the result rounded once).  act: none, relu, leakyrelu (slope 0.2), gelu (erf form), silu.

    keep = "e4m3" / "int8": in training the rows x are held for the weight's gradient as pack_rows keeps them -- a quarter (float32) or half of the memory -- and that
    gradient is d_z^T times the values they stand for; y and every other gradient are those of keep=None.  An activation's argument is held in 16 bits for the
    backward pass of 16-bit rows (silu and gelu: float16); nothing else there is rounded below 32 bits or two values of the rows' type before the gradients themselves are."""
    try:
        y = (_native or _load()).linear(x, weight, bias, residual, ACTS.get(act, -1), 0 if keep is None else KEEPS.get(keep, -1))
    except TypeError:
        y = None
    if y is None:
        _explain_linear(x, weight, bias, residual, act, keep)
    return y


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
    if max(weight.shape) > 1 << 20:
        _fail(who, "weight has shape %s (at most %d a side)" % (tuple(weight.shape), 1 << 20))
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
    """None: arguments that do not fit"""
    try:
        return (_native or _load()).join(x, f, gate, scale, scale_cols, NORMS.get(post.kind, -1), post.eps, post.gain, post.shift,
                                         -1 if pre is None else NORMS.get(pre.kind, -2), 0.0 if pre is None else pre.eps,
                                         None if pre is None else pre.gain, None if pre is None else pre.shift, GATE_ACTS.get(gate_act, -1))
    except (TypeError, AttributeError):
        return None


_PLAIN = Norm("none")


def norm_rows(x, norm):
    """The norm in front of a block: N(x) over the last dimension, norm = Norm(kind, gain, shift, eps); statistics in float32."""
    h = _join(x, None, None, 1.0, None, _PLAIN, norm, "none") if norm is not None else None
    if h is None:
        _check_rows("norm_rows", "x", x)
        _check_width("norm_rows", x)
        _check_norm("norm_rows", "norm", norm, x)
        _check_device("norm_rows", x, norm.gain, norm.shift)
        _fail("norm_rows", "arguments that do not fit")
    return h


def join_rows(x, f, gate=None, scale=1.0, post=None, pre=None, gate_act="sigmoid"):
    """The end of a residual block and the start of the next in one pass over the rows:

        y = x + scale * gate_act(gate) * N_post(f),    h = N_pre(y)

    x, f (..., width) of one type; gate (..., width) or one per row (..., 1), of that type, or None; scale a number or a (width,) tensor; post, pre: Norm or None
    (post: f as it is; pre: no h).  gate_act: none, sigmoid, silu.  Returns (y, h), or y alone without pre.  h is the norm of y before y's rounding.  Parameters
    (scale, gains, shifts) may be float32 beside 16-bit rows; their gradients are sums in float32, returned in their own type."""
    cols = isinstance(scale, torch.Tensor)
    out = _join(x, f, gate, 1.0 if cols else scale, scale if cols else None, _PLAIN if post is None else post, pre, gate_act) if f is not None else None
    if out is None:
        _explain_join(x, f, gate, scale, post, pre, gate_act)
    return out


def _explain_join(x, f, gate, scale, post, pre, gate_act):
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
    if torch.is_tensor(scale):
        _check_rows(who, "scale", scale, True)
        if tuple(scale.shape) != (width,):
            _fail(who, "scale has shape %s, not (%d,)" % (tuple(scale.shape), width))
    for name, norm in (("post", post), ("pre", pre)):
        if norm is not None:
            _check_norm(who, name, norm, x)
    _check_device(who, x, f, gate, scale if torch.is_tensor(scale) else None, *(t for norm in (post, pre) if norm is not None for t in (norm.gain, norm.shift)))
    _fail(who, "arguments that do not fit")
