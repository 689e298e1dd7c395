"""Timed cases of the row-block operators: linear layers with their epilogue, the norms at the joint of a residual block, and rows kept in 8 bits.

    linear  y = act(x W^T + b) + r, forward or forward and backward           (papr_amd.blocks.linear_rows)
    join    y = x + s * act(g) * N_post(f),  h = N_pre(y), forward or both     (papr_amd.blocks.join_rows)
    pack    rows to 8 bits with a power-of-two scale per 32 columns, and back  (papr_amd.blocks.pack_rows, PackedRows.rows)
    kept    a linear layer in training whose input rows are kept in 8 bits     (papr_amd.blocks.linear_rows(keep=...))

`own` = False computes every operator in elementary torch operations in 32 bits; True calls the package.
"""
import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
EPS = 1e-6
BLOCK = 32                                              # columns that share a scale in packed rows


def listed():
    return [
        # one token through a feed-forward layer while serving: latency, bounded by one read of the weight
        dict(name="linear_token_bf16", op="linear", train=False, dtype="bfloat16", rows=1, d_in=1024, d_out=4096, act="silu", bias=True, residual=True),
        # one 100 x 100 chunk of an image in evaluation through the first key layer, whose input is 117 wide (odd row starts)
        dict(name="linear_chunk_fp16", op="linear", train=False, dtype="float16", rows=10000, d_in=117, d_out=256, act="gelu", bias=True, residual=False),
        # a training step of a feed-forward layer over some thousand tokens, every gradient
        dict(name="linear_step_bf16", op="linear", train=True, dtype="bfloat16", rows=8192, d_in=1024, d_out=4096, act="gelu", bias=True, residual=True),
        # the 256 x 256 layer of an embedding MLP over all pair rows of a 25,600-ray step, in the parity type
        dict(name="linear_pairs_fp32", op="linear", train=True, dtype="float32", rows=512000, d_in=256, d_out=256, act="silu", bias=True, residual=True),
        # the joint behind a block for one token while serving
        dict(name="join_token_bf16", op="join", train=False, dtype="bfloat16", rows=1, width=4096, norm="rmsnorm", gate="full", scale="number", params="bfloat16"),
        # a step's rays at the key rows' width: odd rows, the framework's own norm, every gradient
        dict(name="join_rays_fp32", op="join", train=True, dtype="float32", rows=25600, width=117, norm="layernorm", gate="full", scale="columns", params="float32"),
        # prompt tokens through the joint while serving
        dict(name="join_tokens_bf16", op="join", train=False, dtype="bfloat16", rows=16384, width=2048, norm="rmsnorm", gate="full", scale="number", params="bfloat16"),
        # all pair rows of a step at d_model, one gate per row, norms held in 32 bits, every gradient
        dict(name="join_pairs_fp16", op="join", train=True, dtype="float16", rows=512000, width=256, norm="layernorm", gate="row", scale="columns", params="float32"),
        # a few odd rows: the smallest checkpoint
        dict(name="pack_small_fp16", op="pack", dtype="float16", rows=37, width=142, fmt="int8"),
        # the activations of one layer over all pair rows of a step
        dict(name="pack_pairs_bf16", op="pack", dtype="bfloat16", rows=512000, width=256, fmt="e4m3"),
        # a wide layer over a large batch whose input rows would not fit beside the rest
        dict(name="kept_step_bf16", op="kept", train=True, dtype="bfloat16", rows=65536, d_in=1024, d_out=1024, act="silu", bias=True, residual=True, fmt="e4m3"),
        # a step's rays through the first value layer (142 columns) in the parity type
        dict(name="kept_rays_fp32", op="kept", train=True, dtype="float32", rows=25600, d_in=142, d_out=256, act="gelu", bias=True, residual=False, fmt="int8"),
    ]


def _log_int(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:                              # half of the sizes as they fall, half at whole vectors
        n = max(lo, n // 8 * 8)
    return min(max(n, lo), hi)


def draw(rng):
    op = rng.choice(["linear", "linear", "join", "join", "pack", "kept"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if op in ("linear", "kept"):
        d_in, d_out = _log_int(rng, 32, 4096), _log_int(rng, 32, 4096)
        train = op == "kept" or rng.random() < 0.5
        # no dearer than the largest listed pass (three products of 65536 x 1024 x 1024; a third of that in float32)
        cap = (65536 * 1024 * 1024 // (1 if train else 2)) // (3 if dtype == "float32" else 1)
        rows = _log_int(rng, 1, max(1, min(512000, cap // (d_in * d_out), 65536 * 2048 // (d_in + d_out))))
        # (the derivative of the piecewise linear activations jumps at zero: in training the smooth ones)
        act = rng.choice(["none", "gelu", "silu"] + ([] if train else ["relu", "leakyrelu"]))
        case = dict(op=op, train=train, dtype=dtype, rows=rows, d_in=d_in, d_out=d_out, act=act, bias=rng.random() < 0.7, residual=rng.random() < 0.5)
        if op == "kept":
            case["fmt"] = rng.choice(["e4m3", "int8"])
        return case
    width = _log_int(rng, 32, 8192)
    rows = _log_int(rng, 1, min(512000, 512000 * 256 // width))
    if op == "pack":
        return dict(op=op, dtype=dtype, rows=rows, width=width, fmt=rng.choice(["e4m3", "int8"]))
    return dict(op=op, train=rng.random() < 0.5, dtype=dtype, rows=rows if dtype != "float32" else max(1, rows // 2), width=width,
                norm=rng.choice(["rmsnorm", "layernorm"]), gate=rng.choice(["none", "row", "full"]), scale=rng.choice(["number", "columns"]),
                params=rng.choice(["float32", dtype]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = dict(case)
    rows, grad = case["rows"], case.get("train", False)
    if case["op"] in ("linear", "kept"):
        k, n = case["d_in"], case["d_out"]
        s["x"] = normal(rows, k)
        s["w"] = normal(n, k, std=k ** -0.5)
        s["b"] = normal(n, std=0.1) if case["bias"] else None
        s["r"] = normal(rows, n) if case["residual"] else None
        s["d_y"] = normal(rows, n, std=0.1) if grad else None
        leaves = ("x", "w", "b", "r")
    elif case["op"] == "join":
        d, pt = case["width"], DTYPES[case["params"]]
        s["x"], s["f"] = normal(rows, d), normal(rows, d, std=0.5)
        s["g"] = normal(rows, 1 if case["gate"] == "row" else d) if case["gate"] != "none" else None
        s["s"] = normal(d, std=0.05, mean=0.3, dtype=pt) if case["scale"] == "columns" else 0.3
        for name in ("post", "pre"):
            s[name + "_a"] = normal(d, std=0.1, mean=1.0, dtype=pt)
            s[name + "_b"] = normal(d, std=0.1, dtype=pt) if case["norm"] == "layernorm" else None
        s["d_y"], s["d_h"] = (normal(rows, d, std=0.1), normal(rows, d, std=0.1)) if grad else (None, None)
        leaves = ("x", "f", "g", "s", "post_a", "post_b", "pre_a", "pre_b")
    else:
        # activations: most of them small, some columns far out
        x = torch.randn((rows, case["width"]), generator=g, device="cuda") * torch.exp(1.5 * torch.randn((case["width"],), generator=g, device="cuda"))
        s["x"], leaves = x.to(dt), ()
    s["leaves"] = [n for n in leaves if torch.is_tensor(s[n])] if grad else []
    for n in s["leaves"]:
        s[n].requires_grad_(True)
    return s


# ---------------------------------------------------------------------------------------------- the package's calls
def _own_linear(s):
    from papr_amd import blocks
    keep = s.get("fmt")
    if not s["train"]:
        with torch.no_grad():
            return blocks.linear_rows(s["x"], s["w"], s["b"], s["r"], act=s["act"], keep=keep)
    y = blocks.linear_rows(s["x"], s["w"], s["b"], s["r"], act=s["act"], keep=keep)
    return [y.detach()] + list(torch.autograd.grad(y, [s[n] for n in s["leaves"]], s["d_y"]))


def _own_join(s):
    from papr_amd import blocks
    post, pre = blocks.Norm(s["norm"], s["post_a"], s["post_b"], EPS), blocks.Norm(s["norm"], s["pre_a"], s["pre_b"], EPS)
    kw = dict(gate=s["g"], scale=s["s"], post=post, pre=pre, gate_act="sigmoid")
    if not s["train"]:
        with torch.no_grad():
            return list(blocks.join_rows(s["x"], s["f"], **kw))
    y, h = blocks.join_rows(s["x"], s["f"], **kw)
    return [y.detach(), h.detach()] + list(torch.autograd.grad([y, h], [s[n] for n in s["leaves"]], [s["d_y"], s["d_h"]]))


def _own_pack(s):
    from papr_amd import blocks
    return blocks.pack_rows(s["x"], s["fmt"]).rows()


# ---------------------------------------------------------------------------------------------- the plain forms
def _act(z, act):
    """(value, derivative)"""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, 0.0), (z > 0).to(z.dtype)
    if act == "leakyrelu":
        return torch.where(z > 0, z, 0.2 * z), torch.where(z > 0, 1.0, 0.2)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return z * p, p * (1 + z * (1 - p))
    p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
    return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


def _limit(dtype, fmt):
    """The largest magnitude the format keeps: one that the rows' own type still holds."""
    return (1.875 if fmt == "e4m3" else 1.984375) * 2.0 ** (15 if dtype == torch.float16 else 127)


def _pack_plain(x, fmt):
    """The values the packed rows stand for, in float32."""
    dtype, (rows, width) = x.dtype, x.shape
    v = x.float()
    bad = ~torch.isfinite(v)
    v = torch.clamp(torch.where(bad, 0.0, v), -_limit(dtype, fmt), _limit(dtype, fmt))
    pad = -width % BLOCK
    v = torch.cat([v, v.new_zeros(rows, pad)], dim=1).reshape(rows, -1, BLOCK)
    bits = v.abs().amax(dim=2, keepdim=True).view(torch.int32)
    expo, frac = (bits >> 23) - 127, bits & 0x7FFFFF
    # the smallest 2^e with max <= top 2^e: top = 1.75 2^8 (e4m3), 1.984375 2^6 (int8)
    top_e, top_f = (8, 0x600000) if fmt == "e4m3" else (6, 0x7E0000)
    e = torch.clamp(expo - top_e + (frac > top_f).to(torch.int32), min=-120)
    scale, inv = ((e + 127) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)
    q = v * inv
    if fmt == "e4m3":
        qe = torch.clamp((q.abs().view(torch.int32) >> 23) - 127, min=-6)
        step, per_step = ((qe - 3 + 127) << 23).view(torch.float32), ((127 + 3 - qe) << 23).view(torch.float32)
        q = torch.round(q * per_step) * step
    else:
        q = torch.round(q)
    v = (q * scale).reshape(rows, width + pad)[:, :width]
    return torch.where(bad, math.nan, v)


def _plain_linear(s):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    if not s["train"]:
        return y.to(dt)
    d_z = s["d_y"].float() * slope
    xs = _pack_plain(s["x"], s["fmt"]) if "fmt" in s else x
    out = [y, d_z @ w, d_z.t() @ xs]
    if s["b"] is not None:
        out.append(d_z.sum(0))
    if s["r"] is not None:
        out.append(s["d_y"])
    return [t.to(dt) for t in out]


def _norm_plain(v, kind, a, b):
    """(value, standardised rows, their divisor)"""
    if kind == "rmsnorm":
        div = torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
        n = v / div
        return n * a, n, div
    c = v - v.mean(1, keepdim=True)
    std = torch.sqrt((c * c).sum(1, keepdim=True) / (v.shape[1] - 1))
    n = c / (std + EPS)
    return n * a + b, n, (std, std + EPS)


def _norm_plain_bwd(d_out, n, div, kind, a):
    """d_v of the norm from the gradient of its output."""
    d_n = d_out * a
    if kind == "rmsnorm":
        return (d_n - n * (d_n * n).mean(1, keepdim=True)) / div
    std, div = div
    # n = c / (std + eps): d std / d v = c / ((D - 1) std) = n (std + eps) / ((D - 1) std)
    t = d_n - n * ((d_n * n).sum(1, keepdim=True) * div / ((n.shape[1] - 1) * std))
    return (t - t.mean(1, keepdim=True)) / div


def _plain_join(s):
    dt, kind = s["x"].dtype, s["norm"]
    val = lambda t: t.float() if torch.is_tensor(t) else t
    x, f, g, sc = val(s["x"]), val(s["f"]), val(s["g"]), val(s["s"])
    pa, pb, qa, qb = val(s["post_a"]), val(s["post_b"]), val(s["pre_a"]), val(s["pre_b"])
    p, pn, pdiv = _norm_plain(f, kind, pa, pb)
    gate = 1 / (1 + torch.exp(-g)) if g is not None else 1.0
    y = x + sc * gate * p
    h, yn, ydiv = _norm_plain(y, kind, qa, qb)
    if not s["train"]:
        return [y.to(dt), h.to(dt)]
    d_y, d_h = s["d_y"].float(), s["d_h"].float()
    d_y = d_y + _norm_plain_bwd(d_h, yn, ydiv, kind, qa)
    d_p = d_y * sc * gate
    grads = dict(x=d_y, f=_norm_plain_bwd(d_p, pn, pdiv, kind, pa), post_a=(d_p * pn).sum(0), post_b=d_p.sum(0), pre_a=(d_h * yn).sum(0), pre_b=d_h.sum(0))
    if g is not None:
        d_g = d_y * sc * p * gate * (1 - gate)
        grads["g"] = d_g.sum(1, keepdim=True) if g.shape[1] == 1 else d_g
    if torch.is_tensor(sc):
        grads["s"] = (d_y * gate * p).sum(0)
    return [y.to(dt), h.to(dt)] + [grads[n].to(s[n].dtype) for n in s["leaves"]]


def run(state):
    op = state["op"]
    if own:
        return _own_join(state) if op == "join" else _own_pack(state) if op == "pack" else _own_linear(state)
    with torch.no_grad():
        if op == "pack":
            return _pack_plain(state["x"], state["fmt"]).to(state["x"].dtype)
        return _plain_join(state) if op == "join" else _plain_linear(state)


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def _pack_exact(x, fmt):
    """Nearest value of the format's whole table, ties to the even entry."""
    if fmt == "e4m3":
        table = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)]
        table = table[:-1]                              # (the last code is NaN)
    else:
        table = [float(m) for m in range(128)]
    table = torch.tensor(table, dtype=torch.float64, device=x.device)
    powers = torch.tensor([2.0 ** k for k in range(-120, 128)], dtype=torch.float64, device=x.device)
    top, limit = table[-1].item(), _limit(x.dtype, fmt)
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for c in range(0, x.shape[1], BLOCK):
        v = x[:, c:c + BLOCK].double()
        bad = ~torch.isfinite(v)
        v = torch.where(bad, 0.0, v).clamp(-limit, limit)
        # (powers of two from a table: the device's pow need not be exact)
        scale = powers[torch.searchsorted(top * powers, v.abs().amax(dim=1, keepdim=True))]
        q = v.abs() / scale
        hi = torch.searchsorted(table, q.contiguous()).clamp(max=len(table) - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = table[hi] - q, q - table[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        out[:, c:c + BLOCK] = torch.where(bad, math.nan, torch.sign(v) * table[pick] * scale)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "pack":
        return _pack_exact(s["x"], case["fmt"])
    leaf = {n: v.detach().double() for n, v in s.items() if torch.is_tensor(v)}
    for n in s["leaves"]:
        leaf[n].requires_grad_(True)
    with torch.enable_grad():
        if case["op"] == "join":
            def norm(v, a, b):
                if case["norm"] == "rmsnorm":
                    return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + EPS) * a
                return (v - v.mean(-1, keepdim=True)) / (v.std(-1, keepdim=True) + EPS) * a + b
            gate = torch.sigmoid(leaf["g"]) if "g" in leaf else 1.0
            y = leaf["x"] + leaf.get("s", s["s"]) * gate * norm(leaf["f"], leaf["post_a"], leaf.get("post_b"))
            outs, cots = [y, norm(y, leaf["pre_a"], leaf.get("pre_b"))], ["d_y", "d_h"]
        else:
            z = torch.nn.functional.linear(leaf["x"], leaf["w"], leaf.get("b"))
            fn = dict(none=lambda t: t, relu=torch.relu, leakyrelu=lambda t: torch.nn.functional.leaky_relu(t, 0.2), gelu=torch.nn.functional.gelu,
                      silu=torch.nn.functional.silu)[case["act"]]
            y = fn(z) + leaf["r"] if "r" in leaf else fn(z)
            outs, cots = [y], ["d_y"]
        if not case["train"]:
            return [t.detach() for t in outs] if case["op"] == "join" else outs[0].detach()
        d_z = torch.autograd.grad(outs, [z], [leaf["d_y"]], retain_graph=True)[0] if case["op"] == "kept" else None
        grads = dict(zip(s["leaves"], torch.autograd.grad(outs, [leaf[n] for n in s["leaves"]], [leaf[c] for c in cots])))
    if d_z is not None:                                 # (the weight's gradient is defined on the kept rows)
        grads["w"] = d_z.t() @ _pack_exact(s["x"], case["fmt"])
    return [t.detach() for t in outs] + [grads[n] for n in s["leaves"]]


def work(case):
    """Bytes and operations one pass cannot do without: each input once, each output once; products two operations a term."""
    size = lambda name: 4 if name == "float32" else 2
    e, rows = size(case["dtype"]), case["rows"]
    if case["op"] == "pack":
        n = rows * case["width"]
        held = n + rows * (-(-case["width"] // BLOCK))
        return {"bytes": 2 * n * e + held, "flops": 4 * n}
    if case["op"] == "join":
        n, d = rows * case["width"], case["width"]
        gate = {"none": 0, "row": rows, "full": n}[case["gate"]]
        params = (2 if case["norm"] == "rmsnorm" else 4) + (1 if case["scale"] == "columns" else 0)
        # in x, f, g; out y, h; training adds in d_y, d_h and out d_x, d_f, d_g, and the parameters' gradients
        if not case["train"]:
            return {"bytes": (4 * n + gate) * e + params * d * size(case["params"]), "flops": 16 * n}
        return {"bytes": (8 * n + 2 * gate) * e + 2 * params * d * size(case["params"]), "flops": 48 * n}
    k, n = case["d_in"], case["d_out"]
    bias, res = n if case["bias"] else 0, rows * n if case["residual"] else 0
    fwd = rows * k + n * k + bias + res + rows * n
    if not case["train"]:
        return {"bytes": fwd * e, "flops": 2 * rows * n * k}
    held = rows * k + rows * (-(-k // BLOCK)) if case["op"] == "kept" else 0
    return {"bytes": (fwd + rows * n + rows * k + n * k + bias) * e + held, "flops": 6 * rows * n * k}
