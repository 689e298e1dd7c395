"""Row blocks (papr_amd/blocks.py) on the device against their formulas in 64 bits.

Tolerances.  u = eps / 2 is the rounding of the rows' type, e = 2^-24 float32's.  An output is computed in float32 and rounded once, so it is off by u |y| plus what
float32 leaves: a sum of n products is off by at most (n + few) e times the sum of the magnitudes, whatever its order; the three-part products of float32 rows leave
out 2^-26 of each term more and run six sums of n (6 n).  An activation has slope <= 1.13 and second derivative <= 0.8.  The backward pass reads z rounded to the rows'
type (u |z|) and rounds d_z to it (u |d_z|).  Each test writes its bound down as these terms, before any was run."""
import math

import numpy as np
import pytest
import torch

from papr_amd import blocks

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None
unit = lambda dt: torch.finfo(dt).eps / 2
tiny = lambda dt: 2.0 ** -25 if dt == torch.float16 else 1e-37          # half a step of the smallest numbers


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def close(got, ref, tol, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert got.shape == ref.shape and not bad.any(), "%s: %d of %d beyond the bound, worst %.3g times it" % (
        what, int(bad.sum()), bad.numel(), float((err / tol.clamp(min=1e-300)).nan_to_num(1e9).max()))


# ---------------------------------------------------------------------------------------------- linear layers
def act64(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "leakyrelu":
        return torch.where(z > 0, z, 0.2 * z), torch.where(z > 0, 1.0, 0.2).double()
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p * (1 + z * (1 - p))
    p = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    return z * p, p + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def linear_data(M, N, K, dt, seed, bias=True, res=True, whole=False):
    g = gen(seed)
    if whole:            # small whole numbers and halves: z is exact and never zero (relu's slope jumps there)
        r = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda").to(dt)
        x, w = r(M, K), r(N, K)
        b = torch.randint(-2, 3, (N,), generator=g, device="cuda").to(dt) + 0.5
    else:
        r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
        x, w, b = r(M, K), (r(N, K) * K ** -0.5).to(dt), r(N)
    return x, w, b.to(dt) if bias else None, torch.randn((M, N), generator=g, device="cuda").to(dt) if res else None, torch.randn((M, N), generator=g, device="cuda").to(dt)


def check_linear(x, w, b, r, d_y, act, keep=None, grads=True):
    dt, (M, K), N = x.dtype, x.shape, w.shape[0]
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(grads)
    y = blocks.linear_rows(x, w, b, r, act=act, keep=keep)
    assert y.dtype == dt and y.shape == (M, N) and y.is_contiguous()
    f = lambda t: None if t is None else t.detach().double()
    x6, w6, b6, r6, g6 = f(x), f(w), f(b), f(r), f(d_y)
    z = x6 @ w6.t() + (b6 if b is not None else 0)
    S = x6.abs() @ w6.abs().t() + (b6.abs() if b is not None else 0)
    v, slope = act64(z, act)
    ref = v + (r6 if r is not None else 0)
    u, n = unit(dt), (6 * K if dt == torch.float32 else K) + 16
    err_z = n * E32 * S
    close(y, ref, u * ref.abs() + 1.13 * err_z + 16 * E32 * (v.abs() + ref.abs()) + tiny(dt), "y")
    with torch.no_grad():
        assert torch.equal(blocks.linear_rows(x, w, b, r, act=act, keep=keep), y)
    if not grads:
        return
    got = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, d_y)))
    d_z = g6 * slope
    curve = 0.0 if act in ("none", "relu", "leakyrelu") else 0.8
    # d_z from the rounded z, in float32, then rounded to the rows' type (float32: no second rounding; "none" and relu: d_y or 0, exact)
    err_f = curve * (u * z.abs() + err_z) * g6.abs() + (0.0 if act in ("none", "relu") else 16 * E32 * (d_z.abs() + g6.abs()))
    err_d = err_f + (0.0 if act in ("none", "relu") else u * (d_z.abs() + err_f) + tiny(dt))
    m = lambda k: ((6 * k if dt == torch.float32 else k) + 16) * E32
    held = x6 if keep is None else blocks.pack_rows(x.detach(), keep).rows().double()
    ref = d_z @ w6
    close(got["x"], ref, u * ref.abs() + err_d @ w6.abs() + m(N) * (d_z.abs() @ w6.abs()) + tiny(dt), "d_x")
    ref = d_z.t() @ held
    close(got["w"], ref, u * ref.abs() + err_d.t() @ held.abs() + m(M) * (d_z.abs().t() @ held.abs()) + tiny(dt), "d_w")
    if b is not None:
        ref = d_z.sum(0)
        close(got["b"], ref, u * ref.abs() + err_f.sum(0) + (M + 16) * E32 * d_z.abs().sum(0) + tiny(dt), "d_b")
    if r is not None:
        assert torch.equal(got["r"], d_y)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (1, 64, 128), (3, 7, 5), (16, 256, 117), (37, 142, 256), (128, 128, 64), (129, 127, 65), (200, 300, 33), (1, 4096, 1030),
                                     (1000, 40, 257), (257, 512, 512), (5, 3, 2000), (2500, 8, 8), (640, 136, 72)])
def test_linear_rows_against_64_bits(dt, M, N, K):
    check_linear(*linear_data(M, N, K, dt, seed=M + N + K), act="gelu")


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("act", ["none", "relu", "leakyrelu", "silu"])
@pytest.mark.parametrize("bias, res", [(True, False), (False, True), (False, False)])
def test_linear_rows_epilogues(dt, act, bias, res):
    whole = act in ("relu", "leakyrelu")
    check_linear(*linear_data(70, 96, 48, dt, seed=5, bias=bias or whole, res=res, whole=whole), act=act)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("keep", ["e4m3", "int8"])
@pytest.mark.parametrize("M, N, K", [(1, 5, 3), (50, 64, 117), (300, 142, 96), (2048, 128, 160), (77, 33, 31)])
def test_linear_rows_with_kept_rows(dt, keep, M, N, K):
    check_linear(*linear_data(M, N, K, dt, seed=M + K), act="silu", keep=keep)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_linear_rows_split_sums_and_many_rows(dt):
    """d_w's sum over 30,011 rows runs in parts; the forward has more row tiles than workgroups fit at once."""
    check_linear(*linear_data(30011, 72, 40, dt, seed=2), act="silu")


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_linear_rows_strides_and_shapes(dt):
    """Rows inside wider rows (odd starts), a transposed weight, an expanded residual, three leading dimensions, an expanded gradient."""
    g = gen(11)
    wide = torch.randn((4, 9, 301), generator=g, device="cuda").to(dt)
    x = wide[..., 1:142]
    w = (torch.randn((141, 60), generator=g, device="cuda") / 12).to(dt).t()
    r = torch.randn((60,), generator=g, device="cuda").to(dt)
    y = blocks.linear_rows(x, w, None, r.expand(4, 9, 60), act="gelu")
    flat = blocks.linear_rows(x.reshape(-1, 141).contiguous(), w.contiguous(), None, r.expand(36, 60).contiguous(), act="gelu")
    assert y.shape == (4, 9, 60) and torch.equal(y.reshape(36, 60), flat)
    xs, ws, rs = (t.detach().clone().requires_grad_(True) for t in (wide, w, r))
    blocks.linear_rows(xs[..., 1:142], ws, None, rs.expand(4, 9, 60), act="gelu").sum().backward()
    x2, w2, r2 = x.detach().reshape(-1, 141).contiguous().requires_grad_(True), w.detach().contiguous().requires_grad_(True), r.detach().expand(36, 60).contiguous().requires_grad_(True)
    blocks.linear_rows(x2, w2, None, r2, act="gelu").backward(torch.ones((36, 60), device="cuda", dtype=dt))
    assert torch.equal(xs.grad[..., 1:142].reshape(36, 141), x2.grad) and not xs.grad[..., 0].any() and not xs.grad[..., 142:].any()
    assert torch.equal(ws.grad, w2.grad) and torch.equal(rs.grad, torch.full_like(r, 36.0))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("M, N, K, act, keep", [(8191, 1001, 1003, "silu", None), (8192, 1000, 701, "none", None), (6000, 501, 1408, "gelu", None), (9000, 701, 800, "silu", "int8"),
                                                (3001, 1104, 1009, "none", None)])
def test_linear_rows_of_odd_16_bit_rows_that_are_copied_into_whole_vectors(dt, M, N, K, act, keep):
    """Long products of odd rows stream from padded copies (x, W, d_y, each where its own width is odd; d_z leaves its kernel padded)."""
    check_linear(*linear_data(M, N, K, dt, seed=M % 97), act=act, keep=keep)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("M, N, K", [(2048, 2048, 512), (4100, 1040, 264), (700, 3000, 1000)])
def test_linear_rows_large_tiles(dt, M, N, K):
    check_linear(*linear_data(M, N, K, dt, seed=M % 89), act="gelu")


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16], ids=ids)
def test_small_products_lose_nothing_to_a_rounded_d_z(dt):
    """Up to 2^28 terms d_z stays in float32: what is left beside the final rounding (rms u / sqrt 3 of uniform errors, e_out) is z's own, at most 0.8 u |z| rms through the
    slope's derivative -- under half of e_out: together below 1.15 e_out (with d_z rounded too it was 1.45)."""
    x, w, b, r, d_y = linear_data(400, 512, 512, dt, seed=12)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(blocks.linear_rows(x, w, b, r, act="silu"), leaves, d_y)
    x6, w6 = (t.detach().double() for t in (x, w))
    d_z = d_y.double() * act64(x6 @ w6.t() + b.double(), "silu")[1]
    for g, ref in zip(got, (d_z @ w6, d_z.t() @ x6)):
        floor = (ref.to(dt).double() - ref).norm()
        assert (g.double() - ref).norm() <= 1.15 * floor


def test_linear_rows_far_rows_and_single_rows():
    """Rows five million elements apart (their tile's offsets pass 32 bits: a copy), a vector instead of rows, a bias and weight that are views."""
    store = torch.zeros((5_000_000 * 39 + 40,), device="cuda", dtype=torch.float16)
    far = store.as_strided((40, 32), (5_000_000, 1))
    far.copy_(torch.randn((40, 32), generator=gen(3), device="cuda"))
    w, b = torch.randn((2, 64, 50), generator=gen(4), device="cuda").half()[1, :, 3:35], torch.randn((64, 2), generator=gen(5), device="cuda").half()[:, 1]
    assert torch.equal(blocks.linear_rows(far, w, b), blocks.linear_rows(far.contiguous(), w.contiguous(), b.contiguous()))
    assert torch.equal(blocks.norm_rows(far, blocks.Norm("rmsnorm")), blocks.norm_rows(far.contiguous(), blocks.Norm("rmsnorm")))
    one = blocks.linear_rows(far[0], w, b, residual=b, act="silu")
    assert one.shape == (64,) and torch.equal(one, blocks.linear_rows(far[:1], w, b, residual=b[None], act="silu")[0])
    assert blocks.pack_rows(far[0]).rows().shape == (32,)


def test_operands_written_to_and_graphs_run_twice_are_refused():
    x, w = torch.randn((8, 16), device="cuda"), torch.randn((16, 16), device="cuda", requires_grad=True)
    y = blocks.linear_rows(x, w, act="silu")
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    gain = torch.ones(16, device="cuda", requires_grad=True)
    y = blocks.join_rows(x, x * 2, post=blocks.Norm("rmsnorm", gain))
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = blocks.join_rows(x, x * 2, post=blocks.Norm("rmsnorm", gain))
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_linear_rows_of_nothing():
    for dt in DTYPES:
        x, w, b = torch.zeros((0, 24), device="cuda", dtype=dt, requires_grad=True), torch.ones((8, 24), device="cuda", dtype=dt, requires_grad=True), torch.ones((8,), device="cuda", dtype=dt, requires_grad=True)
        y = blocks.linear_rows(x, w, b, act="gelu", keep="e4m3")
        y.sum().backward()
        assert y.shape == (0, 8) and x.grad.shape == (0, 24) and not w.grad.any() and not b.grad.any()


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
def test_linear_rows_only_the_gradients_asked_for(dt):
    x, w, b, r, d_y = linear_data(40, 48, 56, dt, seed=3)
    full = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
    want = torch.autograd.grad(blocks.linear_rows(*full, act="silu"), full, d_y)
    for i in range(4):
        ts = [t.detach().clone().requires_grad_(i == j) for j, t in enumerate((x, w, b, r))]
        got = torch.autograd.grad(blocks.linear_rows(*ts, act="silu"), [ts[i]], d_y)[0]
        assert torch.equal(got, want[i]), i


def test_linear_rows_values_that_are_not_finite_stay_where_they_are():
    """A NaN or an infinity in one row of x reaches that row of y only (and every row of d_w's column); the overflow of float16 is infinite."""
    for dt in DTYPES:
        for bad in (math.nan, math.inf):
            x, w, _, _, d_y = linear_data(150, 130, 70, dt, seed=4)
            clean = blocks.linear_rows(x, w)
            x[77, 69] = bad
            y = blocks.linear_rows(x, w)
            assert torch.equal(y[:77], clean[:77]) and torch.equal(y[78:], clean[78:]) and not torch.isfinite(y[77]).any()
    x = torch.full((2, 64), 200.0, device="cuda", dtype=torch.float16)
    assert torch.isinf(blocks.linear_rows(x, x)).all()


def test_linear_rows_gradient_against_differences():
    """(L(p + t d) - L(p - t d)) / 2t along one direction, L = sum(c y): the third derivative leaves t^2 / 6 of the term's size, float32's forward e n S / t."""
    x, w, b, r, c = (t for t in linear_data(24, 40, 32, torch.float32, seed=9))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(blocks.linear_rows(*leaves, act="silu"), leaves, c)
    g = gen(10)
    dirs = [torch.randn(t.shape, generator=g, device="cuda") for t in leaves]
    t = 2.0 ** -7
    L = lambda sign: (c.double() * blocks.linear_rows(*[(p + sign * t * d).detach() for p, d in zip((x, w, b, r), dirs)], act="silu").double()).sum()
    diff = (L(1) - L(-1)) / (2 * t)
    want = sum((gr.double() * d.double()).sum() for gr, d in zip(grads, dirs))
    scale = sum((gr.double() * d.double()).abs().sum() for gr, d in zip(grads, dirs))
    assert abs(float(diff - want)) <= 2e-3 * float(scale) ** 0.5 * float(c.double().norm()), (float(diff), float(want))


# ---------------------------------------------------------------------------------------------- rows in 8 bits
def packed64(x, fmt):
    """The definition, on the host in numpy: the smallest power of two, the nearest entry of the format's table, ties to the even entry."""
    table = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1] if fmt == "e4m3" else range(128), dtype=np.float64)
    limit = (1.875 if fmt == "e4m3" else 1.984375) * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    v = x.detach().double().cpu().numpy()
    out = np.empty_like(v)
    for c in range(0, v.shape[1], 32):
        s = v[:, c:c + 32]
        bad = ~np.isfinite(s)
        s = np.clip(np.where(bad, 0.0, s), -limit, limit)
        peak = np.abs(s).max(axis=1, keepdims=True)
        e = np.full_like(peak, -120.0)
        while (peak > table[-1] * 2.0 ** e).any():
            e = np.where(peak > table[-1] * 2.0 ** e, e + 1, e)
        q = np.abs(s) / 2.0 ** e
        hi = np.minimum(np.searchsorted(table, q), len(table) - 1)
        lo = np.maximum(hi - 1, 0)
        up, down = table[hi] - q, q - table[lo]
        pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
        out[:, c:c + 32] = np.where(bad, np.nan, np.sign(s) * table[pick] * 2.0 ** e)
    return out


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows, width", [(1, 1), (3, 31), (5, 32), (4, 33), (37, 142), (64, 256), (9, 117), (130, 1000)])
def test_packed_rows_are_the_nearest_values(dt, fmt, rows, width):
    g = gen(rows * width)
    x = (torch.randn((rows, width), generator=g, device="cuda") * torch.exp(3 * torch.randn((rows, 1), generator=g, device="cuda"))).to(dt)
    x[0] = 0
    x[-1, -1] = 0.0 if width == 1 else x[-1, -1]
    p = blocks.pack_rows(x, fmt)
    got = p.rows()
    assert got.dtype == dt and got.shape == x.shape and p.codes.shape == (rows, (width + 31) // 32 * 32) and not p.codes[:, width:].any()
    np.testing.assert_array_equal(got.double().cpu().numpy(), packed64(x, fmt))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_packed_rows_ties_extremes_and_what_is_not_finite(fmt):
    """Every bfloat16 and float16 bit pattern, in blocks of neighbours: ties (most values between two codes of a block are), the smallest and largest scales,
    infinities and NaN; and float32 rows around the borders of a scale."""
    for dt in (torch.float16, torch.bfloat16):
        x = torch.arange(-32768, 32768, device="cuda", dtype=torch.int32).to(torch.int16).view(dt).reshape(-1, 128)
        np.testing.assert_array_equal(blocks.pack_rows(x, fmt).rows().double().cpu().numpy(), packed64(x, fmt))
    top = 448.0 if fmt == "e4m3" else 127.0
    edges = []
    for s in (2.0 ** -140, 2.0 ** -121, 2.0 ** -120, 2.0 ** -3, 1.0, 2.0 ** 100, 2.0 ** 119):
        t = np.float32(top * s)
        edges += [t, np.nextafter(t, np.float32(np.inf)), np.nextafter(t, np.float32(0))]
    edges += [np.float32(3.4028234e38), np.float32(1.4e-45), np.float32(0.0)]
    x = torch.tensor(np.array(edges, dtype=np.float32)[:, None] * np.array([1, -0.5, 0.3, 0.01], dtype=np.float32)[None], device="cuda")
    got = blocks.pack_rows(x, fmt).rows()
    assert torch.isfinite(got).all()
    np.testing.assert_array_equal(got.double().cpu().numpy(), packed64(x, fmt))


def test_packed_rows_strides_and_no_rows():
    g = gen(1)
    wide = torch.randn((6, 7, 200), generator=g, device="cuda")
    for dt in DTYPES:
        w = wide.to(dt)
        for view in (w[..., 3:150], w[:, ::2, :128], w.transpose(1, 2), w[0, 0].expand(5, 200)):
            got, want = blocks.pack_rows(view).rows(), blocks.pack_rows(view.contiguous()).rows()
            assert got.shape == view.shape and torch.equal(got, want)
        assert blocks.pack_rows(w[:0]).rows().shape == (0, 7, 200)


# ---------------------------------------------------------------------------------------------- the joint of a block
def norm64(v, norm):
    """(value, standardised, divisor): the divisor times the deviation's slope handled in the caller through autograd"""
    if norm.kind == "none":
        n = v
    elif norm.kind == "rmsnorm":
        n = v / torch.sqrt((v * v).mean(-1, keepdim=True) + norm.eps)
    else:
        n = (v - v.mean(-1, keepdim=True)) / (v.std(-1, keepdim=True) + norm.eps)
    return n * (1 if norm.gain is None else norm.gain) + (0 if norm.shift is None else norm.shift)


def divisor(v, norm):
    if norm.kind == "none":
        return torch.ones_like(v[..., :1])
    if norm.kind == "rmsnorm":
        return torch.sqrt((v * v).mean(-1, keepdim=True) + norm.eps)
    return v.std(-1, keepdim=True) + norm.eps


def norm_err(v, err, norm):
    """Bound on the standardised value's float32 error, given v's: statistics of `width` terms in trees of 8 + 10 steps (64 e covers them and the divisions), and
    v's own error through the value, the mean and the divisor."""
    if norm.kind == "none":
        return err
    div = divisor(v, norm)
    c = v - v.mean(-1, keepdim=True) if norm.kind == "layernorm" else v
    n = (c / div).abs()
    err = err + 64 * E32 * (v.abs() + v.abs().mean(-1, keepdim=True))
    return (err + err.mean(-1, keepdim=True) + n * torch.sqrt((err * err).mean(-1, keepdim=True)) * 1.5) / div + 64 * E32 * n


def check_join(rows, width, dt, post, pre, gate, scale, params=torch.float32, gate_act="sigmoid", seed=0, use=(True, True), lead=None):
    g = gen(seed)
    r = lambda *s, std=1.0, mean=0.0, t=dt: (torch.randn(s, generator=g, device="cuda") * std + mean).to(t)
    shape = (rows, width) if lead is None else lead + (width,)
    x, f = r(*shape), r(*shape, std=0.7, mean=0.2)
    gt = None if gate == "none" else r(*shape) if gate == "full" else r(*(shape[:-1] + (1,)))
    sc = r(width, std=0.1, mean=0.4, t=params) if scale == "columns" else 0.37
    mk = lambda kind: None if kind is None else blocks.Norm(kind, r(width, std=0.2, mean=1.0, t=params), r(width, std=0.2, t=params) if kind != "rmsnorm" else None)
    post, pre = mk(post), mk(pre)
    named = dict(x=x, f=f, gate=gt, scale=sc, post_gain=post and post.gain, post_shift=post and post.shift, pre_gain=pre and pre.gain, pre_shift=pre and pre.shift)
    leaves = {n: t for n, t in named.items() if torch.is_tensor(t)}
    for t in leaves.values():
        t.requires_grad_(True)
    out = blocks.join_rows(x, f, gate=gt, scale=sc, post=post, pre=pre, gate_act=gate_act)
    out = list(out) if isinstance(out, tuple) else [out]
    with torch.no_grad():
        again = blocks.join_rows(x, f, gate=gt, scale=sc, post=post, pre=pre, gate_act=gate_act)
        assert all(torch.equal(a, b) for a, b in zip(out, again if isinstance(again, tuple) else [again]))
    # the formulas in 64 bits
    L = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    n64 = lambda n, which: None if n is None else blocks.Norm(n.kind, L.get(which + "_gain"), L.get(which + "_shift"), n.eps)
    post6, pre6 = n64(post, "post"), n64(pre, "pre")
    acts = {"none": lambda v: v, "sigmoid": torch.sigmoid, "silu": lambda v: v * torch.sigmoid(v)}
    ga = acts[gate_act](L["gate"]) if gt is not None else torch.ones((), device="cuda", dtype=torch.float64)
    s6 = L.get("scale", 0.37)
    p = norm64(L["f"], post6) if post else L["f"]
    y6 = L["x"] + s6 * ga * p
    refs = [y6] + ([norm64(y6, pre6)] if pre else [])
    u = unit(dt)
    with torch.no_grad():
        e_p = norm_err(L["f"], torch.zeros_like(p), post6) * L["post_gain"].abs() + 4 * E32 * p.abs() if post else torch.zeros_like(p)
        sg = (s6 * ga).abs() * torch.ones_like(p)
        e_y = sg * (e_p + 16 * E32 * (p.abs() + (p * (gt.double().abs() if gt is not None else 0)).abs())) + 4 * E32 * y6.abs()
        close(out[0], y6, u * y6.abs() + e_y + tiny(dt), "y")
        if pre:
            h6 = refs[1]
            e_h = norm_err(y6, e_y, pre6) * L["pre_gain"].abs() + 4 * E32 * h6.abs()
            close(out[1], h6, u * h6.abs() + e_h + tiny(dt), "h")
    cots = [r(*shape) for _ in out]
    pick = [i for i in range(len(out)) if use[i]]
    got = dict(zip(leaves, torch.autograd.grad([out[i] for i in pick], list(leaves.values()), [cots[i] for i in pick], allow_unused=True)))
    ref = dict(zip(L, torch.autograd.grad([refs[i] for i in pick], list(L.values()), [cots[i].double() for i in pick], allow_unused=True)))
    # Every term of a gradient passes at most two norms and a sum over the row or the rows.  Majorant: the same expressions in magnitudes; each factor is good to
    # the relative error k of the standardised rows (their bound over their root mean square), a sum over the rows adds (sequential per lane, then a tree over
    # the partial rows: at most rows / 256 + 64 steps).
    with torch.no_grad():
        rms = lambda t: torch.sqrt((t * t).mean(-1, keepdim=True))
        k = 64 * E32
        if post:
            k = k + (norm_err(L["f"], torch.zeros_like(p), post6) if post.kind != "none" else 0 * p).amax()
        if pre:
            k = k + norm_err(y6, e_y, pre6).amax()
        k = 8 * k
        dy = cots[0].double().abs() if use[0] else torch.zeros_like(y6)
        if pre and use[1]:
            dh = cots[1].double().abs()
            yn = norm64(y6, blocks.Norm(pre.kind, None, None, pre.eps)).abs()
            dn = dh * L["pre_gain"].abs()
            back = dn if pre.kind == "none" else (dn + 2 * yn * (dn * yn).mean(-1, keepdim=True) + dn.mean(-1, keepdim=True)) / divisor(y6, pre6)
            dy = dy + back
            maj = {"pre_gain": dh * yn + dh, "pre_shift": dh}
        else:
            maj = {}
        gv = gt.double().abs() if gt is not None else torch.ones_like(ga)
        ga_m = ga.abs() * torch.ones_like(p)
        fn = norm64(L["f"], blocks.Norm(post.kind, None, None, post.eps)).abs() if post else L["f"].abs()
        pm = fn * (L["post_gain"].abs() if post else 1) + (L["post_shift"].abs() if post and post.shift is not None else 0)
        dp = dy * (s6 * ga).abs()
        dn = dp * (L["post_gain"].abs() if post else 1)
        maj["x"] = dy
        maj["f"] = dn if not post or post.kind == "none" else (dn + 2 * fn * (dn * fn).mean(-1, keepdim=True) + dn.mean(-1, keepdim=True)) / divisor(L["f"], post6)
        maj["scale"] = dy * ga_m * pm
        slope = torch.ones_like(gv) if gate_act == "none" else (1.1 + gv)
        maj["gate"] = dy * (s6 * pm if torch.is_tensor(s6) else abs(s6) * pm) * slope
        maj["post_gain"], maj["post_shift"] = dp * fn, dp
        for n in leaves:
            if ref[n] is None:
                assert got[n] is None or not got[n].any(), n
                continue
            m = maj.get(n, torch.zeros_like(y6)).abs()
            tol = k * m
            if n in ("scale", "post_gain", "post_shift", "pre_gain", "pre_shift"):
                m, tol = m.reshape(-1, width).sum(0), tol.reshape(-1, width).sum(0)
                tol = tol + (rows / 256 + 64) * E32 * m
            elif n == "gate" and gate == "row" and width > 1:
                tol = tol.sum(-1, keepdim=True)
            close(got[n], ref[n], unit(leaves[n].dtype) * ref[n].abs() + tol + tiny(leaves[n].dtype), "d " + n)
            assert got[n].dtype == leaves[n].dtype


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("rows, width", [(1, 2), (3, 7), (1, 64), (33, 117), (40, 256), (7, 142), (130, 512), (5, 1000), (6, 1023), (9, 2048), (3, 4096), (2, 5001), (3, 8192)])
def test_join_rows_against_64_bits(dt, rows, width):
    check_join(rows, width, dt, "layernorm", "layernorm", "full", "columns", seed=rows + width)
    check_join(rows, width, dt, "rmsnorm", "rmsnorm", "row", "number", params=dt, seed=rows + width + 1)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("post", [None, "none", "layernorm", "rmsnorm"])
@pytest.mark.parametrize("pre", [None, "none", "layernorm", "rmsnorm"])
def test_join_rows_every_pair_of_norms(dt, post, pre):
    check_join(21, 96, dt, post, pre, "row", "columns", seed=4)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("gate", ["none", "row", "full"])
@pytest.mark.parametrize("gate_act", ["none", "sigmoid", "silu"])
def test_join_rows_gates(dt, gate, gate_act):
    check_join(18, 50, dt, "rmsnorm", "layernorm", gate, "number", gate_act=gate_act, seed=6)


@pytest.mark.parametrize("use", [(True, False), (False, True)])
def test_join_rows_one_output_used(use):
    for dt in DTYPES:
        check_join(18, 72, dt, "layernorm", "rmsnorm", "full", "columns", use=use, seed=8)


def test_join_rows_many_rows_and_leading_dimensions():
    for dt in DTYPES:
        check_join(20000, 40, dt, "layernorm", "layernorm", "full", "columns", seed=12)
        check_join(30, 40, dt, "layernorm", "layernorm", "row", "columns", seed=13, lead=(2, 3, 5))


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("width", [4104, 4602, 4601])
@pytest.mark.parametrize("post, pre, gate, use", [("layernorm", "rmsnorm", "row", (True, True)), (None, "layernorm", "full", (False, True)), ("rmsnorm", "none", "none", (True, True)),
                                                  ("rmsnorm", "layernorm", "full", (True, False)), ("none", None, "row", (True, True))])
def test_join_rows_widest_rows_several_a_workgroup(dt, width, post, pre, gate, use):
    """Rows above 4096 columns (whole vectors, pairs and single values), more of them than workgroups."""
    check_join(521, width, dt, post, pre, gate, "columns", seed=width, use=use)


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("kind", ["layernorm", "rmsnorm", "none"])
def test_norm_rows(dt, kind):
    g = gen(3)
    x = (torch.randn((50, 117), generator=g, device="cuda") * 2 + 1).to(dt).requires_grad_(True)
    a, b = torch.randn((117,), generator=g, device="cuda").requires_grad_(True), torch.randn((117,), generator=g, device="cuda").requires_grad_(True)
    d = torch.randn((50, 117), generator=g, device="cuda").to(dt)
    h = blocks.norm_rows(x, blocks.Norm(kind, a, b))
    x6, a6, b6 = (t.detach().double().requires_grad_(True) for t in (x, a, b))
    ref = norm64(x6, blocks.Norm(kind, a6, b6))
    got, want = torch.autograd.grad(h, [x, a, b], d), torch.autograd.grad(ref, [x6, a6, b6], d.double())
    with torch.no_grad():
        n = blocks.Norm(kind, a6, b6)
        e = norm_err(x6, 0 * x6, n)
        close(h, ref.detach(), unit(dt) * ref.abs() + e * a6.abs() + 4 * E32 * (ref.abs() + b6.abs()) + tiny(dt), "h")
        xn = norm64(x6, blocks.Norm(kind)).abs()
        k = 8 * (e.amax() + 64 * E32)
        dn = d.double().abs() * a6.abs()
        back = dn if kind == "none" else (dn + 2 * xn * (dn * xn).mean(-1, keepdim=True) + dn.mean(-1, keepdim=True)) / divisor(x6, n)
        close(got[0], want[0], unit(dt) * want[0].abs() + k * back + tiny(dt), "d x")
        close(got[1], want[1], E32 * want[1].abs() + ((k + 66 * E32) * d.double().abs() * (xn + 1)).sum(0), "d gain")
        close(got[2], want[2], E32 * want[2].abs() + (66 * E32 * d.double().abs()).sum(0), "d shift")


def test_join_rows_constant_rows_and_rows_that_are_not_finite():
    """A constant row has deviation 0: its value is the shift and its gradient finite; a NaN row stays alone; no rows at all."""
    for dt in DTYPES:
        x = torch.full((3, 64), 2.0, device="cuda", dtype=dt, requires_grad=True)
        a, b = torch.ones(64, device="cuda", requires_grad=True), torch.full((64,), 0.5, device="cuda", requires_grad=True)
        h = blocks.norm_rows(x, blocks.Norm("layernorm", a, b))
        h.float().square().sum().backward()
        assert torch.equal(h, torch.full_like(h, 0.5)) and torch.isfinite(x.grad).all() and torch.equal(a.grad, torch.zeros_like(a))
        g = gen(2)
        x, f = (torch.randn((40, 96), generator=g, device="cuda").to(dt) for _ in range(2))
        norm = blocks.Norm("rmsnorm", torch.ones(96, device="cuda"))
        clean = blocks.join_rows(x, f, post=norm, pre=norm)
        f2 = f.clone()
        f2[13, 5] = math.nan
        y, h = blocks.join_rows(x, f2, post=norm, pre=norm)
        keep = torch.arange(40, device="cuda") != 13
        assert torch.equal(y[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep]) and torch.isnan(y[13]).all() and torch.isnan(h[13]).all()
        e = torch.zeros((0, 96), device="cuda", dtype=dt, requires_grad=True)
        gain = torch.ones(96, device="cuda", requires_grad=True)
        y, h = blocks.join_rows(e, e, post=blocks.Norm("rmsnorm", gain), pre=norm)
        (y.sum() + h.sum()).backward()
        assert y.shape == (0, 96) and e.grad.shape == (0, 96) and not gain.grad.any()


def test_join_rows_strides_offsets_and_shared_tensors():
    """Views with odd starts give the aligned rows' values up to the order of a row's sums; one tensor as x and f, one norm used twice: its gradient is the sum."""
    g = gen(5)
    wide = torch.randn((30, 300), generator=g, device="cuda")
    norm = blocks.Norm("layernorm", torch.rand(128, generator=g, device="cuda") + 0.5, torch.rand(128, generator=g, device="cuda"))
    for dt in DTYPES:
        w = wide.to(dt)
        y, h = blocks.join_rows(w[:, 1:129], w[:, 150:278], gate=w[:, 3:131], post=norm, pre=norm)
        y2, h2 = blocks.join_rows(w[:, 1:129].contiguous(), w[:, 150:278].contiguous(), gate=w[:, 3:131].contiguous(), post=norm, pre=norm)
        close(y, y2.double(), 2 * unit(dt) * y2.double().abs() + 64 * E32 * 4 + tiny(dt))
        close(h, h2.double(), 2 * unit(dt) * h2.double().abs() + 64 * E32 * 16 + tiny(dt))
    x = torch.randn((20, 128), generator=g, device="cuda").requires_grad_(True)
    gain, shift = (t.clone().requires_grad_(True) for t in norm[1:3])
    y, h = blocks.join_rows(x, x, post=blocks.Norm("layernorm", gain, shift), pre=blocks.Norm("layernorm", gain, shift))
    (y.sum() + (h * h).sum()).backward()
    x6, a6, b6 = (t.detach().double().requires_grad_(True) for t in (x, gain, shift))
    n6 = blocks.Norm("layernorm", a6, b6)
    y6 = x6 + norm64(x6, n6)
    (y6.sum() + norm64(y6, n6).square().sum()).backward()
    for got, want in ((x.grad, x6.grad), (gain.grad, a6.grad), (shift.grad, b6.grad)):
        close(got, want, 1e-4 * want.abs().max() + 0 * want)


# ---------------------------------------------------------------------------------------------- a run of them together
def block64(p, x, keep):
    h = norm64(x, blocks.Norm("layernorm", p["a0"], p["b0"]))
    u, _ = act64(h @ p["w1"].t() + p["c1"], "gelu")
    f = u @ p["w2"].t() + p["c2"]
    y = x + p["s"] * torch.sigmoid(x @ p["wg"].t()) * norm64(f, blocks.Norm("layernorm", p["a1"], p["b1"]))
    return y, norm64(y, blocks.Norm("rmsnorm", p["a2"], None))


def block(p, x, keep):
    h = blocks.norm_rows(x, blocks.Norm("layernorm", p["a0"], p["b0"]))
    u = blocks.linear_rows(h, p["w1"], p["c1"], act="gelu", keep=keep)
    f = blocks.linear_rows(u, p["w2"], p["c2"], keep=keep)
    return blocks.join_rows(x, f, gate=blocks.linear_rows(x, p["wg"]), scale=p["s"], post=blocks.Norm("layernorm", p["a1"], p["b1"]), pre=blocks.Norm("rmsnorm", p["a2"], None))


def block_params(dt, d, hidden, seed):
    g = gen(seed)
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(s, generator=g, device="cuda") * std + mean).to(dt)
    return dict(a0=r(d, std=0.1, mean=1), b0=r(d, std=0.1), w1=r(hidden, d, std=d ** -0.5), c1=r(hidden, std=0.1), w2=r(d, hidden, std=hidden ** -0.5), c2=r(d, std=0.1),
                a1=r(d, std=0.1, mean=1), b1=r(d, std=0.1), s=r(d, std=0.1, mean=0.5), wg=r(1, d, std=d ** -0.5), a2=r(d, std=0.1, mean=1))


@pytest.mark.parametrize("dt", DTYPES, ids=ids)
@pytest.mark.parametrize("keep", [None, "e4m3", "int8"])
@pytest.mark.parametrize("rows, d, hidden", [(64, 117, 256), (1, 64, 128), (300, 256, 512)])
def test_a_residual_block_forward_and_backward(dt, keep, rows, d, hidden):
    """norm -> linear + gelu -> linear -> gated joint, gate a linear layer of its own.  The chain's intermediate rows are rounded to the rows' type between the
    operators (each half a step u); of those about ten a value of y and twice as many a gradient passes, amplified by at most the layers' gains (about 1): 64 u of the
    tensor's largest value (the float32 chain: 2^-17 of it, from sums of up to 6 x 512 terms).  Kept rows change the two weights' gradients only: by their own
    rounding (2^-4 / 2^-7 relative to a block's largest), averaged over the rows."""
    p = block_params(dt, d, hidden, 1)
    x = torch.randn((rows, d), generator=gen(2), device="cuda").to(dt)
    leaves = dict(p, x=x)
    for t in leaves.values():
        t.requires_grad_(True)
    y, h = block(p, x, keep)
    cots = [torch.randn((rows, d), generator=gen(3 + i), device="cuda").to(dt) for i in range(2)]
    got = dict(zip(leaves, torch.autograd.grad([y, h], list(leaves.values()), cots)))
    L = {n: t.detach().double().requires_grad_(True) for n, t in leaves.items()}
    y6, h6 = block64(L, L["x"], keep)
    ref = dict(zip(leaves, torch.autograd.grad([y6, h6], list(L.values()), [c.double() for c in cots])))
    bar = 2.0 ** -17 if dt == torch.float32 else 64 * unit(dt)
    for name, a, b in [("y", y, y6.detach()), ("h", h, h6.detach())] + [(n, got[n], ref[n]) for n in leaves]:
        extra = 0.0 if keep is None or name not in ("w1", "w2") else 2.0 ** -4 if keep == "e4m3" else 2.0 ** -6
        assert torch.isfinite(a).all()
        close(a, b, (bar + extra) * b.abs().max() + 0 * b, name)
    if keep is None:
        return
    with torch.no_grad():
        plain = block(p, x, None)
    assert torch.equal(plain[0], y) and torch.equal(plain[1], h)


def test_runs_repeat_bit_for_bit_and_streams_do_not_disturb_each_other():
    """The same bits on every run; two streams at once (each with its own workspace) give what one after the other gives."""
    dt = torch.bfloat16
    p = {n: t.requires_grad_(True) for n, t in block_params(dt, 256, 512, 1).items()}
    xs = [torch.randn((4096, 256), generator=gen(i), device="cuda").to(dt).requires_grad_(True) for i in (5, 6)]
    cot = [torch.randn((4096, 256), generator=gen(7 + i), device="cuda").to(dt) for i in range(2)]
    step = lambda x: torch.autograd.grad(block(p, x, "e4m3"), [x] + list(p.values()), cot)
    first = [step(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(3):
        torch.cuda.synchronize()
        outs = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                outs.append(step(x))
        torch.cuda.synchronize()
        for a, b in zip(first, outs):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_captured_steps_replay_with_new_inputs():
    """Forward and backward captured into two graphs whose replays alternate with eager work: every replay equals the eager result on the inputs of the moment.  (The
    graphs' leaves are their own: no eager graph of them is alive while they are captured.)"""
    dt = torch.float16
    p = block_params(dt, 142, 256, 1)
    eager = {n: t.clone().requires_grad_(True) for n, t in p.items()}
    runs = []
    for k, keep in enumerate((None, "int8")):
        mine = {n: t.clone().requires_grad_(True) for n, t in p.items()}
        x = torch.zeros((500, 142), device="cuda", dtype=dt, requires_grad=True)
        cot = [torch.ones((500, 142), device="cuda", dtype=dt) for _ in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(block(mine, x, keep), [x] + list(mine.values()), cot)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(mine, x, keep)
            grads = torch.autograd.grad(out, [x] + list(mine.values()), cot)
        runs.append((graph, x, [t.detach() for t in out], grads, keep, cot, mine))      # (the graph reads its parameters where they lie: they live as long as it)
    for turn in range(3):
        for graph, x, out, grads, keep, cot, _ in runs:
            new = torch.randn((500, 142), generator=gen(20 + turn), device="cuda").to(dt)
            with torch.no_grad():
                x.copy_(new)
            graph.replay()
            e = new.clone().requires_grad_(True)
            want = block(eager, e, keep)
            want_g = torch.autograd.grad(want, [e] + list(eager.values()), cot)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)) and all(torch.equal(a, b) for a, b in zip(grads, want_g))


def test_a_step_accumulates_into_leaves_and_tracks_only_what_is_asked():
    """backward() into .grad twice is twice the gradient; without grad mode nothing is tracked; the residual alone passes its gradient through."""
    p = {n: t.requires_grad_(True) for n, t in block_params(torch.bfloat16, 64, 128, 1).items()}
    x = torch.randn((33, 64), generator=gen(2), device="cuda").bfloat16()
    for _ in range(2):
        y, h = block(p, x, "e4m3")
        (y.float().sum() + h.float().square().sum()).backward()
    twice = {n: t.grad.clone() for n, t in p.items()}
    for t in p.values():
        t.grad = None
    y, h = block(p, x, "e4m3")
    (y.float().sum() + h.float().square().sum()).backward()
    assert all(torch.equal(twice[n], p[n].grad * 2) for n in p)
    with torch.no_grad():
        assert not any(t.requires_grad for t in block(p, x, None))
    r = torch.randn((33, 128), device="cuda").bfloat16().requires_grad_(True)
    blocks.linear_rows(x, p["w1"].detach(), None, r, act="gelu").sum().backward()
    assert torch.equal(r.grad, torch.ones_like(r))


def test_second_derivatives_are_refused():
    x, w = torch.randn((4, 8), device="cuda", requires_grad=True), torch.randn((6, 8), device="cuda", requires_grad=True)
    g, = torch.autograd.grad(blocks.linear_rows(x, w, act="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    y, h = blocks.join_rows(x, x, pre=blocks.Norm("rmsnorm"))
    g, = torch.autograd.grad((y * h).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        (g.sum() + x.sum()).backward()


def test_packed_rows_in_other_strides_and_places():
    """Codes that moved to host memory and back, lie with gaps between rows, or start on an odd byte stand for the same values."""
    x = torch.randn((33, 100), generator=gen(1), device="cuda").bfloat16()
    p = blocks.pack_rows(x, "int8")
    want, codes, exps = p.rows(), p.codes, p.exps
    wide = torch.zeros((33, 200), dtype=torch.uint8, device="cuda")
    wide[:, 3:131] = codes
    odd = torch.empty(codes.numel() + 1, dtype=torch.uint8, device="cuda")[1:].view_as(codes).copy_(codes)
    for c, e in ((codes.cpu().cuda(), exps.cpu().cuda()), (wide[:, 3:131], exps.t().contiguous().t()), (odd, exps)):
        p.codes, p.exps = c, e
        assert torch.equal(p.rows(), want)
    p.codes = codes.cpu()
    with pytest.raises((ValueError, RuntimeError)):
        p.rows()


@pytest.mark.parametrize("keep", [None, "e4m3"])
def test_saved_tensors_may_leave_the_device_or_be_recomputed(keep):
    """Hooks of saved tensors and checkpoints bring back what was kept: the same gradients, to the bit, strided and padded rows among them."""
    from torch.utils.checkpoint import checkpoint
    p = {n: t.requires_grad_(True) for n, t in block_params(torch.bfloat16, 142, 256, 1).items()}
    x = torch.randn((37, 160), generator=gen(2), device="cuda").bfloat16()[:, 3:145].requires_grad_(True)
    cot = [torch.randn((37, 142), generator=gen(3 + i), device="cuda").bfloat16() for i in range(2)]
    grads = lambda out: torch.autograd.grad(out, [x] + list(p.values()), cot)
    want = grads(block(p, x, keep))
    with torch.autograd.graph.save_on_cpu():
        out = block(p, x, keep)
    away = grads(out)
    again = grads(checkpoint(lambda t: block(p, t, keep), x, use_reentrant=False))
    for other in (away, again):
        assert all(torch.equal(a, b) for a, b in zip(want, other))


@pytest.mark.parametrize("back", [lambda t: t.cpu(), lambda t: t[:-1], lambda t: t.double()], ids=["host", "shorter", "wider type"])
def test_saved_tensors_that_come_back_as_something_else_are_refused(back):
    x, w = torch.randn((8, 16), device="cuda"), torch.randn((16, 16), device="cuda", requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
        y, j = blocks.linear_rows(x, w, act="silu"), blocks.join_rows(x, x * w[0])
    for out in (y, j):
        with pytest.raises(RuntimeError, match="came back"):
            out.sum().backward()
