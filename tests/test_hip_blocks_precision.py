"""Gradients of linear_rows with 16-bit rows against 64 bits, at every size: nothing between the roundings of z and of the result costs accuracy.

Tolerances as in test_hip_blocks.py (u half a step of the rows' type, e = 2^-24), but d_z = d_y act'(z) is held as the sum of two values of the rows' type: the first leaves
u |d_z| (float16 beyond its largest number: what is above it, at most 0.13 of it), the second u of that, so u^2 |d_z| (float16: 2^-25 where the second is subnormal; beyond
the largest number u 0.13 |d_z|).  Its products are sums of 2 n terms."""
import math

import pytest
import torch

from papr_amd import blocks
from test_hip_blocks import E32, act64, close, gen, ids, linear_data, tiny, unit

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
UZ = 2.0 ** -11                                      # z's rounding in both types (float16; 2^-25 where that is subnormal)


def check_gradients(x, w, b, r, d_y, act, keep=None):
    dt, (M, K), N = x.dtype, x.shape, w.shape[0]
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = blocks.linear_rows(x, w, b, r, act=act, keep=keep)
    got = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, leaves, d_y)))
    x6, w6, g6 = (t.detach().double() for t in (x, w, d_y))
    z = x6 @ w6.t() + (b.detach().double() if b is not None else 0)
    S = x6.abs() @ w6.abs().t() + (b.detach().double().abs() if b is not None else 0)
    d_z = g6 * act64(z, act)[1]
    u = unit(dt)
    err_f = (0.0 if act == "leakyrelu" else 0.8) * (UZ * z.abs() + 2.0 ** -25 + (K + 16) * E32 * S) * g6.abs() + 16 * E32 * (d_z.abs() + g6.abs())
    err_d = err_f + u * u * (d_z.abs() + err_f) + tiny(dt)
    m = lambda k: (2 * k + 16) * E32
    held = x6 if keep is None else blocks.pack_rows(x.detach(), keep).rows().double()
    ref = d_z @ w6
    close(got["x"], ref, u * ref.abs() + err_d @ w6.abs() + m(N) * (d_z.abs() @ w6.abs()) + tiny(dt), "d_x")
    ref = d_z.t() @ held
    close(got["w"], ref, u * ref.abs() + err_d.t() @ held.abs() + m(M) * (d_z.abs().t() @ held.abs()) + tiny(dt), "d_w")
    if b is not None:
        ref = d_z.sum(0)
        close(got["b"], ref, u * ref.abs() + err_f.sum(0) + (M + 16) * E32 * d_z.abs().sum(0) + tiny(dt), "d_b")


@pytest.mark.parametrize("dt", HALVES, ids=ids)
@pytest.mark.parametrize("M, N, K", [(1, 1, 1), (3, 7, 5), (37, 142, 256), (129, 127, 65), (257, 512, 512), (640, 136, 72), (4096, 512, 256), (4100, 1040, 264), (2500, 1001, 203),
                                     (30011, 72, 136), (33, 4096, 1024), (16400, 96, 192)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_of_16_bit_rows_lose_nothing_but_their_own_rounding(dt, M, N, K, act):
    check_gradients(*linear_data(M, N, K, dt, seed=M % 83), act=act)


@pytest.mark.parametrize("dt", HALVES, ids=ids)
@pytest.mark.parametrize("keep", ["e4m3", "int8"])
@pytest.mark.parametrize("M, N, K", [(77, 33, 31), (8192, 256, 256), (9000, 701, 117)])
def test_gradients_of_kept_16_bit_rows(dt, keep, M, N, K):
    check_gradients(*linear_data(M, N, K, dt, seed=M % 79), act="silu", keep=keep)


@pytest.mark.parametrize("dt", HALVES, ids=ids)
def test_gradients_behind_leakyrelu(dt):
    """z is never zero (whole numbers and a half), so its rounding moves no slope."""
    check_gradients(*linear_data(4096, 512, 256, dt, seed=3, whole=True), act="leakyrelu")


@pytest.mark.parametrize("dt", HALVES, ids=ids)
@pytest.mark.parametrize("keep", [None, "e4m3"])
@pytest.mark.parametrize("M, N, K", [(400, 512, 512), (4096, 512, 256), (4096, 519, 261)])
def test_the_error_of_gradients_does_not_grow_with_the_batch(dt, keep, M, N, K):
    """Beside the final rounding (rms e_out) only z's is left: through the slope's derivative at most 0.8 u |z| rms, under half of e_out: below 1.15 e_out at every size."""
    x, w, b, r, d_y = linear_data(M, N, K, dt, seed=12)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(blocks.linear_rows(x, w, b, r, act="silu", keep=keep), leaves, d_y)
    x6, w6 = (t.detach().double() for t in (x, w))
    d_z = d_y.double() * act64(x6 @ w6.t() + b.double(), "silu")[1]
    held = x6 if keep is None else blocks.pack_rows(x.detach(), keep).rows().double()
    for g, ref in zip(got, (d_z @ w6, d_z.t() @ held)):
        assert (g.double() - ref).norm() <= 1.15 * (ref.to(dt).double() - ref).norm()


@pytest.mark.parametrize("act, z", [("gelu", 1.4), ("silu", 2.4)])
@pytest.mark.parametrize("M, N, K", [(64, 64, 16), (32, 256, 7), (16384, 512, 64)])
def test_d_z_beyond_float16_reaches_gradients_that_are_not(act, z, M, N, K):
    """d_y = 65,000 and a slope of 1.13 / 1.10: d_z is beyond 65,504, d_x (N d_z w = d_z / 16) and one column of d_w (M d_z x = d_z / 4) are not.  Column 0 of d_w is: infinite.
    d_z's two parts leave 0.13 u of it; z's rounding moves it by 0.8 u |z|."""
    dt = torch.float16
    x, w = torch.zeros((M, K), device="cuda", dtype=dt), torch.zeros((N, K), device="cuda", dtype=dt)
    x[:, 0], w[:, 0], x[:, 1] = z * 16 * N, 1.0 / (16 * N), 0.25 / M
    d_y = torch.full((M, N), 65000.0, device="cuda", dtype=dt)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    d_x, d_w = torch.autograd.grad(blocks.linear_rows(x, w, act=act), leaves, d_y)
    x6, w6 = (t.detach().double() for t in (x, w))
    v = x6 @ w6.t()
    d_z = d_y.double() * act64(v, act)[1]
    assert (d_z > 65504).all()
    rel = unit(dt) * (1 + 0.13 + 0.8 * float(v.amax())) + (2 * max(M, N) + 32) * E32
    close(d_x, d_z @ w6, rel * (d_z @ w6).abs(), "d_x")
    ref = d_z.t() @ x6
    close(d_w[:, 1:], ref[:, 1:], rel * ref[:, 1:].abs(), "d_w")
    assert torch.isposinf(d_w[:, 0]).all()


@pytest.mark.parametrize("dt", HALVES, ids=ids)
@pytest.mark.parametrize("M, N, K", [(40, 24, 16), (4096, 512, 256)])
def test_gradients_that_are_not_finite_stay_in_their_row_and_column(dt, M, N, K):
    for bad in (math.inf, -math.inf, math.nan):
        x, w, b, r, d_y = linear_data(M, N, K, dt, seed=2)
        leaves = [t.requires_grad_(True) for t in (x, w)]
        clean = torch.autograd.grad(blocks.linear_rows(x, w, b, act="silu"), leaves, d_y)
        d_y[7, 5] = bad
        d_x, d_w = torch.autograd.grad(blocks.linear_rows(x, w, b, act="silu"), leaves, d_y)
        at = torch.arange(M, device="cuda") != 7
        assert torch.equal(d_x[at], clean[0][at]) and not torch.isfinite(d_x[7]).any()
        at = torch.arange(N, device="cuda") != 5
        assert torch.equal(d_w[at], clean[1][at]) and not torch.isfinite(d_w[5]).any()
        if math.isinf(bad):      # (the slope is positive or negative, x and w are not zero: the sign of the definition's infinity)
            v = x.detach().double() @ w.detach().double().t() + b.double()
            slope = act64(v, "silu")[1][7, 5]
            assert torch.equal(d_x[7].double(), (bad * slope) * w.detach()[5].double()) and torch.equal(d_w[5].double(), (bad * slope) * x.detach()[7].double())


@pytest.mark.parametrize("act", ["silu", "gelu", "leakyrelu", "relu"])
@pytest.mark.parametrize("M, N, K", [(1, 64, 64), (20, 40, 33), (50, 37, 16), (300, 128, 64), (4096, 512, 256), (3001, 519, 261)])
def test_an_activation_s_argument_beyond_float16_has_the_slope_of_its_limit(act, M, N, K):
    """A third of the columns of z are at 76,800, a third at -76,800 (float16 ends at 65,504): y is 76,800 -> infinite or zero, the slopes are 1 and 0 (leakyrelu: 1 and 0.2), and
    the gradients finite.  The other third: silu's and gelu's slopes move by 0.8 u |z|."""
    dt, u = torch.float16, unit(torch.float16)
    x, w, b, _, d_y = linear_data(M, N, K, dt, seed=M % 71, res=False)
    x[:, 0] = 256.0
    w[:, 0] = torch.tensor([300.0, -300.0, 0.0], device="cuda").repeat((N + 2) // 3)[:N]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = blocks.linear_rows(x, w, b, act=act)
    d_x, d_w, d_b = torch.autograd.grad(y, leaves, d_y)
    x6, w6, g6 = (t.detach().double() for t in (x, w, d_y))
    z = x6 @ w6.t() + b.detach().double()
    v, slope = act64(z, act)
    S = x6.abs() @ w6.abs().t() + b.detach().double().abs()
    assert torch.isposinf(y[:, ::3]).all() and not torch.isnan(y).any()
    near = z.abs() < 100                         # (elsewhere the slope is constant to 2^-50)
    keeps = (z.abs() > (K + 16) * E32 * S + u * z.abs() + 2.0 ** -24) if act in ("relu", "leakyrelu") else torch.ones_like(near)      # (where z's rounding moves no step of the slope)
    d_z = g6 * slope
    err_f = torch.where(near, (0.8 if act in ("silu", "gelu") else 0.0) * (u * z.abs() + (K + 16) * E32 * S), 0.0) * g6.abs() + 16 * E32 * (d_z.abs() + g6.abs()) + (~keeps) * g6.abs()
    err_d = err_f + u * u * d_z.abs() + tiny(dt)
    ref = d_z @ w6
    close(d_x, ref, u * ref.abs() + err_d @ w6.abs() + (2 * N + 16) * E32 * (d_z.abs() @ w6.abs()) + tiny(dt), "d_x")
    ref = d_z.t() @ x6
    close(d_w, ref, u * ref.abs() + err_d.t() @ x6.abs() + (2 * M + 16) * E32 * (d_z.abs().t() @ x6.abs()) + tiny(dt), "d_w")
    ref = d_z.sum(0)
    close(d_b, ref, u * ref.abs() + err_f.sum(0) + (M + 16) * E32 * d_z.abs().sum(0) + tiny(dt), "d_b")


def test_an_activation_s_argument_that_is_nan_stays_one():
    x, w, b, _, d_y = linear_data(40, 24, 16, torch.float16, seed=1, res=False)
    x[3, 2] = math.nan
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = blocks.linear_rows(x, w, b, act="silu")
    d_x, _, d_b = torch.autograd.grad(y, leaves, d_y)
    at = torch.arange(40, device="cuda") != 3
    assert torch.isnan(y[3]).all() and torch.isnan(d_x[3]).all() and torch.isnan(d_b).all() and torch.isfinite(d_x[at]).all() and torch.isfinite(y[at]).all()


@pytest.mark.parametrize("dt", HALVES, ids=ids)
@pytest.mark.parametrize("M", [20, 700])
def test_gelu_s_tail_is_as_exact_as_its_middle(dt, M):
    """z exact (one term, a weight of one), no bias, no residual: y is gelu(z) rounded once.  Beside that: the erfc form's 6.4e-7 and its float32 steps (48 e together), and the
    exponent z^2 / 2, five roundings, each e of it."""
    x = torch.linspace(-9.0 if dt == torch.float16 else -13.0, 6.0, M, device="cuda", dtype=torch.float64).to(dt)[:, None]
    w = torch.ones((24, 1), device="cuda", dtype=dt)
    x.requires_grad_(True)
    y = blocks.linear_rows(x, w, act="gelu")
    d_x, = torch.autograd.grad(y[:, :1], x, torch.ones_like(x))
    z = x.detach().double()
    cdf, pdf = 0.5 * torch.erfc(-z / math.sqrt(2)), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    rel = (2.5 * z * z + 48) * E32
    ref = z * cdf
    close(y, ref.expand(M, 24), (unit(dt) * ref.abs() + rel * ref.abs() + tiny(dt)).expand(M, 24), "y")
    ref = cdf + z * pdf
    close(d_x, ref, unit(dt) * ref.abs() + rel * (cdf + z.abs() * pdf) + tiny(dt), "d_x")


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("M, N, K", [(400, 512, 512), (4096, 512, 256), (1000, 519, 261)])
def test_gradients_of_bfloat16_rows_are_as_good_as_their_rounding(act, M, N, K):
    """z's rounding (float16: 2^-11) moves d_z by 0.8 2^-11 |z| |d_y| at most, rms 0.8 1.4 2^-11, against the final rounding of gradients whose d_z has rms 0.6 |d_y|, 2^-8: a quarter of
    it at most, together 1.03 (in bfloat16 it was 1.05)."""
    x, w, b, r, d_y = linear_data(M, N, K, torch.bfloat16, seed=12)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    got = torch.autograd.grad(blocks.linear_rows(x, w, b, r, act=act), leaves, d_y)
    x6, w6 = (t.detach().double() for t in (x, w))
    d_z = d_y.double() * act64(x6 @ w6.t() + b.double(), act)[1]
    for g, ref in zip(got, (d_z @ w6, d_z.t() @ x6)):
        assert (g.double() - ref).norm() <= 1.03 * (ref.to(torch.bfloat16).double() - ref).norm()


@pytest.mark.parametrize("act", ["silu", "gelu", "leakyrelu", "relu"])
@pytest.mark.parametrize("M", [31, 300])
def test_an_activation_s_argument_of_bfloat16_rows_far_out_and_close_to_zero(act, M):
    """z = 1e-30 .. 1e30 of both signs (float16 spans 2^-25 .. 65,504): the slopes of the definition.  One term, a weight of one: z is exact but for its keeping."""
    e = torch.linspace(-30, 30, 61, device="cuda", dtype=torch.float64)
    z = torch.cat([10.0 ** e, -(10.0 ** e), torch.zeros(1, device="cuda", dtype=torch.float64)]).bfloat16()
    x = z[torch.linspace(0, z.numel() - 1, M, device="cuda").round().long()][:, None].contiguous().requires_grad_(True)
    w = torch.ones((16, 1), device="cuda", dtype=torch.bfloat16)
    y = blocks.linear_rows(x, w, act=act)
    d_x, = torch.autograd.grad(y[:, :1], x, torch.ones_like(x))
    v = x.detach().double()
    if act == "silu":
        ref = torch.sigmoid(v) * (1 + torch.where(v.abs() < 700, v * torch.sigmoid(-v), 0.0))
    elif act == "gelu":
        ref = 0.5 * torch.erfc(-v / math.sqrt(2)) + torch.where(v.abs() < 40, v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi), 0.0)
    else:
        ref = torch.where(v > 0, 1.0, 0.2 if act == "leakyrelu" else 0.0).double()
    moved = 0.8 * torch.where(v.abs() < 100, UZ * v.abs() + 2.0 ** -25, 0.0) if act in ("silu", "gelu") else 0.0
    close(d_x, ref, unit(torch.bfloat16) * ref.abs() + moved + 64 * E32)
