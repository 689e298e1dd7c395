"""Rows whose elements pass 2^31 (and whose bytes pass 2^32): the far end is what it is alone."""
import pytest
import torch

from papr_amd import blocks
from test_hip_blocks import E32, close, gen, unit

pytestmark = pytest.mark.gpu

ROWS, WIDTH, TAIL = 270_001, 8192, 300              # 2.2e9 elements, 4.4 GB in float16
U = unit(torch.float16)


@pytest.fixture(scope="module")
def far():
    x = torch.empty((ROWS, WIDTH), device="cuda", dtype=torch.float16)
    for at in range(0, ROWS, 30_000):
        x[at:at + 30_000] = torch.randn(x[at:at + 30_000].shape, generator=gen(at), device="cuda")
    yield x
    del x
    torch.cuda.empty_cache()


def test_joins_and_their_gradients(far):
    norm = blocks.Norm("rmsnorm", torch.rand(WIDTH, generator=gen(1), device="cuda") + 0.5)
    gain = norm.gain.requires_grad_(True)
    gate = torch.randn((ROWS, 1), generator=gen(2), device="cuda").half()

    def run(rows):
        x, g = far[rows].detach().requires_grad_(True), gate[rows]
        y, h = blocks.join_rows(x, x, gate=g, post=norm, pre=norm)
        d_x, d_gain = torch.autograd.grad([y, h], [x, gain], [far[rows], far[rows]])
        return (y[-TAIL:].clone(), h[-TAIL:].clone(), d_x[-TAIL:].clone()), d_gain
    whole, d_gain = run(slice(None))
    alone, _ = run(slice(ROWS - TAIL, None))
    assert all(torch.equal(a, b) for a, b in zip(whole, alone)) and torch.isfinite(d_gain).all()


def test_packed_rows(far):
    p = blocks.pack_rows(far, "int8")
    back = p.rows()
    want = blocks.pack_rows(far[-TAIL:], "int8")
    assert torch.equal(p.codes[-TAIL:], want.codes) and torch.equal(p.exps[-TAIL:], want.exps) and torch.equal(back[-TAIL:], want.rows())


@pytest.mark.parametrize("keep", [None, "e4m3"])
def test_linear_layers_and_their_gradients(far, keep):
    """Forward, d_x and (from the kept rows too) the sum over all rows that d_w is: bounds as in test_hip_blocks_precision.py; y far out is silu(z) of 8192 terms."""
    w = (torch.randn((8, WIDTH), generator=gen(3), device="cuda") * WIDTH ** -0.5).half().requires_grad_(True)
    d_y = torch.randn((ROWS, 8), generator=gen(4), device="cuda").half()
    x = far.detach().requires_grad_(True)
    y = blocks.linear_rows(x, w, act="silu", keep=keep)
    d_x, d_w = torch.autograd.grad(y, [x, w], d_y)
    w6, t = w.detach().double(), slice(ROWS - TAIL, None)
    z = far[t].double() @ w6.t()
    S = far[t].double().abs() @ w6.abs().t()
    p = torch.sigmoid(z)
    err = (WIDTH + 16) * E32 * S
    close(y[t], z * p, U * (z * p).abs() + 1.13 * err + 16 * E32 * z.abs() + 2.0 ** -25, "y")
    d_z = d_y[t].double() * p * (1 + z * (1 - p))
    err_d = 0.8 * (U * z.abs() + err) * d_y[t].double().abs() + 16 * E32 * (d_z.abs() + d_y[t].double().abs()) + 2.0 ** -25
    ref = d_z @ w6
    close(d_x[t], ref, U * ref.abs() + err_d @ w6.abs() + 64 * E32 * (d_z.abs() @ w6.abs()) + 2.0 ** -25, "d_x")
    held = far if keep is None else blocks.pack_rows(far, keep).rows()
    ref, tol = torch.zeros((8, WIDTH), device="cuda", dtype=torch.float64), torch.zeros((8, WIDTH), device="cuda", dtype=torch.float64)
    for at in range(0, ROWS, 30_000):
        z = far[at:at + 30_000].double() @ w6.t()
        p, g, h = torch.sigmoid(z), d_y[at:at + 30_000].double(), held[at:at + 30_000].double()
        d_z = g * p * (1 + z * (1 - p))
        ref += d_z.t() @ h
        # (a row's z is off by n e S with S about n^(1/2) sqrt(2 / pi) here: the bound of the tail's rows holds for all)
        tol += (0.8 * (U * z.abs() + float(err.max())) * g.abs() + 16 * E32 * (d_z.abs() + g.abs()) + 2.0 ** -25 + (2 * ROWS + 16) * E32 * d_z.abs()).t() @ h.abs()
    close(d_w, ref, U * ref.abs() + tol, "d_w")
