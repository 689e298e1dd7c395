"""Products of float32 rows at the ends of the type: values are cut into three bfloat16 parts, and six of the nine products are summed (linear_kernels.h).

e = 2^-24.  The parts' sum is the value itself from 2^-109 up; below it is off by 2^-134 at most (half of bfloat16's smallest step).  The three products left out are at
most 2^-24 of a term; a sum of n terms makes 6 n + 16 additions."""
import math

import numpy as np
import pytest
import torch

from papr_amd import blocks
from test_hip_blocks import E32, close, gen, linear_data, unit

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)
BORDER = 2.0 ** 128 * (1 - 2.0 ** -9)                # from here on the nearest bfloat16 is infinite
ENDS = [MOST, -MOST, BORDER, -BORDER, float(np.nextafter(np.float32(BORDER), np.float32(0))), 3.4e38, 3.39e38, -3.395e38, 2.0 ** 127, 1.7e38]
SHAPES = [(1, 8, 8), (20, 40, 33), (70, 96, 48), (300, 128, 64), (301, 129, 67), (4096, 1024, 512)]


def ends(n, seed):
    return torch.tensor(ENDS, device="cuda")[torch.randint(0, len(ENDS), (n,), generator=gen(seed), device="cuda")]


def powers(shape, seed):
    """+-2^-8 .. 1"""
    g = gen(seed)
    return torch.exp2(-torch.randint(0, 9, shape, generator=g, device="cuda").float()) * (torch.randint(0, 2, shape, generator=g, device="cuda") * 2 - 1)


@pytest.mark.parametrize("M, N, K", SHAPES)
def test_finite_values_of_any_size_stay_finite(M, N, K):
    """One value a row (or column) of the other operand that is not zero, times powers of two: every product is one exact number."""
    x, w = torch.zeros((M, K), device="cuda"), powers((N, K), 2)
    k = torch.arange(M, device="cuda") % K
    x[torch.arange(M, device="cuda"), k] = ends(M, 1)
    y = blocks.linear_rows(x, w)
    assert torch.equal(y.double(), x.double() @ w.double().t()) and torch.isfinite(y).all()
    assert torch.equal(blocks.linear_rows(w, x), y.t())                       # (and the weight's side)
    # d_x = d_y W and d_w = d_y^T x, d_y with the large values
    x, w = powers((M, K), 3).requires_grad_(True), powers((N, K), 4).requires_grad_(True)
    n = min(M, N)
    d_y = torch.zeros((M, N), device="cuda")
    d_y[torch.arange(n, device="cuda"), torch.arange(n, device="cuda")] = ends(n, 5)
    d_x, d_w = torch.autograd.grad(blocks.linear_rows(x, w), [x, w], d_y)
    assert torch.equal(d_x.double(), d_y.double() @ w.detach().double()) and torch.equal(d_w.double(), d_y.double().t() @ x.detach().double())


def test_a_mask_s_lowest_value_beside_ordinary_ones():
    """-3.4e38 in one place of a row of ordinary values: that row's results are the definition's -- the large term, the others vanish beside it -- or infinite where it passes the
    type's end, never NaN."""
    x, w, _, _, _ = linear_data(200, 96, 64, torch.float32, seed=4)
    x[::3, 17] = -MOST
    w[::2, 17] = w[::2, 17] * 100
    y = blocks.linear_rows(x, w)
    ref = x.double() @ w.double().t()
    over = ref.abs() > MOST
    assert over.any() and torch.equal(torch.isinf(y), over) and torch.equal(y[over].double(), torch.sign(ref[over]) * math.inf)
    S = x.double().abs() @ w.double().abs().t()
    fine = ~over
    close(y[fine], ref[fine], unit(torch.float32) * ref[fine].abs() + (6 * 64 + 16) * E32 * S[fine])


@pytest.mark.parametrize("M", [4, 64])
def test_values_below_the_parts_range_are_off_by_2_to_the_134th(M):
    g = gen(7)
    x = torch.zeros((M, 32), device="cuda", dtype=torch.float64)
    x[:, 3] = (1 + torch.rand((M,), generator=g, device="cuda", dtype=torch.float64)) * torch.exp2(-torch.linspace(95, 140, M, device="cuda", dtype=torch.float64).round())
    x = x.float()
    w = torch.zeros((40, 32), device="cuda")
    w[:, 3] = 2.0 ** 110
    for y, ref in ((blocks.linear_rows(x, w), x.double() @ w.double().t()), (blocks.linear_rows(w, x), w.double() @ x.double().t())):
        lost = torch.where(ref.abs() < 2.0 ** (110 - 108), 2.0 ** (110 - 134), 0.0)
        close(y, ref, unit(torch.float32) * ref.abs() + lost)


@pytest.mark.parametrize("M, N", [(3, 5), (100, 70)])
def test_what_the_six_products_leave_out_is_2_to_the_24th_of_a_term(M, N):
    """1 + 2^-8 - 2^-17 cuts into 1, 2^-8 and -2^-17, the worst case: one term is off by 2^-24 of it, and n equal terms by n times that, whatever else is right."""
    v = 1 + 2.0 ** -8 - 2.0 ** -17
    for K in (1, 16, 256):
        x, w = torch.full((M, K), v, device="cuda"), torch.full((N, K), v, device="cuda")
        y, ref = blocks.linear_rows(x, w), torch.full((M, N), K * v * v, device="cuda", dtype=torch.float64)
        close(y, ref, (1 + 2.0 ** -9) * 2.0 ** -24 * ref + unit(torch.float32) * ref + (6 * K + 16) * E32 * ref * (0 if K == 1 else 1))


def as_defined(got, ref, S, n):
    """The infinities and NaN of the definition, and finite values within the bound of a sum of n terms."""
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)) and torch.equal(got[torch.isinf(ref)].double(), ref[torch.isinf(ref)])
    close(got[fine], ref[fine], unit(torch.float32) * ref[fine].abs() + (6 * n + 16) * E32 * S[fine])


@pytest.mark.parametrize("M, N, K", SHAPES)
def test_infinities_are_those_of_the_definition(M, N, K):
    """Infinite x, W and d_y here and there, some of them meeting (inf inf, inf - inf, inf 0): the sign of every infinite result, and NaN only where the definition has it."""
    x, w, _, _, d_y = linear_data(M, N, K, torch.float32, seed=6)
    x[0, 1], x[M // 2, K - 1], x[M - 1, 0] = math.inf, -math.inf, math.inf
    x[M - 1, K - 2] = -math.inf
    w[1] *= 1000
    w[3, 1], w[5, K - 1], w[2, 1] = 0.0, math.inf, -math.inf
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = blocks.linear_rows(x, w)
    x6, w6 = x.detach().double(), w.detach().double()
    fin = lambda t: t.abs().nan_to_num(0.0, posinf=0.0)
    as_defined(y, x6 @ w6.t(), fin(x6) @ fin(w6).t(), K)
    d_y[M // 3, N - 1], d_y[M - 1, 2] = math.inf, -math.inf
    d_x, d_w = torch.autograd.grad(y, leaves, d_y)
    g6 = d_y.double()
    as_defined(d_x, g6 @ w6, fin(g6) @ fin(w6), N)
    as_defined(d_w, g6.t() @ x6, fin(g6).t() @ fin(x6), M)
    assert torch.isinf(y).any() and torch.isnan(y).any()


@pytest.mark.parametrize("M, N, K", SHAPES)
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
def test_infinities_pass_the_epilogue_and_its_slopes(M, N, K, act):
    """+inf in rows of x, through the bias, the activation and the residual: y is infinite or act(-inf), with the other rows as they were, to the bit; kept rows hold NaN for it."""
    x, w, b, r, d_y = linear_data(M, N, K, torch.float32, seed=8)
    clean = blocks.linear_rows(x, w, b, r, act=act)
    x[M // 2, K // 2] = math.inf
    y = blocks.linear_rows(x, w, b, r, act=act)
    others = torch.arange(M, device="cuda") != M // 2
    assert torch.equal(y[others], clean[others])
    up = w[:, K // 2] > 0
    assert torch.isposinf(y[M // 2][up]).all()
    assert torch.equal(y[M // 2][~up], r[M // 2][~up]) if act == "relu" else torch.isnan(y[M // 2][~up]).all()          # (silu, gelu: -inf times zero)
    x.requires_grad_(True)
    w.requires_grad_(True)
    d_x, d_w = torch.autograd.grad(blocks.linear_rows(x, w, act="relu", keep="int8"), [x, w], d_y)
    assert torch.isfinite(d_x).all() and torch.isnan(d_w[:, K // 2]).all() and torch.isfinite(d_w[:, torch.arange(K, device="cuda") != K // 2]).all()
