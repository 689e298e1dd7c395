"""Row blocks on the device, called in ways that are not a plain call on plain tensors."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from papr_amd import blocks
from test_hip_blocks import block, block_params, gen

pytestmark = pytest.mark.gpu


def test_a_tangent_on_an_operand_or_a_gradient_is_refused():
    """(It was lost: the result's tangent was None, which is zero.)"""
    p = {n: t.requires_grad_(True) for n, t in block_params(torch.float32, 64, 128, 1).items()}
    x = torch.randn((8, 64), generator=gen(1), device="cuda")
    y, h = block(p, x, None)
    with fwad.dual_level():
        for args in ((fwad.make_dual(x, x), p["w1"]), (x, fwad.make_dual(p["w1"].detach(), p["w1"].detach()))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                blocks.linear_rows(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            blocks.join_rows(x, fwad.make_dual(x, x))
        for out in (h, blocks.linear_rows(x, p["w1"])):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, [p["w1"]], fwad.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
        assert torch.autograd.grad(h, [p["w1"]], torch.ones_like(h), retain_graph=True)[0].abs().sum() > 0
    torch.autograd.grad([y, h], list(p.values()), [torch.ones_like(y), torch.ones_like(h)])
