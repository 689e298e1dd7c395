"""Row blocks called in ways that are not a plain call on plain tensors: refused before a device is touched, by name (papr_amd/csrc/blocks_glue.cpp)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from papr_amd import blocks

X, W, B = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
OPERANDS = {
    "linear x": lambda t: blocks.linear_rows(t(X), W, B, X), "linear weight": lambda t: blocks.linear_rows(X, t(W), B, X), "linear bias": lambda t: blocks.linear_rows(X, W, t(B), X),
    "linear residual": lambda t: blocks.linear_rows(X, W, B, t(X)), "norm x": lambda t: blocks.norm_rows(t(X), blocks.Norm("rmsnorm")),
    "norm gain": lambda t: blocks.norm_rows(X, blocks.Norm("rmsnorm", t(B))), "norm shift": lambda t: blocks.norm_rows(X, blocks.Norm("rmsnorm", B, t(B))),
    "join x": lambda t: blocks.join_rows(t(X), X), "join f": lambda t: blocks.join_rows(X, t(X)), "join gate": lambda t: blocks.join_rows(X, X, t(X)),
    "join row gate": lambda t: blocks.join_rows(X, X, t(X[:, :1])), "join scale": lambda t: blocks.join_rows(X, X, scale=t(B)),
    "join post gain": lambda t: blocks.join_rows(X, X, post=blocks.Norm("rmsnorm", t(B))), "join post shift": lambda t: blocks.join_rows(X, X, post=blocks.Norm("rmsnorm", B, t(B))),
    "join pre gain": lambda t: blocks.join_rows(X, X, pre=blocks.Norm("rmsnorm", t(B))), "join pre shift": lambda t: blocks.join_rows(X, X, pre=blocks.Norm("rmsnorm", B, t(B))),
}
each = pytest.mark.parametrize("call", list(OPERANDS.values()), ids=[n.replace(" ", "_") for n in OPERANDS])


@each
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(call, grad):
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(lambda t: fwad.make_dual(t, torch.ones_like(t)))
        with pytest.raises(RuntimeError, match="no CPU fallback"):                # (the level alone is no reason)
            call(lambda t: t)
