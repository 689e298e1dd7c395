"""Row blocks called in ways that are not a plain call on plain tensors: refused before a device is touched, by name (papr_amd/csrc/blocks_glue.cpp)."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from papr_amd import blocks

X, W, B, G = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8), torch.zeros(4, 1)
OPERANDS = {
    "linear x": lambda t: blocks.linear_rows(t(X), W, B, X), "linear weight": lambda t: blocks.linear_rows(X, t(W), B, X), "linear bias": lambda t: blocks.linear_rows(X, W, t(B), X),
    "linear residual": lambda t: blocks.linear_rows(X, W, B, t(X)), "norm x": lambda t: blocks.norm_rows(t(X), blocks.Norm("rmsnorm")),
    "norm gain": lambda t: blocks.norm_rows(X, blocks.Norm("rmsnorm", t(B))), "norm shift": lambda t: blocks.norm_rows(X, blocks.Norm("rmsnorm", B, t(B))),
    "join x": lambda t: blocks.join_rows(t(X), X), "join f": lambda t: blocks.join_rows(X, t(X)), "join gate": lambda t: blocks.join_rows(X, X, t(X)),
    "join row gate": lambda t: blocks.join_rows(X, X, t(G)), "join scale": lambda t: blocks.join_rows(X, X, scale=t(B)),
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


PACKED = blocks.PackedRows(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 1), dtype=torch.uint8), "e4m3", (4, 8), torch.float32)


def unpacked(t):
    return blocks.PackedRows(t(PACKED.codes), PACKED.exps, "e4m3", (4, 8), torch.float32).rows()


TRACED = dict(OPERANDS, **{"pack x": lambda t: blocks.pack_rows(t(X)).codes, "unpack codes": unpacked})
each_traced = pytest.mark.parametrize("call", list(TRACED.values()), ids=[n.replace(" ", "_") for n in TRACED])


@each_traced
def test_traces_are_refused(call):
    """(They recorded the output's allocation and nothing that fills it.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        torch.jit.trace(lambda x: call(lambda t: x.to(t.dtype).expand_as(t)), torch.zeros(()))
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            make_fx(lambda x: call(lambda t: x.to(t.dtype).expand_as(t)), tracing_mode=mode)(torch.zeros(()))
    with pytest.raises(RuntimeError, match="no CPU fallback"):                    # (once it is over, nothing is left of it)
        call(lambda t: t)


@each_traced
def test_tensors_that_stand_for_others_are_refused(call):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.vmap(lambda x: call(lambda t: x.to(t.dtype).expand_as(t)))(torch.zeros(3))
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.vjp(lambda x: call(lambda t: x.to(t.dtype).expand_as(t)), torch.zeros(()))
    mode = FakeTensorMode()
    with pytest.raises(NotImplementedError, match="plain tensors"):
        call(lambda t: mode.from_tensor(t))
    with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
        call(lambda t: t.to("meta"))
