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


def test_c_entry_points_refuse_strides_and_workspaces_that_do_not_fit():
    import ctypes as C
    from papr_amd import hip
    L, p = hip.lib(), C.c_void_p(4096)                   # (never read: the checks come first)
    refused = lambda code, word: (code != 0 and word in L.papr_last_error().decode()) or pytest.fail("%d %r" % (code, L.papr_last_error()))
    none, rms = hip.BlockNorm(0, 0, 0.0, 0, None, None), hip.BlockNorm(2, 0, 1e-6, 0, None, None)
    J = lambda ldx=8, ldf=8, ldg=8, form=2, rows=4, f=4096, gate=4096: hip.JoinDesc(rows, 8, 0, 4096, ldx, f, ldf, gate, ldg, form, 1, None, 0, 1.0, none, rms)
    grads = hip.JoinGrads(4096, None, None, None, None)
    for bad in (J(ldx=7), J(ldf=7), J(ldg=7), J(ldx=-8), J(ldg=0, form=1), J(ldx=0, f=None, gate=None, form=0)):
        refused(L.papr_join_fwd(bad, None, p, None, None), "row strides")
        refused(L.papr_join_bwd(bad, p, None, p, p, None, None, None, None, None), "row strides")
    refused(L.papr_join_fwd(J(), None, p, C.c_void_p(4098), None), "4 bytes")
    refused(L.papr_join_bwd(J(), C.c_void_p(4098), p, p, p, p, None, None, None, None), "4 bytes")
    refused(L.papr_join_bwd(J(), p, p, p, p, p, None, grads, C.c_void_p(4104), None), "16 bytes")
    refused(L.papr_rows8_pack(0, 1, p, 7, 4, 8, p, p, None), "row stride")
    refused(L.papr_rows8_pack(0, 1, p, -8, 4, 8, p, p, None), "row stride")
    refused(L.papr_linear_fwd(hip.LinearDesc(0, 0, 0, 0, 4, 6, 8), p, 8, p, 8, None, p, 5, p, None, None, None), "residual")


def test_packed_rows_too_wide_for_32_bit_columns_are_refused():
    """(The number of blocks of a row of 2^31 - 1 columns overflowed: nothing was packed, and no error.)"""
    import ctypes as C
    from papr_amd import hip
    L, p = hip.lib(), C.c_void_p(4096)
    for width in (hip.ROWS8_MAX_WIDTH + 1, 2 ** 31 - 40, 2 ** 31 - 1):
        for code in (L.papr_rows8_pack(1, 1, p, width, 1, width, p, p, None), L.papr_rows8_unpack(1, 1, p, p, 1, width, p, None)):
            assert code == 1 and "width %d" % width in L.papr_last_error().decode()
        with pytest.raises(ValueError, match="at most"):
            blocks.pack_rows(torch.zeros(1).expand(1, width))
        with pytest.raises(ValueError, match="at most"):
            blocks.PackedRows(PACKED.codes, PACKED.exps, "e4m3", (1, width), torch.float16).rows()
