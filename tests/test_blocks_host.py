"""Row blocks (papr_amd/blocks.py, papr_linear_* / papr_join_* / papr_rows8_* of include/papr_hip.h) without a GPU: what is refused, and that the refusal comes
before a device is touched."""
import ctypes as C

import pytest
import torch

from papr_amd import blocks, hip

X = torch.zeros(4, 8)
W = torch.zeros(6, 8)


def rows_norm(n=8, dtype=torch.float32, kind="rmsnorm"):
    return blocks.Norm(kind, torch.ones(n, dtype=dtype), torch.zeros(n, dtype=dtype))


@pytest.mark.parametrize("call, word", [
    (lambda: blocks.linear_rows(X, torch.zeros(6, 7)), "weight has shape"),
    (lambda: blocks.linear_rows(X, torch.zeros(0, 8)), "weight has shape"),
    (lambda: blocks.linear_rows(X, torch.zeros(8)), "weight has shape"),
    (lambda: blocks.linear_rows(torch.zeros(1, 1), torch.zeros((1 << 20) + 1, 1)), "at most"),
    (lambda: blocks.linear_rows(X, W.half()), "weight is torch.float16"),
    (lambda: blocks.linear_rows(X.double(), W.double()), "float64"),
    (lambda: blocks.linear_rows(X, W, torch.zeros(8)), "bias has shape"),
    (lambda: blocks.linear_rows(X, W, torch.zeros(6).bfloat16()), "bias is torch.bfloat16"),
    (lambda: blocks.linear_rows(X, W, None, torch.zeros(6)), "residual has shape"),
    (lambda: blocks.linear_rows(X, W, None, torch.zeros(1, 6)), "residual has shape"),
    (lambda: blocks.linear_rows(X, W, act="tanh"), "unknown activation"),
    (lambda: blocks.linear_rows(X, W, keep="e5m2"), "unknown format"),
    (lambda: blocks.linear_rows(torch.zeros(()), W), "at least one column"),
    (lambda: blocks.linear_rows(torch.zeros(4, 0), torch.zeros(6, 0)), "at least one column"),
    (lambda: blocks.linear_rows([1.0], W), "not a tensor"),
    (lambda: blocks.pack_rows(X, "fp8"), "unknown format"),
    (lambda: blocks.pack_rows(X.to(torch.int32)), "int32"),
    (lambda: blocks.norm_rows(X, ("rmsnorm", None, None)), "not a Norm"),
    (lambda: blocks.norm_rows(X, blocks.Norm("batchnorm")), "unknown norm"),
    (lambda: blocks.norm_rows(X[:, :1], blocks.Norm("layernorm")), "two columns"),
    (lambda: blocks.norm_rows(X, rows_norm(7)), "gain has shape"),
    (lambda: blocks.norm_rows(X, blocks.Norm("layernorm", torch.ones(8), torch.zeros(8).half())), "shift torch.float16"),
    (lambda: blocks.norm_rows(torch.zeros(2, hip.JOIN_MAX_WIDTH + 1), blocks.Norm("rmsnorm")), "at most"),
    (lambda: blocks.join_rows(X, torch.zeros(4, 7)), "f is"),
    (lambda: blocks.join_rows(X, X.half()), "f is"),
    (lambda: blocks.join_rows(X, X, gate=torch.zeros(4)), "gate is"),
    (lambda: blocks.join_rows(X, X, gate=torch.zeros(1, 8)), "gate is"),
    (lambda: blocks.join_rows(X, X, gate=X, gate_act="tanh"), "unknown gate activation"),
    (lambda: blocks.join_rows(X, X, scale=torch.zeros(())), "scale has shape"),
    (lambda: blocks.join_rows(X, X, scale=torch.zeros(4, 8)), "scale has shape"),
    (lambda: blocks.join_rows(X, X, post="rmsnorm"), "not a Norm"),
])
def test_arguments_that_do_not_fit_are_refused_by_name(call, word):
    with pytest.raises(ValueError, match=word):
        call()


@pytest.mark.parametrize("call", [
    lambda: blocks.linear_rows(X, W),
    lambda: blocks.linear_rows(X, W.clone().requires_grad_(True), keep="e4m3"),
    lambda: blocks.pack_rows(X),
    lambda: blocks.norm_rows(X, rows_norm()),
    lambda: blocks.join_rows(X, X, post=rows_norm(), pre=rows_norm()),
])
def test_there_is_no_cpu_form(call):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call()


def refused(code, word):
    assert code != 0
    assert word in hip.lib().papr_last_error().decode()


def test_c_entry_points_refuse_before_touching_a_device():
    L = hip.lib()
    p = C.c_void_p(4096)                                 # (never read: the checks come first)
    D = hip.LinearDesc
    refused(L.papr_linear_fwd(None, p, 8, p, 8, None, None, 0, p, None, None, None), "no descriptor")
    refused(L.papr_linear_fwd(D(3, 0, 0, 0, 4, 6, 8), p, 8, p, 8, None, None, 0, p, None, None, None), "row type")
    refused(L.papr_linear_fwd(D(0, 5, 0, 0, 4, 6, 8), p, 8, p, 8, None, None, 0, p, None, None, None), "activation")
    refused(L.papr_linear_fwd(D(0, 0, 0, 0, -1, 6, 8), p, 8, p, 8, None, None, 0, p, None, None, None), "M -1")
    refused(L.papr_linear_fwd(D(0, 0, 0, 0, 4, 6, 0), p, 8, p, 8, None, None, 0, p, None, None, None), "K 0")
    refused(L.papr_linear_fwd(D(0, 0, 0, 0, 4, 6, 8), None, 8, p, 8, None, None, 0, p, None, None, None), "missing")
    refused(L.papr_linear_fwd(D(0, 0, 0, 0, 4, 6, 8), p, 7, p, 8, None, None, 0, p, None, None, None), "row strides")
    refused(L.papr_linear_fwd(D(0, 0, 0, 0, 4, 6, 8), p, (1 << 22) + 1, p, 8, None, None, 0, p, None, None, None), "row strides")
    assert L.papr_linear_fwd(D(0, 0, 0, 0, 0, 6, 8), None, 8, p, 8, None, None, 0, None, None, None, None) == 0        # no rows: nothing to do
    bwd = lambda d, dy=p, z=p, x=p, e=None, w=p, dx=p, dw=p, db=p, ws=p: L.papr_linear_bwd(d, dy, 6, z, x, 8, e, w, 8, dx, dw, db, ws, None)
    refused(bwd(D(0, 0, 0, 0, 0, 6, 8)), "no rows")
    refused(bwd(D(0, 0, 3, 0, 4, 6, 8)), "format")
    refused(bwd(D(0, 1, 0, 0, 4, 6, 8), z=None), "missing")
    refused(bwd(D(0, 0, 0, 0, 4, 6, 8), ws=None), "missing")
    refused(bwd(D(0, 0, 0, 0, 4, 6, 8), w=None), "weight")
    refused(bwd(D(0, 0, 0, 0, 4, 6, 8), x=None), "rows")
    refused(bwd(D(0, 0, 1, 0, 4, 6, 8)), "rows")         # kept rows without their exponents
    refused(bwd(D(0, 0, 1, 0, 4, 6, 8), e=p), "32 codes")    # ... whose rows are not whole blocks
    refused(bwd(D(0, 0, 0, 0, 4, 6, 8), ws=C.c_void_p(4100)), "16 bytes")
    refused(bwd(D(0, 0, 0, 0, 4, 7, 8)), "row strides")      # d_y's rows overlap
    assert L.papr_linear_bwd_workspace_bytes(D(0, 0, 0, 0, 0, 6, 8)) == 0
    refused(L.papr_rows8_pack(0, 0, p, 8, 4, 8, p, p, None), "format")
    refused(L.papr_rows8_pack(4, 1, p, 8, 4, 8, p, p, None), "type")
    refused(L.papr_rows8_pack(0, 1, p, 8, 4, 0, p, p, None), "width")
    refused(L.papr_rows8_pack(0, 1, p, 8, 4, 8, p, None, None), "missing")
    refused(L.papr_rows8_pack(0, 1, p, 8, 4, 8, C.c_void_p(4100), p, None), "8 bytes")
    refused(L.papr_rows8_unpack(0, 1, None, p, 4, 8, p, None), "missing")
    assert L.papr_rows8_pack(0, 1, None, 8, 0, 8, None, None, None) == 0
    N = hip.BlockNorm
    none, rms, ln = N(0, 0, 0.0, 0, None, None), N(2, 0, 1e-6, 0, None, None), N(1, 0, 1e-6, 0, None, None)
    J = lambda rows=4, width=8, type=0, x=4096, f=4096, gate=None, form=0, act=0, post=none, pre=rms: hip.JoinDesc(rows, width, type, x, width, f, width, gate, width, form, act,
                                                                                                                None, 0, 1.0, post, pre)
    refused(L.papr_join_fwd(None, p, p, None, None), "no descriptor")
    refused(L.papr_join_fwd(J(type=7), p, p, None, None), "row type")
    refused(L.papr_join_fwd(J(width=8193), p, p, None, None), "width 8193")
    refused(L.papr_join_fwd(J(width=1, pre=ln), p, p, None, None), "two columns")
    refused(L.papr_join_fwd(J(form=1), p, p, None, None), "disagree")
    refused(L.papr_join_fwd(J(gate=4096), p, p, None, None), "disagree")
    refused(L.papr_join_fwd(J(gate=4096, form=3), p, p, None, None), "gate form")
    refused(L.papr_join_fwd(J(gate=4096, form=2, act=3), p, p, None, None), "gate activation")
    refused(L.papr_join_fwd(J(f=None), p, p, None, None), "without the block's output")
    refused(L.papr_join_fwd(J(f=None, gate=4096, form=2), None, p, None, None), "without the block's output")
    refused(L.papr_join_fwd(J(x=None), p, p, None, None), "x is missing")
    refused(L.papr_join_fwd(J(), None, None, None, None), "neither")
    refused(L.papr_join_fwd(J(pre=N(3, 0, 0.0, 0, None, None)), p, p, None, None), "norm")
    refused(L.papr_join_bwd(J(), None, p, p, p, p, None, None, None, None), "stats")
    refused(L.papr_join_bwd(J(), p, None, None, p, p, None, None, None, None), "neither")
    refused(L.papr_join_bwd(J(f=None), p, None, p, p, p, None, None, None, None), "without f")
    refused(L.papr_join_bwd(J(), p, p, p, p, p, None, hip.JoinGrads(4096, None, None, None, None), None, None), "workspace")


def test_workspaces_grow_with_the_call():
    L = hip.lib()
    ws = lambda act, M: L.papr_linear_bwd_workspace_bytes(hip.LinearDesc(2, act, 0, 0, M, 512, 256))
    assert ws(3, 1000) >= ws(0, 1000) + 1000 * 512 * 2       # an activation: d_z
    assert ws(0, 512000) > ws(0, 1000)
    assert L.papr_join_bwd_workspace_bytes(0, 256) == 0
    assert L.papr_join_bwd_workspace_bytes(1, 256) == 5 * 256 * 4


def packed(rows=(4, 40), codes=(4, 64), exps=(4, 2), fmt="e4m3", dtype=torch.float32, byte=torch.uint8):
    return blocks.PackedRows(torch.zeros(codes, dtype=byte), torch.zeros(exps, dtype=byte), fmt, rows, dtype)


@pytest.mark.parametrize("p, word", [
    (packed(codes=(4, 40)), "codes of rows"),
    (packed(codes=(3, 64)), "codes of rows"),
    (packed(exps=(4, 1)), "exps of rows"),
    (packed(byte=torch.int8), "codes of rows"),
    (packed(rows=(4, 65)), "codes of rows"),
    (packed(rows=(2, 4, 40)), "codes of rows"),
    (packed(rows=()), "at least one column"),
    (packed(fmt="fp8"), "unknown format"),
    (packed(dtype=torch.float64), "float64"),
])
def test_packed_rows_that_do_not_fit_their_shape_are_refused(p, word):
    with pytest.raises(ValueError, match=word):
        p.rows()


def test_packed_rows_held_on_the_host_are_refused():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        packed().rows()


def test_a_forward_workspace_starts_on_16_bytes():
    L, p = hip.lib(), C.c_void_p(4096)
    d = hip.LinearDesc(2, 0, 0, 0, 8192, 1000, 701)       # (its rows are copied into whole vectors)
    assert L.papr_linear_fwd_workspace_bytes(d) == (8192 + 1000) * 704 * 2
    for ws in (None, C.c_void_p(4104)):
        refused(L.papr_linear_fwd(d, p, 701, p, 701, None, None, 0, p, None, ws, None), "16 bytes")
