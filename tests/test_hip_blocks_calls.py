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


def test_traces_and_transforms_are_refused_and_modes_that_watch_are_not():
    """(A trace recorded the output's allocation alone: the traced function returned memory as it was.)"""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    p = block_params(torch.bfloat16, 64, 128, 1)
    x = torch.randn((8, 64), generator=gen(1), device="cuda").bfloat16()
    want = block(p, x, None)
    calls = [lambda t: blocks.linear_rows(t, p["w1"]), lambda t: blocks.norm_rows(t, blocks.Norm("rmsnorm")), lambda t: blocks.join_rows(t, t), lambda t: blocks.pack_rows(t).codes,
             lambda t: blocks.PackedRows(blocks.pack_rows(x).codes, t, "e4m3", (8, 64), torch.bfloat16).rows()]
    for i, call in enumerate(calls):
        t = x if i < 4 else blocks.pack_rows(x).exps
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            torch.jit.trace(call, t)
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            make_fx(call)(t)
        with pytest.raises(NotImplementedError, match="plain tensors"):
            torch.func.vmap(call)(t[None].expand(3, *t.shape))
    with pytest.raises(NotImplementedError, match="plain tensors"):
        torch.func.grad(lambda t: blocks.linear_rows(t, p["w1"]).float().sum())(x)
    out = blocks.linear_rows(x.clone().requires_grad_(True), p["w1"])
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        make_fx(lambda g: torch.autograd.grad(out, [out.grad_fn.next_functions[0][0].variable], g, retain_graph=True))(torch.ones_like(out))

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    with Watch():
        assert all(torch.equal(a, b) for a, b in zip(block(p, x, None), want))


@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16], ids=lambda t: str(t)[6:])
def test_operands_that_torch_negates_lazily(dt):
    """Imaginary parts of a conjugate are views whose memory holds the values with the other sign: as rows, parameters, codes' source and incoming gradients."""
    def lazy(t):
        if dt != torch.float32:
            return torch._neg_view(-t)
        v = torch.complex(t, -t).conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v
    g = gen(3)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dt)
    x, w, b, q, f, gate, gain, shift, c = r(40, 48), r(64, 48), r(64), r(40, 64), r(40, 48), r(40, 1), r(48), r(48), r(40, 64)
    names = [x, w, b, q, f, gate, gain, shift]

    def run(flip):
        leaves = [t.clone().requires_grad_(True) for t in names]
        X, Wt, Bi, Q, F, G, A, S = [torch._neg_view(-t) for t in leaves] if flip else leaves
        assert X.is_neg() == flip and A.is_neg() == flip
        norm = blocks.Norm("rmsnorm", A, S)
        y = blocks.linear_rows(X, Wt, Bi, Q, act="silu", keep="int8")
        j, h = blocks.join_rows(X, F, gate=G, scale=A, post=norm, pre=norm)
        cots = [c, x, f]
        cots = [lazy(t) for t in cots] if flip else cots
        grads = torch.autograd.grad([y, j, h], leaves, cots)
        return [y, j, h, blocks.norm_rows(X, norm), blocks.pack_rows(X).rows()] + list(grads)
    with torch.no_grad():
        assert torch.equal(blocks.linear_rows(lazy(x), w), blocks.linear_rows(x, w))
    for got, want in zip(run(True), run(False)):
        assert torch.equal(got, want)


def test_debug_sync_names_every_library_call_and_waits(capfd, monkeypatch):
    from papr_amd import hip
    p = {n: t.requires_grad_(True) for n, t in block_params(torch.float16, 64, 128, 1).items()}
    x = torch.randn((8, 64), generator=gen(1), device="cuda").half()
    block(p, x, "int8")
    assert capfd.readouterr().err == ""
    waits = []
    wait = torch.cuda.synchronize
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: (waits.append(1), wait()))
    monkeypatch.setattr(hip, "DEBUG_SYNC", True)
    y, h = block(p, x, "int8")
    blocks.pack_rows(x).rows()
    forward = capfd.readouterr().err.splitlines()
    torch.autograd.grad([y, h], list(p.values()), [torch.ones_like(y), torch.ones_like(h)])
    backward = capfd.readouterr().err.splitlines()
    call = lambda *names: ["papr call: papr_" + n for n in names]
    assert forward == call("join_fwd", "linear_fwd", "rows8_pack", "linear_fwd", "rows8_pack", "linear_fwd", "join_fwd", "rows8_pack", "rows8_unpack")
    assert sorted(backward) == call("join_bwd", "join_bwd", "linear_bwd", "linear_bwd", "linear_bwd") and len(waits) == 14


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=lambda t: str(t)[6:])
def test_linear_products_appear_in_the_profile(dt):
    from papr_amd import hip
    x = torch.randn((300, 48), generator=gen(1), device="cuda").to(dt).requires_grad_(True)
    w = torch.randn((64, 48), generator=gen(2), device="cuda").to(dt).requires_grad_(True)
    hip.profile_collect()
    hip.profile_enable(True)
    try:
        y = blocks.linear_rows(x, w, act="silu")
        torch.autograd.grad(y, [x, w], torch.ones_like(y))
        blocks.linear_rows(x[:3].detach(), w.detach())
    finally:
        hip.profile_enable(False)
    records = hip.profile_collect()
    flops = 2 * 300 * 64 * 48
    assert [r[:4] + r[5:] for r in records] == [(13, 300, 64, 48, 0, flops), (14, 300, 64, 48, 0, flops), (15, 300, 64, 48, 0, flops), (13, 3, 64, 48, 0, flops // 100)]
    assert all(0 < r[4] < 100 for r in records)


def test_inference_mode_and_its_tensors():
    """Inside inference mode, and its tensors outside of it, where no gradient is asked for."""
    p = block_params(torch.float16, 64, 128, 1)
    x = torch.randn((8, 64), generator=gen(1), device="cuda").half()
    want = block(p, x, "e4m3")
    with torch.inference_mode():
        inner = x.clone()
        got = block(p, inner, "e4m3")
        assert not got[0].requires_grad and inner.is_inference()
    with torch.no_grad():
        again = block(p, inner, "e4m3")
    for out in (got, again):
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert torch.equal(blocks.pack_rows(inner).rows(), blocks.pack_rows(x).rows())


def test_one_tensor_in_several_places():
    """The rows as residual and gate, the weight as rows: gradients add up as autograd adds them."""
    g = gen(2)
    x = torch.randn((40, 64), generator=g, device="cuda", dtype=torch.float32).requires_grad_(True)
    w = (torch.randn((64, 64), generator=g, device="cuda") / 8).requires_grad_(True)

    def run(f, sep):
        xs = [x.detach().clone().requires_grad_(True) for _ in range(4)] if sep else [x] * 4
        ws = [w.detach().clone().requires_grad_(True) for _ in range(2)] if sep else [w] * 2
        y = blocks.linear_rows(xs[0], ws[0], residual=xs[1], act="silu", keep="int8")
        z = blocks.linear_rows(ws[1], ws[0])
        j = blocks.join_rows(xs[2], y, gate=xs[3], scale=z[0].clone())
        leaves = xs + ws if sep else [x, w]
        got = torch.autograd.grad(j, leaves, torch.ones_like(j))
        return j, (got if not sep else (got[0] + got[1] + got[2] + got[3], got[4] + got[5]))
    a, b = run(None, False), run(None, True)
    assert torch.equal(a[0], b[0])
    for s, t in zip(a[1], b[1]):
        assert (s - t).abs().max() <= 8 * 2.0 ** -24 * t.abs().max() * 4          # (four float32 additions in another order)
