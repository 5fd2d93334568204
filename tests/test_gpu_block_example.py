"""GPU: the example block (norms, selection, FP8 experts, 8-bit dense expert together) against a
plain 64-bit form of each of its steps."""
import importlib.util
from pathlib import Path

import pytest
import torch

import moe_swarm_b200 as M
from oracle import moe_ref as O
from tests import _ops_ref as R

pytestmark = pytest.mark.gpu


def load():
    path = Path(__file__).resolve().parents[1] / "examples" / "moe_block.py"
    spec = importlib.util.spec_from_file_location("moe_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def block():
    return load().MoEBlock(n_experts=4)


@pytest.mark.parametrize("T", [1, 37])
def test_forward_and_backward(block, T):
    ex = load()
    g = torch.Generator(device="cuda").manual_seed(T)
    y, residual = (torch.randn(T, M.H, generator=g, device="cuda").bfloat16() for _ in range(2))
    # experts 0..3 are the ones held here: make tokens choose them
    block.balance.zero_()
    block.balance[:4] = 10.0
    r2, x2, saved = block.forward(y, residual)
    x, logits, sel, out, r2s = saved
    assert r2s is r2
    r1, xr, rm, xm = R.block_norm(y, residual, pre_weight=block.norm_weight)
    R.close(x, xr, xm)
    idx, w, counts = R.select(logits, 8, bias=block.balance, n_group=8, topk_group=4, scale=2.5)
    assert torch.equal(sel.idx.cpu(), idx) and torch.equal(sel.counts.cpu(), counts)
    assert (idx[:, :4] == torch.arange(4)).all()
    R.close(sel.w, w, w.abs(), steps=32)
    # the routed experts, by the oracle, from the same quantised input and choice
    x8 = M.block_norm(None, M.block_norm(y, residual).residual, pre_weight=block.norm_weight,
                      x_dtype=torch.float8_e4m3fn)
    routed = M.run_routed(sel.idx, sel.w, x8.x, x8.x_scale, *block.experts, 0).cpu()
    ref = torch.zeros(T, M.H, dtype=torch.float64)
    a = x8.x.float().cpu().double() * x8.x_scale.cpu().double().t().repeat_interleave(128, dim=1)
    for e in range(4):
        w13, s13, w2, s2 = (t[e].float().cpu().double() for t in block.experts)
        w13 = w13 * s13.repeat_interleave(128, 0).repeat_interleave(128, 1)
        w2 = w2 * s2.repeat_interleave(128, 0).repeat_interleave(128, 1)
        up, gate = (a @ w13.t()).chunk(2, dim=1)
        ref += (torch.nn.functional.silu(gate) * up @ w2.t()) * w[:, e:e + 1]
    rep = O.parity_report(routed, ref.float(), atol=1e-2, rtol=2e-2)   # the layer's own bar
    assert rep["nan"] == 0 and rep["bad"] == 0, rep
    # the dense expert, from the codes that the call itself quantises to
    q, s = M.quantize_int8(x)
    h = (q.double().cpu() @ block.up.double().cpu().t()) * s.double().cpu()[:, None] * block.up_scale.double().cpu()
    hb = M.int8_linear(x, block.up, block.up_scale)
    R.close(hb, h, h.abs(), steps=8)
    q, s = M.quantize_int8(hb, swiglu=True)
    shared = (q.double().cpu() @ block.down.double().cpu().t()) * s.double().cpu()[:, None] * block.down_scale.double().cpu()
    R.close(out, routed.double() + R.d(M.int8_linear(hb, block.down, block.down_scale, swiglu=True)), 0.0)
    R.close(M.int8_linear(hb, block.down, block.down_scale, swiglu=True), shared, shared.abs(), steps=8)
    # the end of the block
    rr, xx, rm, xm = R.block_norm(out, M.block_norm(y, residual).residual, post_weight=block.out_weight, gate=block.out_gate,
                                  pre_weight=block.next_weight)
    R.close(r2, rr, rm)
    R.close(x2, xx, xm)
    # gradients of the parts that are trained
    dx2, dr2 = (torch.randn(T, M.H, generator=g, device="cuda").bfloat16() for _ in range(2))
    dw = torch.randn(T, 8, generator=g, device="cuda")
    norms, drouter = block.backward(saved, dx2, dr2, dw)
    refs = R.block_norm_backward(dx2, dr2, r2, out, post_weight=block.out_weight, gate=block.out_gate,
                                 pre_weight=block.next_weight)
    R.close(norms.post_weight, *refs["post_weight"], steps=3 * R.STEPS + 64)
    R.close(norms.pre_weight, *refs["pre_weight"], steps=3 * R.STEPS + 64)
    x64 = logits.double().cpu().requires_grad_()
    (R.select_weights(x64, sel.idx.cpu(), "sigmoid", True, 2.5) * dw.double().cpu()).sum().backward()
    want = x64.grad.t() @ x.double().cpu()
    # products of 32-bit values summed over T tokens
    bound = 256 * R.U32 * (x64.grad.abs().t() @ x.double().cpu().abs() + 2.5 * float(dw.abs().max()) * x.double().cpu().abs().sum(0))
    assert ((drouter.double().cpu() - want).abs() <= bound).all()
    before = block.balance.clone()
    block.rebalance(sel.counts)
    assert (block.balance[:4] < before[:4]).all() and (block.balance[100:] > before[100:]).sum() > 0
    assert ex.ROUTED_SCALE == 2.5


def test_command(capsys):
    load().main(["--tokens", "64", "--experts", "2"])
    assert "us a block" in capsys.readouterr().out
