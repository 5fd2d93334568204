"""GPU: the choice of experts and its gradient against the 64-bit forms."""
import pytest
import torch

import moe_swarm_b200 as M
from moe_swarm_b200 import workload as W
from tests import _ops_ref as R

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def logits_of(T, E, dtype=F32, seed=0, masked=0.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E + pad, generator=g) + 0.5 * torch.randn(1, E + pad, generator=g)
    if masked:
        x = x.masked_fill(torch.rand(T, E + pad, generator=g) < masked, float("-inf"))
    return x.to(dtype).cuda()[:, :E]


def check(x, K, **kw):
    o = M.select_experts(x, K, counts=True, **kw)
    idx, w, counts = R.select(x, K, **kw)
    assert torch.equal(o.idx.cpu(), idx)
    assert torch.equal(o.counts.cpu(), counts)
    # exponential and quotient (2 units each), the sum of the chosen, quotient, scale
    nan = torch.isnan(w)
    assert torch.equal(torch.isnan(o.w.cpu()), nan)
    R.close(torch.nan_to_num(o.w), torch.nan_to_num(w), torch.nan_to_num(w).abs(), steps=32)
    return o


@pytest.mark.parametrize("T", [1, 7, 65])
@pytest.mark.parametrize("E,K,G,TG", [(1, 1, 1, 1), (2, 1, 1, 1), (8, 2, 4, 2), (31, 5, 1, 1), (32, 32, 1, 1),
                                      (60, 4, 1, 1), (64, 6, 8, 3), (96, 6, 3, 2), (256, 8, 8, 4), (257, 3, 1, 1),
                                      (384, 8, 1, 1), (512, 10, 32, 5), (512, 32, 2, 1)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_selection(T, E, K, G, TG, score, dtype):
    x = logits_of(T, E, dtype, seed=E + T)
    bias = (torch.randn(E, generator=torch.Generator().manual_seed(1)) * (0.1 if score == "sigmoid" else 0.1 / E)).cuda()
    for b in (None, bias, bias.to(BF)):
        for gsc in ("top2", "max"):
            if gsc == "top2" and G > 1 and E // G < 2:
                continue
            check(x, K, score=score, bias=b, n_group=G, topk_group=TG, group_score=gsc, renormalize=gsc == "max",
                  scale=2.5)
            if G == 1:
                break


def test_equals_the_layers_routing():
    """The layer's own configuration gives the layer's own ids, and its weights to 32-bit rounding."""
    T = 300
    x = W.make_activations(T, 5, skew=0.5)
    idx, w, _ = M.select_experts(x["routing_logits"].cuda(), 8, bias=x["routing_bias"].cuda(), n_group=8, topk_group=4,
                                 scale=2.5)
    from oracle import moe_ref as O
    ref_idx, dense = O.route(x["routing_logits"], x["routing_bias"], 2.5)   # dense weights [T, 256]
    ref_idx = ref_idx.long().sort(dim=1).values
    assert torch.equal(idx.cpu().long(), ref_idx)
    ref_w = dense.gather(1, ref_idx)
    R.close(w, ref_w, ref_w.abs(), steps=16)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_go_to_the_lowest_id(score):
    x = torch.zeros(5, 100, device="cuda")
    x[1, 50:] = 1.0
    x[2, ::2] = -3.0
    x[3] = 60.0           # sigmoid saturates: every score is 1
    o = check(x, 6, score=score)
    assert o.idx[0].tolist() == list(range(6)) and o.idx[1].tolist() == list(range(50, 56))
    o = check(x[:, :96], 4, score=score, n_group=8, topk_group=2)
    assert o.idx[0].tolist() == [0, 1, 2, 3]


@pytest.mark.parametrize("dtype", [F32, BF, FP])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("G,TG", [(1, 1), (4, 2)])
def test_masked_experts(dtype, score, G, TG):
    x = logits_of(12, 64, dtype, seed=3, masked=0.5)
    x[0] = float("-inf")                          # nothing to choose from
    x[1] = torch.finfo(dtype).min
    x[2, 3:] = float("-inf")                      # fewer than top_k
    x[3, 1:] = torch.finfo(dtype).min
    x[4, 16:] = float("-inf")
    o = check(x, 6, score=score, n_group=G, topk_group=TG)
    assert (o.idx[:2] == -1).all() and (o.w[:2] == 0).all()
    first = 0 if float(x[3, 0]) > torch.finfo(dtype).min else -1
    assert o.idx[3].tolist() == [first, -1, -1, -1, -1, -1]
    b = torch.zeros(64, device="cuda")
    b[7] = float("-inf")                          # switched off for all tokens
    o = check(x, 6, score=score, n_group=G, topk_group=TG, bias=b)
    assert o.counts[7] == 0


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_nan_and_infinity(score):
    x = logits_of(6, 48, seed=4)
    x[1, 9] = float("nan")
    x[2, 5] = float("inf")
    x[3, 5] = 1e30
    x[4, 5] = -1e30
    o = M.select_experts(x, 4, score=score, counts=True)
    assert (o.idx[1] == -1).all() and torch.isnan(o.w[1]).all()
    if score == "softmax":     # inf - inf
        assert (o.idx[2] == -1).all() and torch.isnan(o.w[2]).all()
    else:
        assert 5 in o.idx[2].tolist()
    keep = [0, 3, 4, 5]
    idx, w, _ = R.select(x[keep], 4, score=score)
    assert torch.equal(o.idx[keep].cpu(), idx)
    R.close(o.w[keep], w, w.abs(), steps=32)
    d = M.select_experts_backward(torch.ones(6, 4, device="cuda"), x, o.idx, score=score)
    assert torch.isnan(d[1]).all() and torch.isfinite(d[keep]).all()


def test_close_scores_are_told_apart():
    """Scores one unit apart keep their order; logits whose 32-bit scores are equal are a tie."""
    g = torch.Generator().manual_seed(6)
    x = (0.3 + 1e-6 * torch.randn(400, 64, generator=g)).cuda()
    check(x, 8)
    check(x, 8, score="softmax")
    check(x, 8, n_group=8, topk_group=3)
    check(x, 8, n_group=8, topk_group=3, bias=(1e-6 * torch.randn(64, generator=g)).cuda())
    x = (18.0 + torch.randn(100, 64, generator=g)).cuda()   # sigmoid near 1
    check(x, 8)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_biases_of_any_size(score):
    """Biases from the tiny to the overflowing, and -inf: chosen by the defined 32-bit sums."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(40, 64, generator=g).cuda()
    for size in (1e-30, 1e-7, 1.0, 1e4, 1e29, 1e32, 2.5e38):
        b = (torch.randn(64, generator=g) * 0.3 + torch.randint(-1, 2, (64,), generator=g)).clamp(-1.3, 1.3) * size
        b[5] = float("-inf")
        for kw in (dict(), dict(n_group=8, topk_group=3), dict(n_group=8, topk_group=3, group_score="max"),
                   dict(n_group=16, topk_group=5)):
            check(x, 6, score=score, bias=b.cuda(), **kw)


@pytest.mark.parametrize("T", [1, 255, 4096])
def test_row_pitch_and_sizes(T):
    x = logits_of(T, 33, seed=7, pad=7)
    if T < 1000:
        check(x, 3)
    o = M.select_experts(x, 3, counts=True)
    c = M.select_experts(x.contiguous(), 3, counts=True)
    assert torch.equal(o.idx, c.idx) and torch.equal(o.w, c.w) and torch.equal(o.counts, c.counts)
    assert int(o.counts.sum()) == 3 * T


def test_empty():
    o = M.select_experts(torch.empty(0, 16, device="cuda"), 2, counts=True)
    assert o.idx.shape == (0, 2) and (o.counts == 0).all()
    d = M.select_experts_backward(torch.empty(0, 2, device="cuda"), torch.empty(0, 16, device="cuda"), o.idx)
    assert d.shape == (0, 16)


@pytest.mark.parametrize("T,E,K", [(1, 2, 1), (3, 8, 2), (65, 33, 4), (17, 256, 8), (5, 512, 32), (9, 100, 7)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_gradient(T, E, K, score, renorm, dtype):
    x = logits_of(T, E, dtype, seed=E, masked=0.2 if E > 8 else 0.0, pad=3)
    idx = M.select_experts(x, K, score=score).idx
    dw = torch.randn(T, K, generator=torch.Generator().manual_seed(2)).cuda()
    got = M.select_experts_backward(dw, x, idx, score=score, renormalize=renorm, scale=2.5)
    x64 = x.double().cpu().requires_grad_()
    c = R.select_weights(x64, idx.cpu(), score, renorm, 2.5)
    (c * dw.double().cpu()).sum().backward()
    ref = torch.nan_to_num(x64.grad)
    # terms: 2.5 |dw| s / S and, renormalised, the mean of all of them, each times at most 1;
    # renormalised weights divide by S >= the largest chosen score
    p = torch.nan_to_num(torch.sigmoid(x64) if score == "sigmoid" else torch.softmax(x64, 1)).detach()
    s = p.gather(1, idx.cpu().clamp(min=0).long()) * (idx.cpu() >= 0)
    S = s.sum(1, keepdim=True).clamp(min=1e-20) if renorm else torch.ones(T, 1, dtype=torch.float64)
    m = 2.5 * dw.double().cpu().abs()
    per = m + (m * s).sum(1, keepdim=True) / S if renorm else m
    terms = per.amax(dim=1, keepdim=True) / S
    mag = p * (terms + (terms * s).sum(1, keepdim=True))
    R.close(got, ref, mag, steps=64)


def test_gradient_against_differences():
    x = logits_of(4, 24, seed=9)
    for score in ("sigmoid", "softmax"):
        for renorm in (False, True):
            idx = M.select_experts(x, 5, score=score).idx
            dw = torch.randn(4, 5, generator=torch.Generator().manual_seed(2)).cuda()
            got = M.select_experts_backward(dw, x, idx, score=score, renormalize=renorm, scale=1.5).double().cpu()
            v = torch.randn(4, 24, generator=torch.Generator().manual_seed(3), dtype=torch.float64)
            h = 1e-4
            f = [(R.select_weights(x.double().cpu() + s * h * v, idx.cpu(), score, renorm, 1.5) * dw.double().cpu()).sum()
                 for s in (1, -1)]
            num = float(f[0] - f[1]) / (2 * h)
            tol = 256 * R.U32 * float(dw.abs().sum()) + 1e-6 * float((got * v).norm())
            assert abs(float((got * v).sum()) - num) <= tol


def test_refusals():
    x = torch.zeros(4, 16, device="cuda")
    idx = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    dw = torch.zeros(4, 2, device="cuda")
    bad = [
        lambda: M.select_experts(x, 0), lambda: M.select_experts(x, 17),
        lambda: M.select_experts(torch.zeros(2, 513, device="cuda"), 1),
        lambda: M.select_experts(torch.zeros(2, 64, device="cuda"), 33),
        lambda: M.select_experts(x, 2, n_group=3), lambda: M.select_experts(x, 2, n_group=4, topk_group=5),
        lambda: M.select_experts(x, 5, n_group=4, topk_group=1),
        lambda: M.select_experts(x, 2, n_group=16, topk_group=4),         # top2 of groups of one
        lambda: M.select_experts(x, 2, score="relu"), lambda: M.select_experts(x, 2, group_score="mean"),
        lambda: M.select_experts(x, 2, bias=torch.zeros(15, device="cuda")),
        lambda: M.select_experts(x.double(), 2), lambda: M.select_experts(x.cpu(), 2),
        lambda: M.select_experts(x.t(), 2),
        lambda: M.select_experts_backward(dw[:, :1], x, idx),
        lambda: M.select_experts_backward(dw, x, idx.long()),
        lambda: M.select_experts_backward(dw[:3], x, idx[:3]),
    ]
    for f in bad:
        with pytest.raises(M.MoEArgumentError):
            f()
