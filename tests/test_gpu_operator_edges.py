"""GPU: where the operators around the layer end: rows that do not fill a CTA, infinite factors, biases that
cancel, rows that overlap, scores next to 0 and 1."""
import pytest
import torch

import moe_swarm_b200 as M
from tests import _ops_ref as R

pytestmark = pytest.mark.gpu
BF, FP, F32, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn
BEHIND = 9   # rows behind a result, more than a CTA holds of any length


def randn(seed, *shape, std=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


# rows of one to four warps on odd boundaries: by their length, their pitch or their base
@pytest.mark.parametrize("T,H,pad,base", [(5, 500, 0, 0), (3, 1001, 0, 0), (3, 1300, 0, 0), (5, 2047, 0, 0), (1, 500, 0, 0),
                                          (5, 512, 1, 0), (3, 1024, 3, 0), (2, 2048, 0, 1), (7, 400, 0, 3), (9, 99, 0, 0),
                                          (3, 250, 0, 0), (5, 300, 0, 0), (3, 3001, 0, 0)])
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("x_dtype", [BF, F32, E4M3])
@pytest.mark.parametrize("post", [False, True])
def test_nothing_is_written_behind_the_last_row(T, H, pad, base, y_dtype, r_dtype, x_dtype, post):
    def rows(seed, dtype):
        flat = randn(seed, base + T * (H + pad), dtype=dtype)
        return flat[base:].view(T, H + pad)[:, :H]

    def buffer(dtype):
        flat = torch.full((base + (T + BEHIND) * (H + pad),), 77, dtype=torch.uint8, device="cuda").to(dtype)
        return flat, flat[base:].view(T + BEHIND, H + pad)[:T, :H]

    y, r = rows(1, y_dtype), rows(2, r_dtype)
    w = (1 + randn(3, H, std=0.2)).to(BF)
    kw = dict(post_weight=w if post else None, gate=torch.rand(T, 1, device="cuda").to(BF), pre_weight=w)
    all_r, ro = buffer(r_dtype)
    all_x, x = buffer(x_dtype)
    o = M.block_norm(y, r, residual_out=ro, out=x, x_dtype=x_dtype, **kw)
    ref_r, ref_x, rm, xm = R.block_norm(y, r, **kw)
    R.close(ro, ref_r, rm)
    if x_dtype != E4M3:
        R.close(x, ref_x, xm)
    else:
        assert torch.isfinite(o.x_scale).all()
        s = o.x_scale.t().double().repeat_interleave(128, dim=1)[:, :H].cpu()
        tol = (ref_x.abs() * 2.0 ** -4).maximum(s * 2.0 ** -10) * 1.001 + 2 * R.STEPS * R.U32 * (xm + ref_x.abs())
        assert ((x.double().cpu() * s - ref_x).abs() <= tol).all()
    for flat, view in ((all_r, ro), (all_x, x)):
        untouched = torch.ones_like(flat, dtype=torch.bool)
        untouched[base:].view(T + BEHIND, H + pad)[:T, :H] = False
        assert (flat[untouched].float() == torch.tensor(77.0).to(flat.dtype).float().item()).all()


def test_a_slice_of_a_live_stream():
    """r' written over the first rows of a stream leaves the rows behind them."""
    stream = randn(1, 40, 1000, dtype=BF)[:, :500]
    before = stream.clone()
    M.block_norm(randn(2, 5, 500, dtype=BF), stream[:5], residual_out=stream[:5])
    assert torch.equal(stream[5:], before[5:]) and not torch.equal(stream[:5], before[:5])


def choice(x, K, score, bias, G, TG, group_score="top2"):
    """ids of select_experts by the definition, many rows at a time: 32-bit scores whose exponential (softmax:
    quotient) is rounded once, their 32-bit sums, stable sorts."""
    x = x.double()
    T, E = x.shape
    s = 1.0 / (1.0 + torch.exp(-x).float()) if score == "sigmoid" else torch.softmax(x, dim=1).float()
    sel = s if bias is None else s + bias
    if G > 1:
        per = sel.view(T, G, -1)
        first = per.sort(dim=2, descending=True).values
        gs = first[..., 0] + first[..., 1] if group_score == "top2" else first[..., 0]
        rank = gs.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        sel = per.masked_fill((rank >= TG).unsqueeze(2), float("-inf")).reshape(T, E)
    return sel.sort(dim=1, descending=True, stable=True).indices[:, :K].sort(dim=1).values.int()


# groups of lanes, of lanes and registers, and of a length that is scored through shared memory
@pytest.mark.parametrize("E,G,TG", [(64, 8, 3), (256, 8, 4), (60, 4, 2), (512, 16, 5)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("size", [0.3, 16.0, 64.0, 1e3, 1e4])
def test_groups_whose_biases_cancel(E, G, TG, score, size):
    """A favoured expert beside disfavoured ones: a group's score is the small sum of two large values."""
    T = 1 << 17
    x = randn(E + int(size), T, E)
    favoured = torch.full((E,), -size, device="cuda")
    favoured[::E // G] = size
    spread = randn(5, E, std=size)
    for bias in (favoured, spread):
        for group_score in ("top2", "max"):
            o = M.select_experts(x, 6, score=score, bias=bias, n_group=G, topk_group=TG, group_score=group_score)
            assert torch.equal(o.idx, choice(x, 6, score, bias, G, TG, group_score))


def overlapping(seed, T, H, step, dtype=F32):
    """[T, H] whose rows begin `step` elements apart, step < H (0: one row, seen T times)."""
    return randn(seed, (T - 1) * step + H, dtype=dtype).as_strided((T, H), (step, 1))


@pytest.mark.parametrize("T,H,step", [(3, 8, 1), (3, 8, 0), (5, 512, 8), (700, 1024, 8), (6, 300, 7), (900, 96, 2)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_overlap(T, H, step, dtype):
    y, r, dx, dr = (overlapping(i, T, H, step, dtype) for i in range(4))
    w = (1 + randn(9, H, std=0.2)).to(dtype)
    o = M.block_norm(y, r, pre_weight=w)
    ref = R.block_norm(y, r, pre_weight=w)
    R.close(o.residual, ref[0], ref[2])
    R.close(o.x, ref[1], ref[3])
    b = M.block_norm_backward(dx, dr, r, y, pre_weight=w, post_weight=w)
    ref = R.block_norm_backward(dx, dr, r, y, pre_weight=w, post_weight=w)
    R.close(b.residual, *ref["residual"])
    R.close(b.y, *ref["y"], steps=3 * R.STEPS)
    for t in (o.residual, o.x, b.residual, b.y):
        assert t.is_contiguous()
    if H > 512:
        return
    logits = overlapping(5, T, H, step, dtype)
    s = M.select_experts(logits, 4)
    assert torch.equal(s.idx, M.select_experts(logits.contiguous(), 4).idx)
    dw = randn(6, T, 4)
    d = M.select_experts_backward(dw, logits, s.idx)
    assert d.is_contiguous() and torch.equal(d, M.select_experts_backward(dw, logits.contiguous(), s.idx))


def test_results_may_not_overlap():
    y = randn(1, 3, 8)
    with pytest.raises(M.MoEArgumentError):
        M.block_norm(y, y, residual_out=overlapping(2, 3, 8, 1))


@pytest.mark.parametrize("T,H", [(301, 128), (2500, 8), (333, 301), (333, 1001), (149, 99), (1301, 256), (700, 5001)])
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
def test_gradients_without_an_epsilon(T, H, gate):
    """Rows that a CTA has room for but the batch has not leave the sums over rows alone, also at eps = 0."""
    y, r, dx, dr = (randn(i, T, H, dtype=BF) for i in range(4))
    w, wp = ((1 + randn(i, H, std=0.2)).to(BF) for i in (8, 9))
    shape = {None: None, "channel": (1, H), "token": (T, 1), "full": (T, H)}[gate]
    kw = dict(pre_weight=w, post_weight=wp, gate=None if shape is None else randn(7, *shape, dtype=BF), eps=0.0)
    b = M.block_norm_backward(dx, dr, r, y, **kw)
    ref = R.block_norm_backward(dx, dr, r, y, **kw)
    steps = 3 * R.STEPS + T // 148 + 64
    R.close(b.pre_weight, *ref["pre_weight"], steps=steps)
    R.close(b.post_weight, *ref["post_weight"], steps=steps)
    if gate == "channel":
        R.close(b.gate, *(t.sum(0, keepdim=True) for t in ref["gate"]), steps=steps)


@pytest.mark.parametrize("renorm", [False, True])
def test_sigmoid_gradient_next_to_0_and_1(renorm):
    """s (1 - s) keeps its bits where s rounds to 1, and where exp(-x) overflows."""
    T, E, K = 40, 16, 4
    x = torch.linspace(-25, 25, T, device="cuda")[:, None] + 0.1 * randn(1, T, E)
    x[0], x[1] = -100.0, 100.0
    idx = torch.arange(K, dtype=torch.int32, device="cuda").expand(T, K).contiguous()
    dw = randn(2, T, K)
    got = M.select_experts_backward(dw, x, idx, renormalize=renorm, scale=2.5)
    p = torch.sigmoid(x[:, :K].double())
    slope = p * torch.sigmoid(-x[:, :K].double())
    d = 2.5 * dw.double()
    mag = d.abs()
    if renorm:
        S = p.sum(1, keepdim=True) + 1e-20
        d, mag = (d - (d * p).sum(1, keepdim=True) / S) / S, (mag + (mag * p).sum(1, keepdim=True) / S) / S
    # exponential (2), sum, quotient, product, slope; renormalised, two sums of 5 and two quotients besides;
    # below 2^-126 numbers have an absolute spacing
    err = (got[:, :K].double() - d * slope).abs()
    assert (err <= 32 * R.U32 * mag * slope + 2.0 ** -148).all()
    assert (got[:, K:] == 0).all() and (got[5:30, 0] != 0).all()


@pytest.mark.parametrize("E,K", [(60, 4), (256, 8), (512, 10), (33, 1)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("spread", [1.0, 9.0])
def test_weights_are_rounded_scores(E, K, score, renorm, spread):
    """Weights within the roundings of their definition, also of experts that a bias chose far below the
    largest logit: score 3 units (exponential, sum, quotient; a softmax's quotient alone 1), their sum one more
    each of five times and 1e-20, quotient, scale."""
    T = 20000
    x = randn(E, T, E, std=spread).clamp(-8 * spread, 8 * spread).to(BF).float()
    if spread > 1:
        x[:, ::5] -= 20.0
    bias = None if spread == 1 else torch.zeros(E, device="cuda").index_fill(0, torch.arange(0, E, 5, device="cuda"), 2.0)
    o = M.select_experts(x, K, score=score, bias=bias, renormalize=renorm, scale=2.5)
    assert torch.equal(o.idx, choice(x, K, score, bias, 1, 1))
    s = (torch.sigmoid(x.double()) if score == "sigmoid" else torch.softmax(x.double(), dim=1)).gather(1, o.idx.long())
    w = 2.5 * (s / (s.sum(1, keepdim=True) + 1e-20) if renorm else s)
    units = (3 if score == "sigmoid" else 1) * (2 if renorm else 1) + (7 if renorm else 0) + 1
    assert ((o.w.double() - w).abs() <= units * R.U32 * w + 2.0 ** -148).all()


@pytest.mark.parametrize("T,H", [(700, 7168), (3, 7168), (900, 512), (301, 1001), (40, 300), (5, 5001), (9, 12000)])
@pytest.mark.parametrize("r_dtype", [BF, F32])
def test_e4m3_codes_are_those_of_the_quotients(T, H, r_dtype):
    """Scales and codes equal the 32-bit quotients of the same norm in fp32, to the last bit."""
    y, r, w = randn(1, T, H, dtype=BF), randn(2, T, H, std=1.5, dtype=r_dtype), (1 + randn(3, H, std=0.2)).to(BF)
    kw = dict(pre_weight=w, post_weight=w)
    x = M.block_norm(y, r, x_dtype=F32, **kw).x.cpu()
    o = M.block_norm(y, r, x_dtype=E4M3, **kw)
    nb = -(-H // 128)
    blocks = torch.nn.functional.pad(x, (0, nb * 128 - H)).view(T, nb, 128)
    scale = blocks.abs().amax(dim=2).clamp(min=1e-12) / torch.tensor(448.0)
    assert torch.equal(o.x_scale.cpu(), scale.t())
    codes = (blocks / scale[:, :, None]).view(T, nb * 128)[:, :H].to(E4M3)
    assert torch.equal(o.x.cpu().view(torch.uint8), codes.view(torch.uint8))


def test_e4m3_blocks_with_infinities():
    """A block whose norm has an infinity (an infinite weight) has its finite elements 0 and the infinity NaN."""
    r, w = randn(2, 5, 600), torch.ones(600, device="cuda")
    w[300] = float("inf")
    for cols in (600, 599):
        o = M.block_norm(None, r[:, :cols], pre_weight=w[:cols], x_dtype=E4M3)
        v = o.x.float()
        assert torch.isinf(o.x_scale[2]).all() and torch.isfinite(o.x_scale[[0, 1, 3, 4]]).all()
        assert torch.isnan(v[:, 300]).all() and (v[:, 256:300] == 0).all() and (v[:, 301:384] == 0).all()
        assert torch.isfinite(v[:, :256]).all() and torch.isfinite(v[:, 384:]).all()


@pytest.mark.parametrize("renorm", [False, True])
def test_softmax_gradient_far_below_the_first(renorm):
    """Gradients of logits up to 85 below the row's largest keep the bits of their scores.  (Differences of
    16-bit values are exact.)  Units: score 12 (exponential 2, sum 8, quotient, product), their products' sum 7 more,
    slope 14 more; renormalised, the sum of the chosen, two quotients and the sum once more."""
    T, E, K = 500, 64, 5
    x = (randn(1, T, E) * 20).clamp(-40, 40).to(BF).float()
    x[:, 0] = 45.0
    idx = torch.tensor([0, 7, 20, 33, 60], dtype=torch.int32, device="cuda").expand(T, K).contiguous()
    if renorm:
        idx = (idx + 1) % E
        idx = idx.sort(dim=1).values.contiguous()
    dw = randn(2, T, K)
    got = M.select_experts_backward(dw, x, idx, score="softmax", renormalize=renorm, scale=2.5).double()
    x64 = x.double().requires_grad_()
    (R.select_weights(x64, idx, "softmax", renorm, 2.5) * dw.double()).sum().backward()
    p = torch.softmax(x.double(), dim=1)
    s, d = p.gather(1, idx.long()), 2.5 * dw.double().abs()
    if renorm:
        S = s.sum(1, keepdim=True) + 1e-20
        d = (d + (d * s).sum(1, keepdim=True) / S) / S
    own = torch.zeros_like(p).scatter_(1, idx.long(), d)
    mag = p * (own + (d * s).sum(1, keepdim=True))
    assert ((got - x64.grad).abs() <= (110 if renorm else 33) * R.U32 * mag + 2.0 ** -140).all()


@pytest.mark.parametrize("T,H", [(600, 1024), (3000, 1024), (700, 7168), (2400, 7168), (600, 8192), (2100, 8192)])
@pytest.mark.parametrize("x_dtype", [None, BF, F32, E4M3])
@pytest.mark.parametrize("block", [False, True])
def test_a_32_bit_stream_on_both_sides_of_the_ring(T, H, x_dtype, block):
    y, r, w = randn(1, T, H, dtype=BF), randn(2, T, H), (1 + randn(3, H, std=0.2)).to(BF)
    if not block and x_dtype is None:
        return
    o = M.block_norm(y if block else None, r, pre_weight=None if x_dtype is None else w, x_dtype=x_dtype)
    ref_r, ref_x, rm, xm = R.block_norm(y if block else None, r, pre_weight=w)
    R.close(o.residual, ref_r, rm)
    if x_dtype == E4M3:
        s = o.x_scale.t().double().repeat_interleave(128, dim=1)[:, :H].cpu()
        tol = (ref_x.abs() * 2.0 ** -4).maximum(s * 2.0 ** -10) * 1.001 + 2 * R.STEPS * R.U32 * (xm + ref_x.abs())
        assert ((o.x.double().cpu() * s - ref_x).abs() <= tol).all()
    elif x_dtype is not None:
        R.close(o.x, ref_x, xm)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_of_an_expert_that_is_off(score, renorm, dtype):
    """Ids of experts that are switched off by now have score 0: no gradient, and no part in the others'."""
    T, E = 6, 40
    x = randn(3, T, E, dtype=dtype)
    x[:3, 5], x[3:, 5] = float("-inf"), torch.finfo(dtype).min
    idx = torch.tensor([2, 5, 9], dtype=torch.int32, device="cuda").expand(T, 3).contiguous()
    dw = randn(4, T, 3)
    got = M.select_experts_backward(dw, x, idx, score=score, renormalize=renorm)
    without = idx.clone()
    without[:, 1] = -1
    assert (got[:, 5] == 0).all()
    assert torch.equal(got, M.select_experts_backward(dw, x, without, score=score, renormalize=renorm))


# factors per column of 42 to 48 KB, beside 6 KB of other shared memory: odd rows, and aligned ones without dx
@pytest.mark.parametrize("T,H", [(9, 5376), (9, 5377), (160, 5501), (3, 5889), (9, 6001), (9, 6144), (9, 6145), (9, 5120), (9, 5632), (2, 6136)])
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("with_dx", [False, True])
def test_gradients_at_the_limit_of_shared_memory(T, H, pad, with_dx):
    y, dr, dx = (randn(i, T, H + pad, dtype=BF)[:, :H] for i in range(3))
    w = (1 + randn(9, H, std=0.2)).to(BF)
    kw = dict(post_weight=w, pre_weight=w if with_dx else None)
    b = M.block_norm_backward(dx if with_dx else None, dr, y, y, **kw)
    ref = R.block_norm_backward(dx if with_dx else None, dr, y, y, **kw)
    R.close(b.residual, *ref["residual"])
    R.close(b.y, *ref["y"], steps=3 * R.STEPS)
    R.close(b.post_weight, *ref["post_weight"], steps=3 * R.STEPS + T // 148 + 64)
