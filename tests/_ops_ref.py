"""Plain 64-bit forms of the operators around the layer, and the error bounds of the tests.

Bounds are derived, not fitted: a result in a type with p significant bits is off by at most
2^-p of its value for its one rounding, and the 32-bit arithmetic before it by a few units
(2^-24) of the terms it adds up.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24
# 32-bit steps of one element: row sum (16 in a thread, 5 + 5 shuffles), mean, rsqrt (2 units),
# products and sums around them: fewer than 64 roundings of terms no larger than `mag`.
STEPS = 64


def close(got, ref, mag, steps=STEPS):
    """got within one rounding of its type and `steps` 32-bit roundings of `mag` (per element)."""
    got64, ref = got.double().cpu(), ref.double().cpu()
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0   # fp16 subnormals: absolute spacing
    tol = U[got.dtype] * ref.abs() * 1.001 + steps * U32 * torch.as_tensor(mag).double().cpu() + tiny
    # what exceeds the type's range rounds to its infinity
    over = torch.isinf(ref.to(got.dtype)) & torch.isfinite(ref)
    bad = torch.where(over, got64 != ref.sign() * float("inf"), ~((got64 - ref).abs() <= tol))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got64 - ref).abs() / tol.clamp(min=1e-300)).max()} of the bound"


def rstd(v, eps):
    return (v.square().mean(dim=1, keepdim=True) + eps).rsqrt()


def d(t):
    return None if t is None else t.double().cpu()


def block_norm(y, residual, post_weight=None, gate=None, scale=1.0, pre_weight=None, eps=1e-6, off=0.0):
    """(r', x, magnitude of the terms of r', magnitude of x's)."""
    y, residual, post_weight, gate, pre_weight = map(d, (y, residual, post_weight, gate, pre_weight))
    if y is None:
        r, mag = residual, residual.abs()
    else:
        n = y if post_weight is None else y * rstd(y, eps) * (post_weight + off)
        n = n if gate is None else n * gate
        r = (0 if residual is None else residual) + scale * n
        mag = (scale * n).abs() + (0 if residual is None else residual.abs())
    if pre_weight is None:
        return r, None, mag, None
    s = rstd(r, eps)
    x = r * s * (pre_weight + off)
    # r's own error moves the row's mean square as well: all of the row's terms count
    row = (mag.square().mean(dim=1, keepdim=True)).sqrt() * s
    return r, x, mag, mag * s * (pre_weight + off).abs() + x.abs() * row


def loss(y, residual, post_weight, gate, scale, pre_weight, eps, off, dx, dr):
    """sum(dx * x) + sum(dr * r') of the forward, differentiable, for gradients by differences."""
    n = y if post_weight is None else y * rstd(y, eps) * (post_weight + off)
    n = n if gate is None else n * gate
    r = residual + scale * n
    total = (dr * r).sum()
    if pre_weight is not None:
        total = total + (dx * r * rstd(r, eps) * (pre_weight + off)).sum()
    return total


def block_norm_backward(dx, dr, r, y, post_weight=None, gate=None, scale=1.0, pre_weight=None, eps=1e-6, off=0.0):
    """{name: (gradient, magnitude of its terms)}; the gate's gradient per element."""
    dx, dr, r, y, wp, g, w = map(d, (dx, dr, r, y, post_weight, gate, pre_weight))
    out = {}
    G, Gm = (torch.zeros_like(r), torch.zeros_like(r)) if dr is None else (dr, dr.abs())
    if dx is not None:
        s = rstd(r, eps)
        rh, wdx = r * s, (w + off) * dx
        m = (wdx * rh).abs().mean(dim=1, keepdim=True)
        G = G + s * (wdx - rh * (wdx * rh).mean(dim=1, keepdim=True))
        Gm = Gm + s * (wdx.abs() + rh.abs() * m)
        out["pre_weight"] = ((dx * rh).sum(0), (dx * rh).abs().sum(0))
    out["residual"] = (G, Gm)
    if y is None:
        return out
    ys = rstd(y, eps) if wp is not None else None
    yh = y if wp is None else y * ys
    n = yh if wp is None else yh * (wp + off)
    gv = 1.0 if g is None else g
    out["gate"] = (scale * G * n, (scale * Gm * n).abs())
    dn, dnm = scale * G * gv, (scale * Gm * gv).abs()
    if wp is None:
        out["y"] = (dn, dnm)
    else:
        out["post_weight"] = ((dn * yh).sum(0), (dnm * yh.abs()).sum(0))
        a, am = (wp + off) * dn, (wp + off).abs() * dnm
        out["y"] = (ys * (a - yh * (a * yh).mean(dim=1, keepdim=True)),
                    ys * (am + yh.abs() * (am * yh.abs()).mean(dim=1, keepdim=True)))
    return out


def scores(x, score):
    """64-bit scores and the 32-bit values the choice goes by; NaN where the logits make it."""
    x = x.double().cpu()
    if score == "sigmoid":
        return torch.sigmoid(x), 1.0 / (1.0 + torch.exp(-x).float())
    p = torch.softmax(x, dim=1)
    p = torch.where(torch.isneginf(x), torch.zeros_like(p), p)
    return p, p.float()


def select(logits, top_k, score="sigmoid", bias=None, n_group=1, topk_group=1, group_score="top2",
           renormalize=True, scale=1.0):
    """(idx, w, counts) row by row, by sorting (score, -id) pairs."""
    T, E = logits.shape
    low = torch.finfo(logits.dtype).min
    off = logits.cpu() <= low
    p64, p32 = scores(torch.where(off, torch.full_like(logits.float().cpu(), float("-inf")), logits.float().cpu()), score)
    sel = p32 if bias is None else p32 + bias.float().cpu()
    idx = torch.full((T, top_k), -1, dtype=torch.int32)
    w = torch.zeros(T, top_k, dtype=torch.float64)
    counts = torch.zeros(E, dtype=torch.int32)
    gs = E // n_group
    ninf = float("-inf")
    for t in range(T):
        v = [ninf if off[t, e] else float(sel[t, e]) for e in range(E)]
        if any(u != u for u in v):
            w[t] = float("nan")
            continue
        if n_group > 1:
            best = []
            for g in range(n_group):
                top = sorted(v[g * gs:(g + 1) * gs], reverse=True)
                second = top[1] if gs > 1 and top[1] != ninf else 0.0
                s = float(torch.tensor(top[0]) + torch.tensor(second)) if group_score == "top2" else top[0]
                best.append((-s, g))
            kept = {g for _, g in sorted(best)[:topk_group]}
            v = [u if e // gs in kept else ninf for e, u in enumerate(v)]
        ids = sorted(e for u, e in sorted((-u, e) for e, u in enumerate(v))[:top_k] if v[e] != ninf)
        ws = p64[t, ids]
        if renormalize:
            ws = ws / (ws.sum() + 1e-20)
        idx[t, :len(ids)] = torch.tensor(ids, dtype=torch.int32)
        w[t, :len(ids)] = ws * scale
        for e in ids:
            counts[e] += 1
    return idx, w, counts


def select_weights(x, idx, score, renormalize, scale):
    """The chosen weights as a differentiable function of 64-bit logits (ids fixed, -1: weight 0)."""
    p = torch.sigmoid(x) if score == "sigmoid" else torch.softmax(x, dim=1)
    some = (idx >= 0).double()
    c = p.gather(1, idx.clamp(min=0).long()) * some
    if renormalize:
        c = c / (c.sum(1, keepdim=True) + 1e-20)
    return c * scale


def quantize(v):
    """(codes, scale, distance of v / scale from the nearest rounding boundary) in 64 bits."""
    v = v.double().cpu()
    s = (v.abs().amax(dim=1) / 127.0).clamp(min=2.0 ** -126)
    u = v / s[:, None]
    return u.round().clamp(-127, 127), s, ((u - u.floor()) - 0.5).abs()


def swiglu(x):
    x = x.double().cpu()
    up, gate = x.chunk(2, dim=1)
    return torch.nn.functional.silu(gate) * up
