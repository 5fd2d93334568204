"""Cases of the operators around the expert layer: the block norm, the expert selection and the
8-bit linear layer.

A case is one call that a transformer block with routed experts makes: the norm that ends one
block and begins the next (forward and backward), the choice of experts from the router's logits
(forward and backward), and the projections of the dense (shared-expert) path in 8-bit integers.
``run`` computes a case in plain torch operations, or, with ``own`` set, through the package's
entry points; ``exact`` computes it in 64 bits.
"""

import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
_SZ = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
_FP8_MAX = 448.0
_FLT_MIN = 2.0 ** -126
_EPS = 1e-6


def _norm(op, name, T, H, y="bf16", r="bf16", x="bf16", post=False, gate="none", scale=1.0, pad=0):
    return {"name": name, "op": op, "T": T, "H": H, "y": y, "r": r, "x": x, "post": post, "gate": gate,
            "scale": scale, "pad": pad}


def _select(op, name, T, E, K, score="sigmoid", logits="fp32", bias=True, n_group=1, topk_group=1,
            group_score="top2", renormalize=True, scale=1.0, masked=0.0):
    return {"name": name, "op": op, "T": T, "E": E, "K": K, "score": score, "logits": logits, "bias": bias,
            "n_group": n_group, "topk_group": topk_group, "group_score": group_score,
            "renormalize": renormalize, "scale": scale, "masked": masked}


def _linear(name, T, K, N, x="bf16", swiglu=False, bias=False, y="bf16"):
    return {"name": name, "op": "linear", "T": T, "K": K, "N": N, "x": x, "swiglu": swiglu, "bias": bias, "y": y}


def listed():
    return [
        # one decoded token of one sequence: residual sum and norm before the next block
        _norm("norm", "norm_decode_1", 1, 7168),
        # prefill: the residual sum, norm and 1x128 quantisation that make the expert layer's input
        _norm("norm", "norm_prefill_e4m3", 4096, 7168, x="e4m3"),
        # norms on both sides of the block, a gate per token, an odd width, a 32-bit residual stream
        _norm("norm", "norm_sandwich_odd", 901, 5001, r="fp32", post=True, gate="token", scale=0.5),
        # training, a small batch with a gate per channel
        _norm("norm_bwd", "norm_bwd_64", 64, 7168, post=True, gate="channel"),
        # training, a whole micro-batch: both norms, a gate per channel, all gradients
        _norm("norm_bwd", "norm_bwd_4096", 4096, 7168, post=True, gate="channel"),
        # a decode batch of 16 with the layer's own routing (256 experts, 8 groups, 8 of them)
        _select("select", "select_decode_16", 16, 256, 8, n_group=8, topk_group=4, scale=2.5),
        # prefill of a long batch with the same routing
        _select("select", "select_prefill_16384", 16384, 256, 8, n_group=8, topk_group=4, scale=2.5),
        # a softmax router of few experts on 16-bit logits (many ties), some experts masked
        _select("select", "select_softmax_odd", 4097, 60, 4, score="softmax", logits="bf16", bias=False,
                renormalize=False, masked=0.1),
        # training: the gradient of the chosen experts' weights to all logits
        _select("select_bwd", "select_bwd_16384", 16384, 256, 8, score="softmax", bias=False),
        # one decoded token through the shared expert's gate and up projections (2 * 2048 x 7168)
        _linear("linear_decode_1", 1, 7168, 4096),
        # a decode batch through its down projection, with the activation between the two
        _linear("linear_swiglu_80", 80, 2048, 7168, swiglu=True),
        # prefill through the gate and up projections
        _linear("linear_prefill_8192", 8192, 7168, 4096),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "select", "select_bwd", "linear", "linear"])
    if op in ("norm", "norm_bwd"):
        H = _log(rng, 96, 8192)
        H = H // 128 * 128 if H > 256 and rng.random() < 0.6 else H
        T = _log(rng, 1, min(16384, 4096 * 7168 // H))
        c = _norm(op, "", T, H, y=rng.choice(["bf16", "bf16", "fp16"]), r=rng.choice(["bf16", "fp32"]),
                  x="e4m3" if op == "norm" and rng.random() < 0.4 else "bf16", post=rng.random() < 0.5,
                  gate=rng.choice(["none", "channel", "token", "full" if T > 1 else "channel"]), scale=rng.choice([1.0, 0.5]),
                  pad=rng.choice([0, 0, 8, 24]))
    elif op in ("select", "select_bwd"):
        G = rng.choice([1, 1, 4, 8])
        E = G * max(2, _log(rng, 8, 512) // G)
        # one expert whose weight is renormalised to 1 has no gradient: training takes two or more
        K = rng.randint(1 if op == "select" else 2, min(16, max(2, E // 2)))
        tg = G if G == 1 else max(rng.randint(1, G), -(-K // (E // G)))
        score = rng.choice(["sigmoid", "softmax"])
        c = _select(op, "", _log(rng, 1, 16384), E, K, score=score, logits=rng.choice(["fp32", "fp32", "bf16"]),
                    bias=rng.random() < 0.6, n_group=G, topk_group=tg, group_score=rng.choice(["top2", "max"]),
                    renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), masked=rng.choice([0.0, 0.0, 0.1]))
    else:
        K, N = 16 * _log(rng, 8, 448), _log(rng, 64, 8192)
        most = 8192 * 4096 * 7168
        T = _log(rng, 1, max(2, min(8192, most // (K * N))))
        c = _linear("", T, K, N, x=rng.choice(["bf16", "bf16", "int8"]), bias=rng.random() < 0.4,
                    y=rng.choice(["bf16", "bf16", "fp16"]))
        c["swiglu"] = c["x"] != "int8" and rng.random() < 0.3
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ inputs

def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _rows(g, T, H, std, dtype, pad):
    """[T, H] with a row pitch of H + pad: a slice of a wider buffer where pad is not 0."""
    return _randn(g, T, H + pad, std=std, dtype=dtype)[:, :H]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 13)
    s = {"case": case}
    T = case["T"]
    if case["op"] in ("norm", "norm_bwd"):
        H, yd, rd, pad = case["H"], _DT[case["y"]], _DT[case["r"]], case["pad"]
        # a residual stream has a few channels far larger than the others
        wide = 1.0 + 15.0 * (torch.rand(H, generator=g, device="cuda") < 0.004)
        s["y"] = _rows(g, T, H, 0.5, yd, pad)
        s["residual"] = (_rows(g, T, H, 1.5, torch.float32, pad) * wide).to(rd)
        s["pre_weight"] = (1.0 + _randn(g, H, std=0.2)).to(torch.bfloat16)
        s["post_weight"] = (1.0 + _randn(g, H, std=0.2)).to(torch.bfloat16) if case["post"] else None
        shape = {"none": None, "channel": (1, H), "token": (T, 1), "full": (T, H)}[case["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(_randn(g, *shape)).to(yd)
        if case["op"] == "norm_bwd":
            s["dx"] = _rows(g, T, H, 1.0, yd, pad)
            s["dresidual"] = _rows(g, T, H, 1.0, rd, pad)
    elif case["op"] in ("select", "select_bwd"):
        E, K = case["E"], case["K"]
        # experts differ in how often they are chosen
        logits = _randn(g, T, E) + _randn(g, 1, E, std=0.5)
        if case["masked"]:   # experts that are switched off for a token
            off = torch.rand(T, E, generator=g, device="cuda") < case["masked"]
            off[T // 2] |= T > 1   # a padding token: nothing to choose from
            logits = logits.masked_fill(off, float("-inf"))
        s["logits"] = logits.to(_DT[case["logits"]])
        s["bias"] = _randn(g, E, std=0.1 if case["score"] == "sigmoid" else 0.1 / E) if case["bias"] else None
        if case["op"] == "select_bwd":
            # what the selection gives: ascending, and -1 where it found none
            pick = torch.topk(torch.rand(T, E, generator=g, device="cuda") + s["logits"].float(), K, dim=1)
            idx = torch.sort(torch.where(torch.isinf(pick.values), E, pick.indices), dim=1).values
            s["idx"] = torch.where(idx == E, -1, idx).to(torch.int32)
            s["dw"] = _randn(g, T, K)
    else:
        K, N = case["K"], case["N"]
        cols = 2 * K if case["swiglu"] else K
        if case["x"] == "int8":
            s["x"] = torch.clamp(torch.round(_randn(g, T, K, std=36.0)), -127, 127).to(torch.int8)
            s["x_scale"] = torch.rand(T, generator=g, device="cuda") * 0.02 + 0.01
        else:
            # activations: tokens of different size, a few large channels
            wide = 1.0 + 9.0 * (torch.rand(cols, generator=g, device="cuda") < 0.004)
            s["x"] = (_randn(g, T, cols) * wide * (0.5 + torch.rand(T, 1, generator=g, device="cuda"))).to(_DT[case["x"]])
            s["x_scale"] = None
        s["weight"] = torch.clamp(torch.round(_randn(g, N, K, std=36.0)), -127, 127).to(torch.int8)
        s["weight_scale"] = (torch.rand(N, generator=g, device="cuda") + 0.5) * 0.02 / 36.0
        s["bias"] = _randn(g, N, std=0.5) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------ plain forms

def _rms(v):
    return torch.rsqrt(v.square().mean(dim=1, keepdim=True) + _EPS)


def _quantize_e4m3(x):
    """1x128 blocks of each row: codes e4m3 [T, H], scales f32 [ceil(H / 128), T]."""
    T, H = x.shape
    nb = -(-H // 128)
    p = torch.zeros(T, nb * 128, dtype=x.dtype, device=x.device)
    p[:, :H] = x
    p = p.view(T, nb, 128)
    scale = torch.clamp(p.abs().amax(dim=2), min=1e-12) / _FP8_MAX
    q = (p / scale.unsqueeze(2)).view(T, nb * 128)[:, :H].to(torch.float8_e4m3fn).contiguous()
    return q, scale.t().contiguous()


def _plain_norm(s):
    c = s["case"]
    n = s["y"].float()
    if s["post_weight"] is not None:
        n = n * _rms(n) * s["post_weight"].float()
    if s["gate"] is not None:
        n = n * s["gate"].float()
    r = s["residual"].float() + c["scale"] * n
    x = r * _rms(r) * s["pre_weight"].float()
    if c["x"] == "e4m3":
        q, scale = _quantize_e4m3(x)
        return {"residual": r.to(_DT[c["r"]]), "x": q, "x_scale": scale}
    return {"residual": r.to(_DT[c["r"]]), "x": x.to(_DT[c["x"]])}


def _plain_norm_bwd(s):
    c = s["case"]
    r, dx, w = s["residual"].float(), s["dx"].float(), s["pre_weight"].float()
    rstd = _rms(r)
    rhat = r * rstd
    wdx = w * dx
    G = s["dresidual"].float() + rstd * (wdx - rhat * (wdx * rhat).mean(dim=1, keepdim=True))
    out = {"residual": G.to(_DT[c["r"]]), "pre_weight": (dx * rhat).sum(dim=0)}
    y = s["y"].float()
    if s["post_weight"] is not None:
        ystd = _rms(y)
        yhat = y * ystd
        n = yhat * s["post_weight"].float()
    else:
        n = y
    dn = c["scale"] * G
    if s["gate"] is not None:
        dg = dn * n
        if c["gate"] == "channel":
            out["gate"] = dg.sum(dim=0, keepdim=True)
        elif c["gate"] == "token":
            out["gate"] = dg.sum(dim=1, keepdim=True)
        else:
            out["gate"] = dg.to(_DT[c["y"]])
        dn = dn * s["gate"].float()
    if s["post_weight"] is not None:
        out["post_weight"] = (dn * yhat).sum(dim=0)
        wdn = s["post_weight"].float() * dn
        dn = ystd * (wdn - yhat * (wdn * yhat).mean(dim=1, keepdim=True))
    out["y"] = dn.to(_DT[c["y"]])
    return out


def _scores(x, score):
    """The scores experts are chosen by: 32-bit values by definition, the exponential (and the
    softmax's quotient) rounded to 32 bits once, so that no order of summing changes a choice."""
    if score == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x.double()).float())
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(x.double() - m)
    return (e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)).float()


def _lowest(n):
    return torch.tensor(float("-inf"), device=n.device)


def _plain_select(s):
    c = s["case"]
    x = s["logits"].float()
    T, E = x.shape
    K, G = c["K"], c["n_group"]
    p = _scores(x, c["score"])
    sel = p if s["bias"] is None else p + s["bias"].float()
    sel = torch.where(torch.isinf(x), _lowest(x), sel)
    if G > 1:
        grouped = sel.view(T, G, E // G)
        if c["group_score"] == "top2":
            two = torch.topk(grouped, 2, dim=2).values
            gs = two[..., 0] + torch.where(torch.isinf(two[..., 1]), torch.zeros_like(two[..., 1]), two[..., 1])
        else:
            gs = grouped.amax(dim=2)
        kept = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=x.device).scatter_(1, kept, True)
        sel = torch.where(keep.unsqueeze(2), grouped, _lowest(x)).view(T, E)
    # the K highest, equal ones from the lowest index up, listed by index; -1 where none is left
    best = torch.sort(sel, dim=1, descending=True, stable=True)
    idx = torch.where(torch.isinf(best.values[:, :K]), E, best.indices[:, :K])
    idx = torch.sort(idx, dim=1).values
    none = idx == E
    w = torch.where(none, torch.zeros_like(x[:, :1]), p.gather(1, idx.clamp(max=E - 1)))
    if c["renormalize"]:
        w = w / (w.sum(dim=1, keepdim=True) + 1e-20)
    return {"idx": torch.where(none, -1, idx).to(torch.int32), "w": w * c["scale"],
            "counts": torch.bincount(idx.view(-1), minlength=E + 1)[:E].to(torch.int32)}


def _plain_select_bwd(s):
    c = s["case"]
    x, idx, dw = s["logits"].float(), s["idx"].long(), s["dw"] * c["scale"]
    p = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.exp(x - x.amax(dim=1, keepdim=True))
    if c["score"] == "softmax":
        p = p / p.sum(dim=1, keepdim=True)
    p = torch.where(torch.isinf(x), torch.zeros_like(p), p)   # also a row with nothing to choose from
    none, idx = idx < 0, idx.clamp(min=0)
    ps = torch.where(none, torch.zeros_like(dw), p.gather(1, idx))
    dw = torch.where(none, torch.zeros_like(dw), dw)
    if c["renormalize"]:
        total = ps.sum(dim=1, keepdim=True) + 1e-20
        dw = (dw - (dw * ps).sum(dim=1, keepdim=True) / total) / total
    dp = torch.zeros_like(x).scatter_add_(1, idx, torch.where(none, torch.zeros_like(dw), dw))
    if c["score"] == "sigmoid":
        dx = dp * p * (1.0 - p)
    else:
        dx = p * (dp - (dp * p).sum(dim=1, keepdim=True))
    return {"logits": dx.to(_DT[c["logits"]])}


def _plain_linear(s):
    c = s["case"]
    v = s["x"].float()
    if c["x"] == "int8":
        q, scale = v, s["x_scale"].unsqueeze(1)
    else:
        if c["swiglu"]:
            a, b = v[:, :c["K"]], v[:, c["K"]:]
            v = b / (1.0 + torch.exp(-b)) * a
        scale = torch.clamp(v.abs().amax(dim=1, keepdim=True) / 127.0, min=_FLT_MIN)
        q = torch.clamp(torch.round(v / scale), -127, 127)
    y = (q @ s["weight"].float().t()) * scale * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(_DT[c["y"]])


_PLAIN = {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "select": _plain_select,
          "select_bwd": _plain_select_bwd, "linear": _plain_linear}


# ------------------------------------------------------------------------------------ own calls

def _own(s):
    import moe_swarm_b200 as M

    c = s["case"]
    op = c["op"]
    if op == "norm":
        o = M.block_norm(s["y"], s["residual"], post_weight=s["post_weight"], gate=s["gate"], scale=c["scale"],
                         pre_weight=s["pre_weight"], eps=_EPS, x_dtype=_DT[c["x"]])
        return {"residual": o.residual, "x": o.x, "x_scale": o.x_scale}
    if op == "norm_bwd":
        o = M.block_norm_backward(s["dx"], s["dresidual"], s["residual"], s["y"], post_weight=s["post_weight"],
                                  gate=s["gate"], scale=c["scale"], pre_weight=s["pre_weight"], eps=_EPS)
        return {"residual": o.residual, "y": o.y, "pre_weight": o.pre_weight, "post_weight": o.post_weight,
                "gate": o.gate}
    if op == "select":
        o = M.select_experts(s["logits"], c["K"], score=c["score"], bias=s["bias"], n_group=c["n_group"],
                             topk_group=c["topk_group"], group_score=c["group_score"],
                             renormalize=c["renormalize"], scale=c["scale"], counts=True)
        return {"idx": o.idx, "w": o.w, "counts": o.counts}
    if op == "select_bwd":
        return {"logits": M.select_experts_backward(s["dw"], s["logits"], s["idx"], score=c["score"],
                                                    renormalize=c["renormalize"], scale=c["scale"])}
    return M.int8_linear(s["x"], s["weight"], s["weight_scale"], x_scale=s["x_scale"], bias=s["bias"],
                         swiglu=c["swiglu"], out_dtype=_DT[c["y"]])


@torch.no_grad()
def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ work

def work(case):
    T = case["T"]
    if case["op"] == "norm":
        H = case["H"]
        row = H * (_SZ[case["y"]] + 2 * _SZ[case["r"]] + _SZ[case["x"]])
        row += 4 * -(-H // 128) if case["x"] == "e4m3" else 0
        fixed = 2 * H * (2 if case["post"] else 1)
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]] * _SZ[case["y"]]
        return {"bytes": T * row + fixed + gate, "flops": T * H * (14 if case["post"] else 8)}
    if case["op"] == "norm_bwd":
        H = case["H"]
        row = H * (3 * _SZ[case["y"]] + 3 * _SZ[case["r"]])
        fixed = (2 + 4) * H * (2 if case["post"] else 1)
        gate = {"none": 0, "channel": H * (_SZ[case["y"]] + 4), "token": T * (_SZ[case["y"]] + 4),
                "full": 2 * T * H * _SZ[case["y"]]}[case["gate"]]
        return {"bytes": T * row + fixed + gate, "flops": T * H * (24 if case["post"] else 14)}
    if case["op"] == "select":
        E, K = case["E"], case["K"]
        return {"bytes": T * (E * _SZ[case["logits"]] + 8 * K) + 4 * E + (4 * E if case["bias"] else 0),
                "flops": T * E * 4}
    if case["op"] == "select_bwd":
        E, K = case["E"], case["K"]
        return {"bytes": T * (2 * E * _SZ[case["logits"]] + 8 * K), "flops": T * E * 6}
    K, N = case["K"], case["N"]
    x = K + 4 / T if case["x"] == "int8" else K * _SZ[case["x"]] * (2 if case["swiglu"] else 1)
    return {"bytes": T * (x + N * _SZ[case["y"]]) + N * K + N * (8 if case["bias"] else 4), "flops": 2 * T * N * K}


# ------------------------------------------------------------------------------------ 64 bits

def _d(t):
    return None if t is None else t.to(torch.float64)


def _exact_norm(s):
    c = s["case"]
    y, r, w, wp, g = _d(s["y"]), _d(s["residual"]), _d(s["pre_weight"]), _d(s["post_weight"]), _d(s["gate"])
    H = y.shape[1]
    if wp is not None:
        y = y / ((y * y).sum(1, keepdim=True) / H + _EPS).sqrt() * wp
    r = r + c["scale"] * (y if g is None else g * y)
    x = r / ((r * r).sum(1, keepdim=True) / H + _EPS).sqrt() * w
    if c["x"] != "e4m3":
        return {"residual": r, "x": x}
    nb = -(-H // 128)
    blocks = torch.nn.functional.pad(x, (0, nb * 128 - H)).reshape(-1, 128)
    scale = blocks.abs().max(dim=1).values.clamp(min=1e-12) / _FP8_MAX
    codes = (blocks / scale[:, None]).reshape(-1, nb * 128)[:, :H]
    return {"residual": r, "x": codes.to(torch.float8_e4m3fn).to(torch.float64),
            "x_scale": scale.reshape(-1, nb).t().contiguous()}


def _exact_norm_bwd(s):
    """The same gradients from the definition: d/dv of v / sqrt(mean(v^2) + eps)."""
    c = s["case"]
    dx, dr, r, y = _d(s["dx"]), _d(s["dresidual"]), _d(s["residual"]), _d(s["y"])
    w, wp, g = _d(s["pre_weight"]), _d(s["post_weight"]), _d(s["gate"])
    H = r.shape[1]

    def back(v, up):
        ms = (v * v).sum(1, keepdim=True) / H + _EPS
        return up / ms.sqrt() - v * ((up * v).sum(1, keepdim=True) / H) / ms.pow(1.5)

    G = dr + back(r, dx * w)
    out = {"residual": G, "pre_weight": (dx * r / ((r * r).sum(1, keepdim=True) / H + _EPS).sqrt()).sum(0)}
    u = y if wp is None else y / ((y * y).sum(1, keepdim=True) / H + _EPS).sqrt()
    n = u if wp is None else u * wp
    if g is not None:
        full = c["scale"] * G * n
        out["gate"] = {"channel": full.sum(0, keepdim=True), "token": full.sum(1, keepdim=True)}.get(c["gate"], full)
    dn = c["scale"] * G * (1.0 if g is None else g)
    if wp is not None:
        out["post_weight"] = (dn * u).sum(0)
        dn = back(y, dn * wp)
    out["y"] = dn
    return out


def _exact_select(s):
    """The choice by the 32-bit scores that the definition names, the weights of the chosen in 64 bits."""
    c = s["case"]
    x = _d(s["logits"])
    T, E = x.shape
    K, G = c["K"], c["n_group"]
    off = x == float("-inf")
    if c["score"] == "sigmoid":
        p = torch.sigmoid(x)
        chosen_by = 1.0 / (1.0 + torch.exp(-x).to(torch.float32))
    else:
        p = torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
        chosen_by = p.to(torch.float32)
    if s["bias"] is not None:
        chosen_by = chosen_by + s["bias"]
    chosen_by = chosen_by.masked_fill(off, float("-inf"))
    if G > 1:
        per = chosen_by.reshape(T, G, -1)
        first = per.sort(dim=2, descending=True).values
        if c["group_score"] == "top2":
            gs = first[..., 0] + first[..., 1].masked_fill(first[..., 1] == float("-inf"), 0.0)
        else:
            gs = first[..., 0]
        order = gs.argsort(dim=1, descending=True, stable=True)
        rank = order.argsort(dim=1)
        per = per.masked_fill((rank >= c["topk_group"]).unsqueeze(2), float("-inf"))
        chosen_by = per.reshape(T, E)
    rank = chosen_by.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
    taken = (rank < K) & (chosen_by > float("-inf"))
    key = torch.where(taken, torch.arange(E, device=x.device).expand(T, E), E)
    idx = key.sort(dim=1).values[:, :K]
    w = torch.cat([p, torch.zeros(T, 1, dtype=p.dtype, device=p.device)], dim=1).gather(1, idx)
    if c["renormalize"]:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return {"idx": idx.masked_fill(idx == E, -1).to(torch.int32), "w": w * c["scale"],
            "counts": taken.sum(0).to(torch.int32)}


def _exact_select_bwd(s):
    c = s["case"]
    x, idx, dw = _d(s["logits"]), s["idx"].long(), _d(s["dw"]) * c["scale"]
    p = torch.sigmoid(x) if c["score"] == "sigmoid" else torch.nan_to_num(torch.softmax(x, dim=1), nan=0.0)
    some, idx = (idx >= 0).to(torch.float64), idx.clamp(min=0)
    chosen = p.gather(1, idx) * some
    dw = dw * some
    if c["renormalize"]:
        S = chosen.sum(1, keepdim=True) + 1e-20
        dw = dw / S - (dw * chosen).sum(1, keepdim=True) / (S * S)
    if c["score"] == "sigmoid":
        return {"logits": torch.zeros_like(x).scatter_add_(1, idx, dw * chosen * (1.0 - chosen))}
    dx = -p * (dw * chosen).sum(1, keepdim=True)
    return {"logits": dx.scatter_add_(1, idx, dw * chosen)}


def _exact_linear(s):
    c = s["case"]
    v = _d(s["x"])
    if s["x_scale"] is not None:
        scale = _d(s["x_scale"])
    else:
        if c["swiglu"]:
            up, gated = v.split(c["K"], dim=1)
            v = up * gated * torch.sigmoid(gated)
        scale = (v.abs().max(dim=1).values / 127.0).clamp(min=_FLT_MIN)
        v = (v / scale[:, None]).round().clamp(-127, 127)
    y = torch.matmul(v, _d(s["weight"]).t()) * scale[:, None] * _d(s["weight_scale"])[None]
    return y if s["bias"] is None else y + _d(s["bias"])[None]


_EXACT = {"norm": _exact_norm, "norm_bwd": _exact_norm_bwd, "select": _exact_select,
          "select_bwd": _exact_select_bwd, "linear": _exact_linear}


@torch.no_grad()
def exact(case, seed):
    return _EXACT[case["op"]](prepare(case, seed))
