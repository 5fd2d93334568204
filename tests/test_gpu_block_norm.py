"""GPU: the norms around a block (block_norm) and their gradients against the 64-bit forms."""
import pytest
import torch

import moe_swarm_b200 as M
from moe_swarm_b200 import workload as W
from tests import _ops_ref as R

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make(T, H, y_dtype, r_dtype, post, gate, seed=0, pad=0, wdt=BF):
    g = gen(seed)

    def t(rows, cols, std, dtype):
        return (torch.randn(rows, cols + pad, generator=g, device="cuda") * std).to(dtype)[:, :cols]

    shape = {None: None, "channel": (1, H), "vector": (H,), "token": (T, 1), "full": (T, H), "one": (1, 1)}[gate]
    return dict(
        y=t(T, H, 0.7, y_dtype), residual=t(T, H, 2.0, r_dtype),
        post_weight=(1 + torch.randn(H, generator=g, device="cuda") * 0.3).to(wdt) if post else None,
        pre_weight=(1 + torch.randn(H, generator=g, device="cuda") * 0.3).to(wdt),
        gate=None if shape is None else torch.rand(shape, generator=g, device="cuda").to(y_dtype))


# (few rows: one CTA or warp each; many: the ring, below)
SHAPES = [(1, 1), (1, 7168), (3, 7), (5, 8), (9, 129), (17, 512), (2, 513), (33, 1000), (7, 4096), (3, 5001),
          (2, 8192), (2, 8193), (1, 16384), (300, 64)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (BF, F32), (FP, FP), (FP, F32), (F32, F32), (FP, BF), (BF, FP)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "token"), (True, "channel"), (False, "full")])
def test_forward(T, H, y_dtype, r_dtype, post, gate):
    a = make(T, H, y_dtype, r_dtype, post, gate)
    o = M.block_norm(**a, scale=0.75, eps=1e-5)
    r, x, rm, xm = R.block_norm(**a, scale=0.75, eps=1e-5)
    assert o.residual.dtype == r_dtype and o.x.dtype == y_dtype and o.x_scale is None
    R.close(o.residual, r, rm)
    R.close(o.x, x, xm)


@pytest.mark.parametrize("pad", [1, 2, 8, 24])
@pytest.mark.parametrize("H", [640, 641])
def test_row_pitch(H, pad):
    a = make(13, H, BF, F32, True, "full", seed=3, pad=pad)
    out = torch.zeros(13, H + pad, dtype=BF, device="cuda")
    res = torch.full((13, H + pad), 7.0, device="cuda")
    o = M.block_norm(**a, out=out[:, :H], residual_out=res[:, :H])
    r, x, rm, xm = R.block_norm(**a)
    R.close(o.residual, r, rm)
    R.close(o.x, x, xm)
    assert (out[:, H:] == 0).all() and (res[:, H:] == 7.0).all()   # nothing beside the rows


@pytest.mark.parametrize("offset", [1, 3, 4])
def test_unaligned_base(offset):
    H, T = 256, 4
    g = gen(5)
    y = torch.randn(T * H + 8, generator=g, device="cuda").to(BF)[offset:offset + T * H].view(T, H)
    r = torch.randn(T * H + 8, generator=g, device="cuda").to(BF)[offset:offset + T * H].view(T, H)
    w = torch.rand(H + 8, generator=g, device="cuda").to(BF)[offset:offset + H]
    o = M.block_norm(y, r, pre_weight=w)
    ref = R.block_norm(y, r, pre_weight=w)
    R.close(o.residual, ref[0], ref[2])
    R.close(o.x, ref[1], ref[3])


def test_partial_forms():
    a = make(6, 384, BF, BF, True, "one", seed=8, wdt=F32)
    r, x, rm, xm = R.block_norm(**a, off=1.0)
    o = M.block_norm(**a, weight_offset=1.0, x_dtype=F32)
    R.close(o.residual, r, rm)
    R.close(o.x, x, xm)
    # no next norm
    o = M.block_norm(a["y"], a["residual"], post_weight=a["post_weight"])
    assert o.x is None
    ref = R.block_norm(a["y"], a["residual"], post_weight=a["post_weight"])
    R.close(o.residual, ref[0], ref[2])
    # the norm of the residual alone: the stream itself comes back
    o = M.block_norm(None, a["residual"], pre_weight=a["pre_weight"])
    assert o.residual.data_ptr() == a["residual"].data_ptr()
    ref = R.block_norm(None, a["residual"], pre_weight=a["pre_weight"])
    R.close(o.x, ref[1], ref[3])
    # no residual: the first block's output starts the stream
    o = M.block_norm(a["y"], None, pre_weight=a["pre_weight"], scale=3.0)
    ref = R.block_norm(a["y"], None, pre_weight=a["pre_weight"], scale=3.0)
    R.close(o.residual, ref[0], ref[2])
    R.close(o.x, ref[1], ref[3])
    # in place
    ref = R.block_norm(a["y"], a["residual"])
    o = M.block_norm(a["y"], a["residual"], residual_out=a["residual"])
    R.close(a["residual"], ref[0], ref[2])


@pytest.mark.parametrize("T,H", [(1500, 512), (650, 7168), (700, 2880), (600, 8192), (2000, 96), (700, 1001)])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_partial_forms_of_many_rows(T, H, dtype):
    a = make(T, H, dtype, dtype, True, None, seed=T)
    w = dict(pre_weight=a["pre_weight"])
    o = M.block_norm(None, a["residual"], **w, weight_offset=1.0)
    ref = R.block_norm(None, a["residual"], **w, off=1.0)
    R.close(o.x, ref[1], ref[3])
    e = M.block_norm(None, a["residual"], **w, weight_offset=1.0, x_dtype=torch.float8_e4m3fn)
    val = e.x.double() * e.x_scale.t().double().repeat_interleave(128, dim=1)[:, :H]
    assert ((val.cpu() - ref[1]).abs() <= ref[1].abs() * 2.0 ** -4 * 1.01 + e.x_scale.max().item() * 2.0 ** -9).all()
    for kw in (w, dict(post_weight=a["post_weight"]), dict(post_weight=a["post_weight"], **w)):
        o = M.block_norm(a["y"], None, scale=3.0, **kw)
        ref = R.block_norm(a["y"], None, scale=3.0, **kw)
        R.close(o.residual, ref[0], ref[2])
        if "pre_weight" in kw:
            R.close(o.x, ref[1], ref[3])


@pytest.mark.parametrize("T,H", [(1, 7168), (5, 128), (3, 130), (4, 1000), (2, 7), (70, 512), (3, 5001)])
@pytest.mark.parametrize("r_dtype", [BF, F32])
def test_e4m3_blocks(T, H, r_dtype):
    a = make(T, H, BF, r_dtype, True, "token", seed=11)
    a["residual"][0, : min(H, 128)] = 0
    a["y"][0, : min(H, 128)] = 0          # a block of zeros
    o = M.block_norm(**a, x_dtype=torch.float8_e4m3fn)
    r, x, rm, xm = R.block_norm(**a)
    nb = -(-H // 128)
    assert o.x.dtype == torch.float8_e4m3fn and o.x_scale.shape == (nb, T)
    xp = torch.nn.functional.pad(x, (0, nb * 128 - H)).view(T, nb, 128)
    mp = torch.nn.functional.pad(xm, (0, nb * 128 - H)).view(T, nb, 128)
    amax = xp.abs().amax(dim=2)
    # the maximum carries the 32-bit error of its element, the quotient one rounding more
    R.close(o.x_scale.t().contiguous(), amax.clamp(min=1e-12) / 448, (mp.amax(dim=2) + amax) / 448)
    val = o.x.float().cpu().double() * o.x_scale.t().cpu().double().repeat_interleave(128, dim=1)[:, :H]
    # e4m3: half a unit of 4 significant bits, or of the subnormals' 2^-9, and the 32-bit error before it
    s = o.x_scale.t().cpu().double().repeat_interleave(128, dim=1)[:, :H]
    tol = (x.abs() * 2.0 ** -4).maximum(s * 2.0 ** -10) * 1.001 + 2 * R.STEPS * R.U32 * (xm + x.abs())
    assert ((val - x).abs() <= tol).all()


def test_e4m3_is_the_layers_input():
    """A norm's e4m3 result has the layout and the scales of the layer's hidden states."""
    T = 9
    a = make(T, M.H, BF, F32, False, None, seed=4)
    o = M.block_norm(**a, x_dtype=torch.float8_e4m3fn)
    x32 = M.block_norm(**a, x_dtype=F32).x
    q, s = W.quantize_tokens(x32)
    R.close(o.x_scale, s, s, steps=2)   # torch may divide by 448 as a product with its reciprocal
    # codes differ at most where the quotient lies on a rounding boundary: reciprocal against quotient
    assert (o.x.float() != q.float()).float().mean() < 1e-4


def test_rows_do_not_touch_each_other():
    """Infinities, NaN and zeros stay in their rows; a zero row's norm is zero."""
    a = make(6, 300, BF, F32, True, "token", seed=2)
    clean = M.block_norm(**a)
    a["y"][1, 5] = float("inf")
    a["residual"][2, 7] = float("nan")
    a["y"][4] = 0
    a["residual"][4] = 0
    o = M.block_norm(**a)
    for t in (0, 3, 5):
        assert torch.equal(o.x[t], clean.x[t]) and torch.equal(o.residual[t], clean.residual[t])
    assert torch.isnan(o.x[2]).all()
    assert (o.x[4] == 0).all() and (o.residual[4] == 0).all()
    q = M.block_norm(**a, x_dtype=torch.float8_e4m3fn)
    assert torch.isnan(q.x_scale[:, 2]).all() and torch.isfinite(q.x_scale[:, [0, 3, 4, 5]]).all()


@pytest.mark.parametrize("T,H", [(1, 1), (1, 7168), (2, 513), (5, 129), (64, 640), (300, 96), (333, 1001), (700, 2048),
                                 (3, 8200), (2, 16384)])
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (BF, F32), (FP, F32), (F32, F32), (FP, BF), (BF, FP)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "token"), (True, "channel"), (True, "full"),
                                       (False, "one"), (False, "vector")])
def test_backward(T, H, y_dtype, r_dtype, post, gate):
    a = make(T, H, y_dtype, r_dtype, post, gate, seed=1)
    g = gen(77)
    dx = torch.randn(T, H, generator=g, device="cuda").to(y_dtype)
    dr = torch.randn(T, H, generator=g, device="cuda").to(r_dtype)
    kw = dict(post_weight=a["post_weight"], gate=a["gate"], scale=0.5, pre_weight=a["pre_weight"], eps=1e-5)
    o = M.block_norm_backward(dx, dr, a["residual"], a["y"], **kw)
    ref = R.block_norm_backward(dx, dr, a["residual"], a["y"], **kw)
    R.close(o.residual, *ref["residual"])
    R.close(o.y, *ref["y"], steps=3 * R.STEPS)
    # sums over rows: at most 8 + 8 parts of at most ceil(T / 148) + 1 rows each, one after another
    steps = 3 * R.STEPS + T // 148 + 64
    R.close(o.pre_weight, *ref["pre_weight"], steps=steps)
    if post:
        R.close(o.post_weight, *ref["post_weight"], steps=steps)
    else:
        assert o.post_weight is None
    if gate is None:
        assert o.gate is None
        return
    assert o.gate.shape == a["gate"].shape
    dg, mag = ref["gate"]
    if gate in ("channel", "vector"):
        dg, mag = dg.sum(0), mag.sum(0)
    elif gate == "token":
        dg, mag = dg.sum(1), mag.sum(1)
    elif gate == "one":
        dg, mag = dg.sum(), mag.sum()
    summed = gate != "full" or T == 1 or H == 1
    assert o.gate.dtype == (F32 if summed else y_dtype)
    R.close(o.gate.reshape(dg.shape), dg, mag, steps=steps)


@pytest.mark.parametrize("T,H", [(1500, 512), (800, 1536), (700, 2880), (650, 7168), (620, 4104), (3000, 96), (600, 8192)])
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (FP, F32), (F32, F32)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "token"), (True, "channel"), (True, "full"), (False, "one"),
                                       (False, "full"), (False, "token")])
def test_many_rows(T, H, y_dtype, r_dtype, post, gate):
    """Sizes at which rows stream through shared memory, in every combination of their parts."""
    a = make(T, H, y_dtype, r_dtype, post, gate, seed=T)
    kw = dict(scale=0.75, eps=1e-5, off=0.5)
    o = M.block_norm(**a, scale=0.75, eps=1e-5, weight_offset=0.5)
    r, x, rm, xm = R.block_norm(**a, **kw)
    R.close(o.residual, r, rm)
    R.close(o.x, x, xm)
    g = gen(5)
    dx = torch.randn(T, H, generator=g, device="cuda").to(y_dtype)
    dr = torch.randn(T, H, generator=g, device="cuda").to(r_dtype)
    w = dict(post_weight=a["post_weight"], gate=a["gate"], scale=0.5, pre_weight=a["pre_weight"])
    for d in (dr, None):
        b = M.block_norm_backward(dx, d, a["residual"], a["y"], weight_offset=0.5, **w)
        ref = R.block_norm_backward(dx, d, a["residual"], a["y"], off=0.5, **w)
        R.close(b.residual, *ref["residual"])
        R.close(b.y, *ref["y"], steps=3 * R.STEPS)
        steps = 3 * R.STEPS + T // 148 + 64
        R.close(b.pre_weight, *ref["pre_weight"], steps=steps)
        if post:
            R.close(b.post_weight, *ref["post_weight"], steps=steps)
        if gate is not None:
            dg, mag = ref["gate"]
            if gate == "channel":
                dg, mag = dg.sum(0, keepdim=True), mag.sum(0, keepdim=True)
            elif gate == "token":
                dg, mag = dg.sum(1, keepdim=True), mag.sum(1, keepdim=True)
            elif gate == "one":
                dg, mag = dg.sum().view(1, 1), mag.sum().view(1, 1)
            R.close(b.gate, dg, mag, steps=steps)


@pytest.mark.parametrize("T,H", [(2500, 8), (257, 16), (9, 24), (1000, 200), (1301, 128), (130, 256), (5, 250), (700, 257)])
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (FP, F32)])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "token"), (True, "channel"), (True, "full"), (False, "one")])
def test_short_rows(T, H, y_dtype, r_dtype, post, gate):
    """Several rows to a warp, whose last ones do not fill theirs."""
    test_many_rows(T, H, y_dtype, r_dtype, post, gate)


@pytest.mark.parametrize("T,H", [(1, 7168), (64, 640), (1500, 512), (700, 2880), (650, 7168), (600, 8192), (40, 12000),
                                 (300, 96), (700, 1001)])
@pytest.mark.parametrize("y_dtype,r_dtype", [(BF, BF), (BF, F32), (FP, BF), (F32, F32)])
def test_backward_of_the_norm_alone(T, H, y_dtype, r_dtype):
    a = make(T, H, y_dtype, r_dtype, False, None, seed=T + H)
    g = gen(6)
    dx = torch.randn(T, H, generator=g, device="cuda").to(y_dtype)
    dr = torch.randn(T, H, generator=g, device="cuda").to(r_dtype)
    for d in (dr, None):
        b = M.block_norm_backward(dx, d, a["residual"], None, pre_weight=a["pre_weight"], weight_offset=0.5)
        ref = R.block_norm_backward(dx, d, a["residual"], None, pre_weight=a["pre_weight"], off=0.5)
        assert b.y is None and b.gate is None and b.post_weight is None
        R.close(b.residual, *ref["residual"])
        R.close(b.pre_weight, *ref["pre_weight"], steps=3 * R.STEPS + T // 148 + 64)


def test_backward_partial_forms():
    a = make(50, 520, BF, BF, True, "token", seed=6)
    g = gen(7)
    dx, dr = (torch.randn(50, 520, generator=g, device="cuda").to(BF) for _ in range(2))
    # no gradient from behind; only the residual sum (no next norm); only the norm (no block)
    for kw, args in (
            (dict(pre_weight=a["pre_weight"]), (dx, None, a["residual"], a["y"])),
            (dict(post_weight=a["post_weight"], gate=a["gate"]), (None, dr, a["residual"], a["y"])),
            (dict(pre_weight=a["pre_weight"]), (dx, dr, a["residual"], None)),
            (dict(), (None, dr, a["residual"], a["y"]))):
        o = M.block_norm_backward(*args, **kw)
        ref = R.block_norm_backward(*args, **kw)
        R.close(o.residual, *ref["residual"])
        for name in ("y", "pre_weight", "post_weight"):
            got = getattr(o, name)
            if got is not None:
                R.close(got, *ref[name], steps=3 * R.STEPS + 64)
        assert (o.y is None) == (args[3] is None) and (o.pre_weight is None) == (args[0] is None)


def test_backward_against_differences():
    """The gradients along random directions against central differences of the 64-bit forward."""
    T, H, eps, off = 7, 90, 1e-3, 0.25
    a = make(T, H, F32, F32, True, "token", seed=21, wdt=F32)
    g = gen(22)
    dx, dr = (torch.randn(T, H, generator=g, device="cuda") for _ in range(2))
    fwd = M.block_norm(**a, scale=0.8, eps=eps, weight_offset=off)
    o = M.block_norm_backward(dx, dr, fwd.residual, a["y"], post_weight=a["post_weight"], gate=a["gate"], scale=0.8,
                              pre_weight=a["pre_weight"], eps=eps, weight_offset=off)
    p = {k: R.d(v) for k, v in a.items()}
    cg = torch.Generator().manual_seed(3)
    for name in ("y", "residual", "post_weight", "pre_weight", "gate"):
        v = torch.randn(p[name].shape, generator=cg, dtype=torch.float64)
        h = 1e-4
        at = [R.loss(p["y"] if name != "y" else p["y"] + s * h * v,
                     p["residual"] if name != "residual" else p["residual"] + s * h * v,
                     p["post_weight"] if name != "post_weight" else p["post_weight"] + s * h * v,
                     p["gate"] if name != "gate" else p["gate"] + s * h * v, 0.8,
                     p["pre_weight"] if name != "pre_weight" else p["pre_weight"] + s * h * v, eps, off, R.d(dx), R.d(dr))
              for s in (1, -1)]
        num = float(at[0] - at[1]) / (2 * h)
        grad = getattr(o, name).double().cpu()
        # 32-bit gradients: some hundred roundings; differences: h^2 times the third derivative
        tol = 512 * R.U32 * float((grad * v).abs().sum()) + 1e-5 * float((grad * v).norm())
        assert abs(float((grad * v).sum()) - num) <= tol, name


def test_repeated_calls_are_bitwise_equal():
    a = make(1000, 768, BF, BF, True, "channel", seed=9)
    g = gen(10)
    dx, dr = (torch.randn(1000, 768, generator=g, device="cuda").to(BF) for _ in range(2))
    first = None
    for _ in range(3):
        o = M.block_norm_backward(dx, dr, a["residual"], a["y"], post_weight=a["post_weight"], gate=a["gate"],
                                  pre_weight=a["pre_weight"])
        if first is not None:
            assert all(torch.equal(p, q) for p, q in zip(first, o))
        first = o


def test_empty_and_streams():
    w = torch.ones(64, device="cuda")
    o = M.block_norm(torch.empty(0, 64, device="cuda"), torch.empty(0, 64, device="cuda"), pre_weight=w)
    assert o.residual.shape == (0, 64) and o.x.shape == (0, 64)
    b = M.block_norm_backward(torch.empty(0, 64, device="cuda"), None, torch.empty(0, 64, device="cuda"),
                              torch.empty(0, 64, device="cuda"), pre_weight=w, gate=torch.ones(64, device="cuda"))
    assert (b.pre_weight == 0).all() and (b.gate == 0).all() and b.y.shape == (0, 64)
    # a call on another stream orders itself there
    s = torch.cuda.Stream()
    a = make(64, 2048, BF, BF, True, None, seed=30)
    ref = M.block_norm(**a)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        y = a["y"].clone()
        o = M.block_norm(y, a["residual"], post_weight=a["post_weight"], pre_weight=a["pre_weight"])
    s.synchronize()
    assert torch.equal(o.x, ref.x)


def test_refusals():
    y = torch.zeros(4, 32, device="cuda", dtype=BF)
    w = torch.ones(32, device="cuda")
    bad = [
        lambda: M.block_norm(None, None),
        lambda: M.block_norm(None, y),                                    # nothing to compute
        lambda: M.block_norm(y, y[:, :16]),
        lambda: M.block_norm(y.float(), y),                               # a 16-bit residual of a 32-bit y
        lambda: M.block_norm(y.t(), y.t()),                               # rows not contiguous
        lambda: M.block_norm(y, y, pre_weight=w[:16]),
        lambda: M.block_norm(y, y, pre_weight=w.double()),
        lambda: M.block_norm(y, y, gate=w[:5]),
        lambda: M.block_norm(y, y, gate=torch.ones(4, 1, device="cuda").expand(4, 32)),
        lambda: M.block_norm(y, y, pre_weight=w, x_dtype=torch.int8),
        lambda: M.block_norm(y, y, pre_weight=w, out=torch.empty(4, 1, device="cuda", dtype=BF).expand(4, 32)),
        lambda: M.block_norm(y.cpu(), y.cpu()),
        lambda: M.block_norm(y, y.cpu()),
        lambda: M.block_norm(torch.zeros(1, 16385, device="cuda"), None),
        lambda: M.block_norm_backward(None, None, y, y),
        lambda: M.block_norm_backward(y, None, y, y),                     # dx without its weight
        lambda: M.block_norm_backward(None, y, y, None, gate=w),
        lambda: M.block_norm_backward(None, y.half(), y, y),              # dresidual of another type
        lambda: M.block_norm_backward(None, y, y, y.float()),
    ]
    for f in bad:
        with pytest.raises(M.MoEArgumentError):
            f()
