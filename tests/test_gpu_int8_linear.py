"""GPU: 8-bit quantisation and the 8-bit linear layer against exact integer and 64-bit forms."""
import pytest
import torch

import moe_swarm_b200 as M
from tests import _ops_ref as R

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def codes(rows, cols, seed, full=False):
    g = torch.Generator().manual_seed(seed)
    if full:
        return torch.randint(-128, 128, (rows, cols), generator=g, dtype=torch.int8)
    return torch.clamp(torch.round(torch.randn(rows, cols, generator=g) * 36), -127, 127).to(torch.int8)


def exact(q, w, sx, sw, bias=None):
    acc = q.double().cpu() @ w.double().cpu().t()      # integers below 2^53: exact
    y = acc * sx.double().cpu()[:, None] * sw.double().cpu()[None]
    mag = y.abs()
    if bias is not None:
        y = y + bias.double().cpu()
        mag = mag + bias.double().cpu().abs()
    return y, mag


def run_exact(T, N, K, out=BF, bias=None, seed=0, full=False, w_pad=0, x_pad=0):
    g = torch.Generator().manual_seed(seed + 1)
    q = codes(T, K + x_pad, seed, full).cuda()[:, :K]
    w = codes(N, K + w_pad, seed + 9, full).cuda()[:, :K]
    sx, sw = (torch.rand(n, generator=g).cuda() + 0.1 for n in (T, N))
    b = None if bias is None else torch.randn(N, generator=g).to(bias).cuda() * 50
    y = M.int8_linear(q, w, sw, x_scale=sx, bias=b, out_dtype=out)
    ref, mag = exact(q, w, sx, sw, b)
    assert y.shape == (T, N) and y.dtype == out
    R.close(y, ref, mag, steps=8)     # integer to 32 bits, three products, one sum


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 33, 64, 65, 127, 128, 129, 200, 257, 300, 513, 700])
@pytest.mark.parametrize("N,K", [(1, 16), (64, 128), (100, 144), (129, 1040), (300, 272), (512, 2048), (1001, 640)])
def test_int8_input(T, N, K):
    run_exact(T, N, K, out=F32, seed=T + N + K)


@pytest.mark.parametrize("out", [BF, FP, F32])
@pytest.mark.parametrize("bias", [None, BF, F32])
@pytest.mark.parametrize("T", [3, 70, 600])
def test_types_and_bias(T, out, bias):
    run_exact(T, 264, 272, out=out, bias=bias, seed=5)
    run_exact(T, 263, 272, out=out, bias=bias, seed=6)


@pytest.mark.parametrize("T", [1, 2, 40, 300])
def test_extreme_codes_and_long_sums(T):
    run_exact(T, 96, 4096, out=F32, full=True, seed=3)
    # the largest sums that 32-bit integers hold: 131056 * 128 * 128 < 2^31
    K = 131056
    q = torch.full((T, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((40, K), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(max(T, 40), device="cuda")
    y = M.int8_linear(q, w, one[:40], x_scale=one[:T], out_dtype=F32)
    assert (y == float(K * 128 * 128)).all()


@pytest.mark.parametrize("T", [1, 2, 5, 150, 600])
def test_row_pitch(T):
    run_exact(T, 130, 208, out=F32, w_pad=16, x_pad=48, seed=8)
    q, w = codes(T, 64, 1).cuda(), codes(50, 64, 2).cuda()
    sx, sw = torch.ones(T, device="cuda"), torch.ones(50, device="cuda")
    for pad in (1, 14):
        buf = torch.full((T, 50 + pad), 9.0, device="cuda", dtype=BF)
        y = M.int8_linear(q, w, sw, x_scale=sx, out=buf[:, :50])
        ref, mag = exact(q, w, sx, sw)
        R.close(y, ref, mag, steps=8)
        assert (buf[:, 50:] == 9.0).all()


@pytest.mark.parametrize("rows,cols", [(1, 7168), (3, 16), (5, 17), (70, 1000), (2, 1024), (2, 1025), (9, 8192),
                                       (1, 32768), (300, 64), (4, 5001)])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("swiglu", [False, True])
def test_quantize(rows, cols, dtype, swiglu):
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(rows, 2 * cols if swiglu else cols, generator=g) * 3).to(dtype).cuda()
    q, s = M.quantize_int8(x, swiglu=swiglu)
    v = R.swiglu(x) if swiglu else x.double().cpu()
    ref, scale, margin = R.quantize(v)
    # silu: exponential, quotient, product; then one quotient
    R.close(s, scale, scale, steps=16)
    err = 16 * R.U32 * 127 * 2       # a code may differ only this close to a rounding boundary
    diff = (q.double().cpu() - ref).abs()
    assert diff.max() <= 1 and (diff[margin > err] == 0).all()
    assert q.abs().max() <= 127


def test_quantize_special_rows():
    x = torch.randn(8, 100, device="cuda")
    x[1] = 0
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4] *= 1e-39          # subnormal
    x[5] = 3e38
    q, s = M.quantize_int8(x)
    assert (q[1] == 0).all() and s[1] > 0
    assert torch.isnan(s[2]) and torch.isnan(s[3])
    assert torch.isfinite(s[[0, 1, 4, 5, 6, 7]]).all() and (q[5] == 127).all()
    w, sw = codes(20, 112, 1).cuda(), torch.ones(20, device="cuda")
    y = M.int8_linear(torch.nn.functional.pad(x, (0, 12)), w, sw)
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    assert (y[1] == 0).all() and torch.isfinite(y[[0, 1, 4, 6, 7]]).all()


@pytest.mark.parametrize("T", [1, 2, 9, 64, 80, 150, 600])
@pytest.mark.parametrize("N,K", [(96, 272), (1000, 1024)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("swiglu", [False, True])
def test_quantised_in_the_call(T, N, K, dtype, swiglu):
    """Equals the two calls apart, and the 64-bit product of the codes that quantize_int8 gives."""
    g = torch.Generator().manual_seed(T + N)
    x = torch.randn(T, 2 * K if swiglu else K, generator=g).to(dtype).cuda()
    w, sw = codes(N, K, 4).cuda(), torch.rand(N, generator=g).cuda()
    y = M.int8_linear(x, w, sw, swiglu=swiglu)
    assert y.dtype == dtype
    q, s = M.quantize_int8(x, swiglu=swiglu)
    assert torch.equal(y, M.int8_linear(q, w, sw, x_scale=s, out_dtype=dtype))
    ref, mag = exact(q, w, s, sw)
    R.close(y, ref, mag, steps=8)


def test_strided_float_input():
    x = torch.randn(37, 200, device="cuda").to(BF)
    w, sw = codes(65, 96, 4).cuda(), torch.rand(65, device="cuda")
    for off in (0, 1, 8):
        v = x[:, off:off + 96]
        assert torch.equal(M.int8_linear(v, w, sw), M.int8_linear(v.contiguous(), w, sw))


def test_streams_and_repeats():
    q, w = codes(300, 512, 1).cuda(), codes(700, 512, 2).cuda()
    sx, sw = torch.rand(300, device="cuda"), torch.rand(700, device="cuda")
    ref = M.int8_linear(q, w, sw, x_scale=sx)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(M.int8_linear(q[: 300 - 20 * i], w, sw, x_scale=sx[: 300 - 20 * i]))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert torch.equal(o, ref[: 300 - 20 * i])


def test_graph_capture():
    x = torch.randn(20, 512, device="cuda").to(BF)
    w, sw = codes(256, 512, 2).cuda(), torch.rand(256, device="cuda")
    ref = M.int8_linear(x, w, sw)
    out = torch.empty_like(ref)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        M.int8_linear(x, w, sw, out=out)
    x2 = torch.randn(20, 512, device="cuda").to(BF)
    want = M.int8_linear(x2, w, sw)
    x.copy_(x2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda", dtype=BF)
    q, s = torch.zeros(4, 64, device="cuda", dtype=torch.int8), torch.ones(4, device="cuda")
    w, sw = torch.zeros(8, 64, device="cuda", dtype=torch.int8), torch.ones(8, device="cuda")
    bad = [
        lambda: M.int8_linear(x, w[:, :48], sw), lambda: M.int8_linear(x[:, :40], w[:, :40], sw),   # K % 16
        lambda: M.int8_linear(q, w, sw), lambda: M.int8_linear(x, w, sw, x_scale=s),
        lambda: M.int8_linear(q, w, sw, x_scale=s[:3]), lambda: M.int8_linear(x, w, sw[:7]),
        lambda: M.int8_linear(x, w, sw.half()), lambda: M.int8_linear(x, w.float(), sw),
        lambda: M.int8_linear(q[:, :32], w[:, 8:40], sw, x_scale=s),        # weight rows off 16 bytes
        lambda: M.int8_linear(q[:, 8:40], w[:, :32], sw, x_scale=s),        # x rows off 16 bytes
        lambda: M.int8_linear(q, w[:, :32], sw, x_scale=s, swiglu=True),
        lambda: M.int8_linear(x, w, sw, out_dtype=torch.int8),
        lambda: M.int8_linear(x, w, sw, bias=sw[:5]),
        lambda: M.int8_linear(x, w, sw, out=torch.empty(4, 9, device="cuda")),
        lambda: M.int8_linear(x.cpu(), w, sw), lambda: M.int8_linear(x, w.cpu(), sw),
        lambda: M.quantize_int8(x[:, :33], swiglu=True), lambda: M.quantize_int8(q),
        lambda: M.quantize_int8(torch.zeros(1, 32769, device="cuda")),
    ]
    for f in bad:
        with pytest.raises(M.MoEArgumentError):
            f()


def exact_codes(x):
    """Codes and scales in 64 bits."""
    v = x.double()
    scale = torch.clamp(v.abs().amax(dim=1) * (1.0 / 127.0), min=2.0 ** -126)
    return torch.round(v / scale[:, None]), scale


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("T,K", [(3000, 2048), (700, 7168), (40, 20000), (900, 1001), (5000, 40), (30, 8192)])
def test_codes_are_those_of_64_bits(T, K, dtype):
    """Millions of codes, thousands of ties among them, without one on the other side."""
    g = torch.Generator(device="cuda").manual_seed(T + K)
    x = (torch.randn(T, K, generator=g, device="cuda") * 3).to(dtype)
    q, s = M.quantize_int8(x)
    ref, scale = exact_codes(x)
    assert torch.equal(q.double(), ref)
    assert ((s.double() - scale).abs() <= 2.0 ** -23 * scale).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("size", [6e37, 1e-36, 3e-39])
def test_codes_of_large_and_small_values(dtype, size):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(500, 1024, generator=g, device="cuda").clamp(-4, 4) * size).to(dtype)
    q, s = M.quantize_int8(x)
    ref, scale = exact_codes(x)
    assert torch.equal(q.double(), ref)
    assert ((s.double() - scale).abs() <= 2.0 ** -23 * scale).all()


@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_few_tokens_codes_are_those_of_64_bits(T, dtype):
    """One or two tokens are quantised inside the product: an identity for weights returns their codes."""
    K = 2048
    w, one = torch.eye(K, dtype=torch.int8, device="cuda"), torch.ones(K, device="cuda")
    for seed in range(40):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = (torch.randn(T, K, generator=g, device="cuda") * 3).to(dtype)
        y = M.int8_linear(x, w, one, out_dtype=F32)
        ref, scale = exact_codes(x)
        assert torch.equal(torch.round(y.double() / scale[:, None]), ref)
