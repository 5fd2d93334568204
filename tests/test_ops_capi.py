"""CPU: the C entries of the operators around the layer refuse what they cannot do, before any CUDA
call, with a status code and a text; their workspace sizes; the Python checks (no kernel is launched)."""
import ctypes

import pytest
import torch

import moe_swarm_b200 as M
from moe_swarm_b200 import _native as N

PTR = 0x10000   # never dereferenced: a refusal comes first


def norm_args(**kw):
    a = N.NormArgs(y=PTR, residual=PTR, pre_weight=PTR, residual_out=PTR, x=PTR, y_stride=64, residual_stride=64,
                   residual_out_stride=64, x_stride=64, rows=2, cols=64, scale=1.0, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def refused(rc, code=N.ERR_ARG):
    assert rc == code and N.last_error()


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=16385), dict(y=None, residual=None), dict(residual_out=None), dict(x=None),
    dict(x_type=7), dict(x_type=N.E4M3), dict(residual_type=N.E4M3), dict(y_type=N.E4M3), dict(y_type=N.FP32),
    dict(pre_weight_type=N.E4M3), dict(gate=PTR, gate_type=N.INT8), dict(y=None, gate=PTR), dict(y=None, pre_weight=None)])
def test_block_norm_refusals(kw):
    refused(N.lib().moe_b200_block_norm(norm_args(**kw), None))


def test_null_arguments():
    lib = N.lib()
    for f in (lib.moe_b200_block_norm, lib.moe_b200_select_experts, lib.moe_b200_select_experts_backward,
              lib.moe_b200_quantize_int8):
        refused(f(None, None))
    refused(lib.moe_b200_block_norm_backward(None, None, 0, None))
    refused(lib.moe_b200_int8_linear(None, None, 0, None))


def back_args(**kw):
    a = N.NormBackwardArgs(dx=PTR, dresidual=PTR, residual=PTR, y=PTR, pre_weight=PTR, dpre_weight=PTR, dresidual_in=PTR,
                           dy=PTR, rows=2, cols=64, scale=1.0, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=(1 << 30) + 1), dict(cols=0), dict(cols=16385), dict(dx=None, dresidual=None), dict(pre_weight=None),
    dict(dpre_weight=None), dict(residual=None), dict(post_weight=PTR), dict(gate=PTR), dict(y=None, post_weight=PTR),
    dict(y=None), dict(y_type=N.FP32), dict(residual_type=N.INT8)])
def test_block_norm_backward_refusals(kw):
    refused(N.lib().moe_b200_block_norm_backward(back_args(**kw), PTR, 1 << 40, None))


def test_workspaces():
    lib = N.lib()
    need = lib.moe_b200_block_norm_backward_workspace_size(2, 64)
    assert need > 0
    refused(lib.moe_b200_block_norm_backward(back_args(), None, 0, None), N.ERR_WORKSPACE)
    refused(lib.moe_b200_block_norm_backward(back_args(), PTR, need - 1, None), N.ERR_WORKSPACE)
    refused(lib.moe_b200_block_norm_backward(back_args(), PTR + 8, need, None))
    for rows, cols in ((-1, 64), (1, 0), (1, 16385)):
        assert lib.moe_b200_block_norm_backward_workspace_size(rows, cols) == 0
    for rows in (0, 1, 7, 300, 5000, 1 << 20):
        for cols in (1, 100, 512, 513, 7168, 16384):
            assert lib.moe_b200_block_norm_backward_workspace_size(rows, cols) > 0
    assert lib.moe_b200_int8_linear_workspace_size(-1, 8, 16, 0) == 0
    assert lib.moe_b200_int8_linear_workspace_size(4, 8, 64, N.BF16) >= 4 * 64 + 4 * 4
    big = lib.moe_b200_int8_linear_workspace_size(1 << 22, 8, 16384, N.BF16)
    assert big > 1 << 36   # sizes beyond 32 bits


def test_empty_calls_need_no_device():
    lib = N.lib()
    assert lib.moe_b200_block_norm(norm_args(rows=0), None) == N.OK
    assert lib.moe_b200_quantize_int8(N.QuantizeArgs(rows=0, cols=8), None) == N.OK
    a = N.LinearArgs(num_tokens=0, out_features=8, in_features=16)
    assert lib.moe_b200_int8_linear(a, None, 0, None) == N.OK


@pytest.mark.parametrize("kw", [
    dict(num_tokens=-1), dict(num_tokens=(1 << 30) + 1), dict(num_experts=0), dict(num_experts=513), dict(top_k=0), dict(top_k=33), dict(n_group=0),
    dict(n_group=33), dict(n_group=5), dict(topk_group=0), dict(topk_group=9), dict(top_k=20, topk_group=1),
    dict(group_score=2), dict(n_group=32, topk_group=32, num_experts=32), dict(score=2), dict(logits_type=N.E4M3),
    dict(bias_type=N.INT8), dict(logits=None), dict(idx=None), dict(weight=None)])
def test_select_refusals(kw):
    a = N.SelectArgs(logits=PTR, bias=PTR, idx=PTR, weight=PTR, logits_stride=128, num_tokens=4, num_experts=128, top_k=4,
                     logits_type=N.FP32, bias_type=N.FP32, n_group=8, topk_group=4, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(N.lib().moe_b200_select_experts(a, None))


@pytest.mark.parametrize("kw", [
    dict(num_tokens=-1), dict(num_tokens=(1 << 30) + 1), dict(num_experts=0), dict(num_experts=513), dict(top_k=0), dict(top_k=33), dict(top_k=9),
    dict(score=5), dict(logits_type=N.INT8), dict(logits=None), dict(idx=None), dict(dweight=None), dict(dlogits=None)])
def test_select_backward_refusals(kw):
    a = N.SelectBackwardArgs(logits=PTR, idx=PTR, dweight=PTR, dlogits=PTR, logits_stride=8, dlogits_stride=8, num_tokens=4,
                             num_experts=8, top_k=2, logits_type=N.FP32, scale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(N.lib().moe_b200_select_experts_backward(a, None))


@pytest.mark.parametrize("kw", [
    dict(num_tokens=-1), dict(num_tokens=(1 << 30) + 1), dict(out_features=(1 << 30) + 1), dict(out_features=0), dict(in_features=8), dict(in_features=40), dict(in_features=131072),
    dict(in_features=65536), dict(x_type=N.E4M3), dict(x_type=N.INT8, swiglu=1), dict(x_type=N.INT8), dict(y_type=N.INT8),
    dict(bias=PTR, bias_type=N.E4M3), dict(x=None), dict(weight=None), dict(weight_scale=None), dict(y=None),
    dict(weight=PTR + 8), dict(weight_stride=72), dict(weight_stride=48),
    dict(x_type=N.INT8, x_scale=PTR, x=PTR + 4), dict(x_type=N.INT8, x_scale=PTR, x_stride=72)])
def test_linear_refusals(kw):
    a = N.LinearArgs(x=PTR, weight=PTR, weight_scale=PTR, y=PTR, x_stride=64, weight_stride=64, y_stride=32, num_tokens=4,
                     out_features=32, in_features=64)
    for k, v in kw.items():
        setattr(a, k, v)
    refused(N.lib().moe_b200_int8_linear(a, PTR, 1 << 40, None))


def test_linear_workspace_refusals():
    a = N.LinearArgs(x=PTR, weight=PTR, weight_scale=PTR, y=PTR, x_stride=64, weight_stride=64, y_stride=32, num_tokens=4,
                     out_features=32, in_features=64)
    lib = N.lib()
    need = lib.moe_b200_int8_linear_workspace_size(4, 32, 64, N.BF16)
    refused(lib.moe_b200_int8_linear(a, None, 0, None), N.ERR_WORKSPACE)
    refused(lib.moe_b200_int8_linear(a, PTR, need - 1, None), N.ERR_WORKSPACE)
    refused(lib.moe_b200_int8_linear(a, PTR + 16, need, None))


def test_python_refuses_cpu_tensors():
    y, w = torch.zeros(2, 32), torch.ones(32)
    q, s = torch.zeros(2, 32, dtype=torch.int8), torch.ones(2)
    for f in (lambda: M.block_norm(y, y, pre_weight=w), lambda: M.block_norm(None, y, pre_weight=w),
              lambda: M.block_norm_backward(y, None, y, y, pre_weight=w), lambda: M.select_experts(y, 2),
              lambda: M.select_experts_backward(s, y, q), lambda: M.quantize_int8(y),
              lambda: M.int8_linear(y, q, s), lambda: M.int8_linear(q, q, s, x_scale=s)):
        with pytest.raises(M.MoEArgumentError):
            f()


def test_structures_match_the_header():
    """Field order and size of the ctypes structures against the C declarations."""
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "moe_b200.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for cls in (N.NormArgs, N.NormBackwardArgs, N.SelectArgs, N.SelectBackwardArgs, N.QuantizeArgs, N.LinearArgs):
        name = cls.__doc__.split()[0]
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
        names = [re.sub(r".*[\s\*]", "", n.strip()) for line in body.split(";") for n in line.split(",") if n.strip()]
        assert names == [n for n, _ in cls._fields_]
        kinds = [k for line in body.split(";") if line.strip() for k in [line.strip()] for _ in k.split(",")]
        want = [ctypes.c_void_p if "*" in k else ctypes.c_int64 if "int64_t" in k else ctypes.c_float if "float" in k
                else ctypes.c_int32 for k in kinds]
        assert want == [t for _, t in cls._fields_]
