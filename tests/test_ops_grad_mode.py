"""CPU: the operators around the layer record no graph, and say so instead of dropping a gradient."""
import pytest
import torch

import moe_swarm_b200 as M


def leaf(*shape, **kw):
    return torch.zeros(*shape, requires_grad=True, **kw)


CALLS = [
    lambda: M.block_norm(leaf(2, 8), None),
    lambda: M.block_norm(torch.zeros(2, 8), leaf(2, 8)),
    lambda: M.block_norm(torch.zeros(2, 8), None, pre_weight=leaf(8)),
    lambda: M.block_norm(torch.zeros(2, 8), None, post_weight=leaf(8)),
    lambda: M.block_norm(torch.zeros(2, 8), None, gate=leaf(1, 8)),
    lambda: M.block_norm_backward(leaf(2, 8), None, torch.zeros(2, 8), None, pre_weight=torch.zeros(8)),
    lambda: M.block_norm_backward(None, leaf(2, 8), torch.zeros(2, 8), None),
    lambda: M.select_experts(leaf(2, 8), 2),
    lambda: M.select_experts(torch.zeros(2, 8), 2, bias=leaf(8)),
    lambda: M.select_experts_backward(leaf(2, 2), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32)),
    lambda: M.quantize_int8(leaf(2, 16)),
    lambda: M.int8_linear(leaf(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4)),
    lambda: M.int8_linear(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), leaf(4)),
    lambda: M.int8_linear(torch.zeros(2, 16), torch.zeros(4, 16, dtype=torch.int8), torch.ones(4), bias=leaf(4)),
]


@pytest.mark.parametrize("call", CALLS)
def test_a_lost_gradient_is_an_error(call):
    with pytest.raises(M.MoEArgumentError, match="records no graph"):
        call()
    # the same call without gradients goes on to the next check: there is no CPU path
    for off in (torch.no_grad, torch.inference_mode):
        with off(), pytest.raises(M.MoEArgumentError, match="CUDA"):
            call()
