"""The feed-forward half of a transformer block with routed experts, on this package's operators.

    residual, x = block_norm(attention output, residual)        norm in bf16 and in e4m3 blocks
    ids, w      = select_experts(x @ router)                     256 experts, 8 groups, 8 chosen
    routed      = run_routed(ids, w, x in e4m3)                  the FP8 expert layer
    shared      = int8_linear(swiglu(int8_linear(x)))            the dense expert in 8-bit integers
    residual, x = block_norm(routed + shared, residual)          gate, sum and the next block's norm

``python examples/moe_block.py [--tokens T] [--experts E]`` builds a block with random weights, runs
it, computes the gradients of its router and of the norms at its end for random gradients of its results, moves
the selection's bias once, and prints what it took.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import moe_swarm_b200 as M  # noqa: E402
from moe_swarm_b200 import workload as W  # noqa: E402

TOP_K, N_GROUP, TOPK_GROUP, ROUTED_SCALE = 8, 8, 4, 2.5
SHARED = 2048   # width of the dense expert


class MoEBlock:
    """Weights of one block (random) and its passes.  Routed experts 0 .. n_experts - 1 of 256 are
    held here; tokens that choose others get those experts' share from elsewhere (or not at all)."""

    def __init__(self, n_experts: int = 32, seed: int = 0, device: str = "cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape, std=1.0):
            return torch.randn(*shape, generator=g, device=device) * std

        self.norm_weight = (1 + randn(M.H, std=0.1)).bfloat16()        # before the block
        self.out_weight = (1 + randn(M.H, std=0.1)).bfloat16()         # on its output
        self.next_weight = (1 + randn(M.H, std=0.1)).bfloat16()        # before the next block
        self.out_gate = torch.sigmoid(randn(1, M.H)).bfloat16()
        self.router = randn(M.E_GLOBAL, M.H, std=M.H ** -0.5).bfloat16()
        self.balance = torch.zeros(M.E_GLOBAL, device=device)
        w13, s13, w2, s2 = [], [], [], []
        for _ in range(n_experts):
            q, s = W.quantize_blocks(randn(2 * M.I, M.H, std=0.02))
            w13.append(q), s13.append(s)
            q, s = W.quantize_blocks(randn(M.H, M.I, std=0.02))
            w2.append(q), s2.append(s)
        self.experts = [torch.stack([t.view(torch.uint8) for t in w13]).view(torch.float8_e4m3fn), torch.stack(s13),
                        torch.stack([t.view(torch.uint8) for t in w2]).view(torch.float8_e4m3fn), torch.stack(s2)]
        self.up, self.up_scale = M.quantize_int8(randn(2 * SHARED, M.H, std=0.02))
        self.down, self.down_scale = M.quantize_int8(randn(M.H, SHARED, std=0.02))

    def forward(self, y, residual):
        """y: the attention's output, residual: the stream before it (both bf16 [T, 7168]).
        Returns (stream behind this block, input of the next, what the backward pass needs)."""
        r1, x, _ = M.block_norm(y, residual, pre_weight=self.norm_weight)
        x8 = M.block_norm(None, r1, pre_weight=self.norm_weight, x_dtype=torch.float8_e4m3fn)
        logits = x.float() @ self.router.float().t()
        sel = M.select_experts(logits, TOP_K, bias=self.balance, n_group=N_GROUP, topk_group=TOPK_GROUP,
                               scale=ROUTED_SCALE, counts=True)
        routed = M.run_routed(sel.idx, sel.w, x8.x, x8.x_scale, *self.experts, 0)
        h = M.int8_linear(x, self.up, self.up_scale)
        shared = M.int8_linear(h, self.down, self.down_scale, swiglu=True)
        out = routed + shared
        r2, x2, _ = M.block_norm(out, r1, post_weight=self.out_weight, gate=self.out_gate,
                                 pre_weight=self.next_weight)
        return r2, x2, (x, logits, sel, out, r2)

    def rebalance(self, counts, step: float = 1e-3):
        """Moves the selection's bias toward experts that were chosen less often than the mean."""
        n = counts.float()
        self.balance += step * torch.sign(n.mean() - n)

    def backward(self, saved, dx2, dr2, dw):
        """Gradients of the output norms and of the router from those of the block's results (dx2,
        dr2) and of the selection's weights (dw, as the experts' outputs give them)."""
        x, logits, sel, out, r2 = saved
        norms = M.block_norm_backward(dx2, dr2, r2, out, post_weight=self.out_weight, gate=self.out_gate,
                                      pre_weight=self.next_weight)
        dlogits = M.select_experts_backward(dw, logits, sel.idx, scale=ROUTED_SCALE)
        return norms, dlogits.t() @ x.float()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--experts", type=int, default=32)
    a = ap.parse_args(argv)
    block = MoEBlock(a.experts)
    for T in (1, a.tokens):
        y, residual = (torch.randn(T, M.H, device="cuda").bfloat16() for _ in range(2))
        for _ in range(3):
            r2, x2, saved = block.forward(y, residual)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        start.record()
        for _ in range(10):
            r2, x2, saved = block.forward(y, residual)
        end.record()
        torch.cuda.synchronize()
        print(f"T={T}: {start.elapsed_time(end) * 100:.1f} us a block, |x| {x2.float().norm(dim=1).mean().item():.2f}")
    block.rebalance(saved[2].counts)
    norms, drouter = block.backward(saved, torch.randn_like(x2), torch.randn_like(r2), torch.randn_like(saved[2].w))
    print(f"|d router| {drouter.norm().item():.3f}, |d out_weight| {norms.post_weight.norm().item():.3f}, "
          f"|d gate| {norms.gate.norm().item():.3f}, busiest expert {int(saved[2].counts.max())} tokens")
    assert M.operator_status() == 0 and M.device_status() == 0


if __name__ == "__main__":
    main()
