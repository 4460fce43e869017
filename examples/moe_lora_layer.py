"""A feed-forward block with mixture-of-experts weights and LoRA adapters, served and trained.

Serving (``MoeLoraServer``): the experts are kept in MXFP4 and the requests' adapters in 16 bits
beside them.  A batch goes router -> quantised activations -> gate/up product -> SwiGLU ->
down product -> weighted sum, and every token's adapter adds ``scale * B (A h)`` to the block's
output through the grouped shrink/expand.  The tables stay on the device, so a step can be
captured in a CUDA graph.

Training (``moe_block``): the same block with BF16 experts as autograd functions over the
explicit gradients of the router, the products and the sum.

    python examples/moe_lora_layer.py
"""

import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from loraforge_b200.ops.experts import (  # noqa: E402
    ExpertRouting, combine_experts, combine_experts_backward, expert_linear, expert_linear_backward, route_experts,
    route_experts_backward)
from loraforge_b200.ops.fused import lora_shrink_expand  # noqa: E402
from loraforge_b200.ops.grouping import group_tokens  # noqa: E402
from loraforge_b200.ops.mxfp4 import expert_linear_mxfp4, mxfp4_quantize  # noqa: E402


def swiglu(gate_up):
    gate, up = gate_up.chunk(2, dim=1)
    return torch.nn.functional.silu(gate) * up


class MoeLoraServer:
    """One block for serving: MXFP4 experts and a slab of resident adapters."""

    def __init__(self, router, gate_up, down, top_k: int, lora_a, lora_b, ranks, scales):
        """``router`` [E, H]; ``gate_up`` [E, 2 I, H] and ``down`` [E, H, I] in any floating type;
        ``lora_a`` [slots, r, H], ``lora_b`` [slots, H, r] (BF16), ``ranks`` and ``scales`` [slots]."""
        self.router, self.top_k = router, top_k
        self.gate_up, self.down = mxfp4_quantize(gate_up.contiguous()), mxfp4_quantize(down.contiguous())
        slots, width, rank = lora_b.shape
        device = router.device
        self.slots = slots
        self.lora = dict(
            b_offsets=torch.arange(slots, dtype=torch.int64, device=device) * width * rank,
            b_strides=torch.full((slots,), rank, dtype=torch.int32, device=device), ranks=ranks, scales=scales,
            slice_offsets=torch.tensor([0, width], dtype=torch.int32, device=device),
        )
        self.a, self.b = lora_a, lora_b.reshape(-1)

    def __call__(self, hidden, adapters):
        """``hidden`` BF16 [T, H], ``adapters`` int32 [T] (-1: none) -> BF16 [T, H]."""
        routing = route_experts(hidden @ self.router.T, self.top_k)
        mid = expert_linear_mxfp4(mxfp4_quantize(hidden), self.gate_up, routing.offsets, rows=routing.rows)
        rows = expert_linear_mxfp4(mxfp4_quantize(swiglu(mid)), self.down, routing.offsets)
        out = combine_experts(rows, routing.weights, routing.positions)
        groups = group_tokens(adapters, self.slots, chunk=16)
        lora_shrink_expand(hidden, self.a, self.b, out, segment_indptr=groups.segment_indptr,
                           segment_slots=groups.segment_slots, token_indices=groups.token_indices,
                           segment_count=groups.segment_count, **self.lora)
        return out


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_k):
        routing = route_experts(logits.detach(), top_k)
        # Saved, not kept on ctx: an output there would hold its own graph, and changes of it go unseen.
        ctx.save_for_backward(logits, *routing)
        ctx.mark_non_differentiable(*routing[1:])
        return tuple(routing)

    @staticmethod
    def backward(ctx, grad_weights, *_):
        logits, *routing = (t.detach() for t in ctx.saved_tensors)
        return route_experts_backward(logits, ExpertRouting(*routing), grad_weights.contiguous()), None


class _ExpertLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, rows, positions):
        ctx.save_for_backward(x, weight, offsets, rows, positions)
        return expert_linear(x.detach(), weight.detach(), offsets, rows=rows)

    @staticmethod
    def backward(ctx, grad):
        x, weight, offsets, rows, positions = ctx.saved_tensors
        grad_x, grad_weight = expert_linear_backward(grad.contiguous(), x.detach(), weight.detach(), offsets, rows=rows)
        if rows is not None:  # by row: a token's rows are added up
            grad_x = combine_experts(grad_x, None, positions)
        return grad_x, grad_weight, None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, positions):
        ctx.save_for_backward(y, weights, positions)
        return combine_experts(y.detach(), weights.detach(), positions)

    @staticmethod
    def backward(ctx, grad):
        y, weights, positions = ctx.saved_tensors
        return (*combine_experts_backward(grad.contiguous(), y.detach(), weights.detach(), positions), None)


def moe_block(hidden, router, gate_up, down, top_k: int):
    """The block for training: differentiable in all four tensors (BF16)."""
    weights, _, offsets, rows, positions = _Route.apply(hidden @ router.T, top_k)
    mid = swiglu(_ExpertLinear.apply(hidden, gate_up, offsets, rows, positions))
    return _Combine.apply(_ExpertLinear.apply(mid, down, offsets, None, positions), weights, positions)


def make_weights(experts, hidden, inner, slots, rank, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return (torch.randn(shape, generator=g, device=device) / math.sqrt(shape[-1])).bfloat16()

    return dict(router=normal(experts, hidden), gate_up=normal(experts, 2 * inner, hidden),
                down=normal(experts, hidden, inner), lora_a=normal(slots, rank, hidden),
                lora_b=normal(slots, hidden, rank))


def main():
    device = torch.device("cuda", 0)
    H, inner, E, k, slots, rank, T = 1024, 1024, 16, 4, 8, 16, 256
    w = make_weights(E, H, inner, slots, rank, device)
    g = torch.Generator(device=device).manual_seed(1)
    server = MoeLoraServer(w["router"], w["gate_up"], w["down"], k, w["lora_a"], w["lora_b"],
                           torch.full((slots,), rank, dtype=torch.int32, device=device),
                           torch.full((slots,), 2.0, device=device))
    for tokens in (1, T):
        hidden = torch.randn(tokens, H, generator=g, device=device).bfloat16()
        adapters = torch.randint(-1, slots, (tokens,), generator=g, device=device).to(torch.int32)
        out = server(hidden, adapters)
        print(f"served {tokens} tokens over {E} experts, {slots} adapters: output rms {out.float().square().mean().sqrt():.3f}")
    leaves = [w[n].clone().requires_grad_() for n in ("router", "gate_up", "down")]
    hidden = torch.randn(T, H, generator=g, device=device).bfloat16()
    target = torch.randn(T, H, generator=g, device=device)
    optimizer = torch.optim.SGD(leaves, lr=20.0)
    for step in range(5):
        loss = (moe_block(hidden, *leaves, k).float() - target).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        print(f"training step {step}: loss {loss.item():.4f}")


if __name__ == "__main__":
    main()
