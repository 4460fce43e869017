"""The mixture-of-experts example on the B200: a served block and a trained one."""

import gc
import importlib.util
import math
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

PATH = Path(__file__).resolve().parent.parent / "examples" / "moe_lora_layer.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_lora_layer", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens", [1, 37, 700])
def test_served_block(example, tokens):
    from loraforge_b200.ops.experts import route_experts
    from loraforge_b200.ops.mxfp4 import mxfp4_dequantize, mxfp4_quantize

    device = torch.device("cuda", 0)
    H, inner, E, k, slots, rank = 256, 192, 6, 2, 5, 16
    w = example.make_weights(E, H, inner, slots, rank, device, seed=tokens)
    scales = torch.linspace(0.5, 2.0, slots, device=device)
    server = example.MoeLoraServer(w["router"], w["gate_up"], w["down"], k, w["lora_a"], w["lora_b"],
                                   torch.full((slots,), rank, dtype=torch.int32, device=device), scales)
    g = torch.Generator(device=device).manual_seed(3)
    hidden = torch.randn(tokens, H, generator=g, device=device).bfloat16()
    adapters = torch.randint(-1, slots, (tokens,), generator=g, device=device).to(torch.int32)
    out = server(hidden, adapters)
    # The same steps on the dequantised weights in 64 bits, with the activations' roundings to 4 bits.
    r = route_experts(hidden @ w["router"].T, k)
    up, down = (mxfp4_dequantize(q, torch.float32).double() for q in (server.gate_up, server.down))
    h4 = mxfp4_dequantize(mxfp4_quantize(hidden), torch.float32).double()
    want = torch.zeros(tokens, H, dtype=torch.float64, device=device)
    for j in range(k):
        e = r.experts[:, j].long()
        mid = torch.einsum("th,tih->ti", h4, up[e]).bfloat16()
        mid4 = mxfp4_dequantize(mxfp4_quantize(example.swiglu(mid)), torch.float32).double()
        want += r.weights[:, j, None].double() * torch.einsum("ti,thi->th", mid4, down[e])
    for t in range(tokens):
        s = int(adapters[t])
        if s >= 0:
            want[t] += scales[s].double() * (w["lora_b"][s].double() @ (w["lora_a"][s].double() @ hidden[t].double()))
    # Three roundings to BF16 (2^-9 each); a middle value at a tie may fall to the other 4-bit neighbour.
    assert (out.double() - want).norm() <= 2.0**-6 * want.norm()


def test_gradients_of_the_block(example):
    device = torch.device("cuda", 0)
    T, H, inner, E, k = 60, 64, 96, 5, 2
    w = example.make_weights(E, H, inner, 1, 16, device, seed=5)
    g = torch.Generator(device=device).manual_seed(6)
    hidden = torch.randn(T, H, generator=g, device=device).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (hidden, w["router"], w["gate_up"], w["down"])]
    out = example.moe_block(*leaves, k)
    grad = torch.randn(T, H, generator=g, device=device).bfloat16()
    out.backward(grad)
    # 64-bit autograd over the same experts.
    x, router, gate_up, down = (t.detach().double().requires_grad_() for t in leaves)
    from loraforge_b200.ops.experts import route_experts

    experts = route_experts(hidden @ w["router"].T, k).experts.long()
    p = torch.gather(torch.softmax(x @ router.T, 1), 1, experts)
    p = p / p.sum(1, keepdim=True)
    want = sum(p[:, j, None] * torch.einsum("ti,thi->th", example.swiglu(torch.einsum("th,tih->ti", x, gate_up[experts[:, j]])),
                                            down[experts[:, j]]) for j in range(k))
    want.backward(grad.double())
    assert (out.double() - want).norm() <= 2.0**-6 * want.norm()
    for got, ref in zip(leaves, (x, router, gate_up, down)):
        # A handful of roundings to BF16 (2^-9 relative each) along each path.
        assert (got.grad.double() - ref.grad).norm() <= 2.0**-5 * ref.grad.norm()


def test_main_trains(example, capsys):
    example.main()
    losses = [float(line.split()[-1]) for line in capsys.readouterr().out.splitlines() if line.startswith("training")]
    assert len(losses) == 5 and losses[-1] < losses[0] and all(math.isfinite(v) for v in losses)


def test_training_steps_keep_no_memory(example):
    # Without the cycle collector: what a step's graph holds goes with it.
    device = torch.device("cuda", 0)
    w = example.make_weights(5, 64, 96, 1, 16, device, seed=5)
    leaves = [w[n].clone().requires_grad_() for n in ("router", "gate_up", "down")]
    hidden = torch.randn(600, 64, device=device).bfloat16()
    held = []
    gc.collect()
    gc.disable()
    try:
        for _ in range(6):
            example.moe_block(hidden, *leaves, 2).float().square().mean().backward()
            for leaf in leaves:
                leaf.grad = None
            held.append(torch.cuda.memory_allocated())
    finally:
        gc.enable()
    assert len(set(held[1:])) == 1, held


def test_changed_routing_weights_are_noticed(example):
    logits = torch.randn(5, 4, device="cuda").requires_grad_()
    weights = example._Route.apply(logits, 2)[0]
    loss = weights.sum()
    with torch.no_grad():
        weights.mul_(2.0)  # the gradient's formula reads them
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
