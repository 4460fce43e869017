"""The expert and MXFP4 operators and autograd, on the B200: no gradient is dropped in silence."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200.ops.experts import (  # noqa: E402
    combine_experts, combine_experts_backward, expert_linear, expert_linear_backward, route_experts,
    route_experts_backward)
from loraforge_b200.ops.mxfp4 import expert_linear_mxfp4, mxfp4_quantize  # noqa: E402


def layer():
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(6, 4, generator=g, device="cuda")
    x = torch.randn(6, 64, generator=g, device="cuda").bfloat16()
    w = torch.randn(4, 32, 64, generator=g, device="cuda").bfloat16()
    return logits, x, w, route_experts(logits, 2), torch.randn(12, 32, generator=g, device="cuda").bfloat16()


def leaf(t):
    return t.detach().clone().requires_grad_()


def calls():
    """name -> a call with one argument that requires a gradient."""
    logits, x, w, r, y = layer()
    out, wide = torch.empty_like(y), torch.empty(6, 32, device="cuda").bfloat16()
    mx, mw = mxfp4_quantize(x), mxfp4_quantize(w)
    tables = dict(rows=r.rows)
    return {
        "logits": lambda: route_experts(leaf(logits), 2),
        "logits of the gradient": lambda: route_experts_backward(leaf(logits), r, r.weights),
        "grad_weights": lambda: route_experts_backward(logits, r, leaf(r.weights)),
        "routing.weights": lambda: route_experts_backward(logits, r._replace(weights=leaf(r.weights)), r.weights),
        "out.weights": lambda: route_experts(logits, 2, out=r._replace(weights=leaf(r.weights))),
        "y": lambda: combine_experts(leaf(y), r.weights, r.positions),
        "weights": lambda: combine_experts(y, leaf(r.weights), r.positions),
        "out of the sum": lambda: combine_experts(y, r.weights, r.positions, out=leaf(wide)),
        "grad": lambda: combine_experts_backward(leaf(wide), y, r.weights, r.positions),
        "x": lambda: expert_linear(leaf(x), w, r.offsets, **tables),
        "weight": lambda: expert_linear(x, leaf(w), r.offsets, **tables),
        "out of the products": lambda: expert_linear(x, w, r.offsets, **tables, out=leaf(out)),
        "grad of the products": lambda: expert_linear_backward(leaf(y), x, w, r.offsets, **tables),
        "weight of the gradient": lambda: expert_linear_backward(y, x, leaf(w), r.offsets, **tables),
        "quantised": lambda: mxfp4_quantize(leaf(x)),
        "out in MXFP4": lambda: expert_linear_mxfp4(mx, mw, r.offsets, **tables, out=leaf(out)),
    }


@pytest.mark.parametrize("name", [
    "logits", "logits of the gradient", "grad_weights", "routing.weights", "out.weights", "y", "weights", "out of the sum",
    "grad", "x", "weight", "out of the products", "grad of the products", "weight of the gradient", "quantised", "out in MXFP4"])
def test_tensors_that_require_a_gradient(name):
    call = calls()[name]
    with pytest.raises(ValueError, match="requires a gradient"):
        call()
    with torch.no_grad():  # nothing is lost where autograd does not record
        call()
    with torch.inference_mode():
        call()
