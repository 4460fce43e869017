"""What the expert operators refuse, by kind of object and by value, on the B200."""

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200.ops.experts import (  # noqa: E402
    combine_experts, expert_linear, expert_linear_backward, route_experts, route_experts_backward)


def test_tables_that_are_not_tensors():
    logits = torch.randn(4, 8, device="cuda")
    r = route_experts(logits, 2)
    with pytest.raises(TypeError, match="out.weights must be a torch.Tensor"):
        route_experts(logits, 2, out=tuple(r))
    x = torch.randn(4, 64, device="cuda").bfloat16()
    w = torch.randn(8, 16, 64, device="cuda").bfloat16()
    grad = torch.zeros(8, 16, device="cuda").bfloat16()
    for rows in (r.rows.cpu().numpy(), r.rows.tolist()):
        with pytest.raises(TypeError, match="rows must be a torch.Tensor"):
            expert_linear(x, w, r.offsets, rows=rows)
        with pytest.raises(TypeError, match="rows must be a torch.Tensor"):
            expert_linear_backward(grad, x, w, r.offsets, rows=rows)
    for table in (r.positions.cpu().numpy(), r.positions.tolist()):
        with pytest.raises(TypeError, match="positions must be a torch.Tensor"):
            combine_experts(x, None, table)


@pytest.mark.parametrize("scale", [1e-50, 1e-46, 3.5e38, -1.0, float("nan")])
def test_scales_that_fp32_does_not_hold(scale):
    logits = torch.randn(4, 8, device="cuda")
    r = route_experts(logits, 2)
    with pytest.raises(ValueError, match="scale must be positive and finite"):
        route_experts(logits, 2, scale=scale)
    with pytest.raises(ValueError, match="scale must be positive and finite"):
        route_experts_backward(logits, r, r.weights, scale=scale)
