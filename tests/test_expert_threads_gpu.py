"""The expert operators called from several host threads at once, each on a stream of its own."""

import math
from concurrent.futures import ThreadPoolExecutor

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


def layer(seed, tokens):
    """Everything a layer computes on a batch of its own."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(tokens, 6, generator=g, device="cuda")
    x = torch.randn(tokens, 128, generator=g, device="cuda").bfloat16()
    w = (torch.randn(6, 136, 128, generator=g, device="cuda") / math.sqrt(128)).bfloat16()
    r = route_experts(logits, 2)
    y = expert_linear(x, w, r.offsets, rows=r.rows)
    out = combine_experts(y, r.weights, r.positions)
    grad_y, grad_weights = combine_experts_backward(out, y, r.weights, r.positions)
    y4 = expert_linear_mxfp4(mxfp4_quantize(x), mxfp4_quantize(w), r.offsets, rows=r.rows)
    return [out, y4, route_experts_backward(logits, r, grad_weights),
            *expert_linear_backward(grad_y, x, w, r.offsets, rows=r.rows)]


def test_threads_with_streams_of_their_own():
    sizes = [3, 40, 700, 5]  # few rows, a split contraction, pairs

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results = [layer(i, sizes[i]) for _ in range(5)]
        stream.synchronize()
        return results

    with ThreadPoolExecutor(len(sizes)) as pool:
        found = list(pool.map(work, range(len(sizes))))
    for i, results in enumerate(found):
        want = layer(i, sizes[i])
        assert all(torch.equal(a, b) for result in results for a, b in zip(result, want))
