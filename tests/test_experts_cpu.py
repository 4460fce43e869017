"""The expert and MXFP4 entry points refuse bad sizes on the host, before any device work."""

from concurrent.futures import ThreadPoolExecutor

import pytest

from loraforge_b200 import _native


def call(entry, args):
    """In a thread of its own: the library keeps its last error message by thread."""
    with ThreadPoolExecutor(1) as pool:
        pool.submit(_native.call, entry, *args).result()


@pytest.mark.parametrize("entry,args,match", [
    ("lf_route_experts", (0, 16, 8, 4, 8, 9, 1, 1.0, 16, 16, 16, 16, 16, 16, 99, None), "top_k"),
    ("lf_route_experts", (7, 16, 8, 4, 8, 2, 1, 1.0, 16, 16, 16, 16, 16, 16, 99, None), "element type"),
    ("lf_route_experts", (0, 16, 8, 4, 8, 2, 1, 0.0, 16, 16, 16, 16, 16, 16, 99, None), "scale"),
    ("lf_route_experts", (0, 16, 8, 4, 8, 2, 1, float("nan"), 16, 16, 16, 16, 16, 16, 99, None), "scale"),
    ("lf_route_experts", (0, 16, 7, 4, 8, 2, 1, 1.0, 16, 16, 16, 16, 16, 16, 99, None), "stride"),
    ("lf_route_experts", (0, None, 8, 4, 8, 2, 1, 1.0, 16, 16, 16, 16, 16, 16, 99, None), "null"),
    ("lf_route_experts", (0, 16, 8, 100, 8, 2, 1, 1.0, 16, 16, 16, 16, 16, None, 0, None), "workspace"),
    ("lf_route_experts_backward", (0, 16, 8, 16, 16, 16, 1, 4, 8, 2, 1, 1.0, 16, 8, None), "stride"),
    ("lf_combine_experts", (0, 16, 8, 4, 16, 16, 2, 33, 8, 16, 8, None), "top_k"),
    ("lf_combine_experts", (0, 16, 7, 4, 16, 16, 2, 2, 8, 16, 8, None), "stride"),
    ("lf_combine_experts_backward", (0, 16, 8, 16, 8, 4, 16, 16, 2, 2, 8, 16, 7, 16, None), "stride"),
    ("lf_expert_linear", (0, 16, 64, 4, None, 16, 4096, 64, 16, 1, 4, 64, 64, 16, 64, None, 0, None), "BF16 or FP16"),
    ("lf_expert_linear", (2, 16, 64, 4, None, 16, 4096, 64, 16, 1, 4, 60, 64, 16, 64, None, 0, None), "multiples of 8"),
    ("lf_expert_linear", (2, 24, 64, 4, None, 16, 4096, 64, 16, 1, 4, 64, 64, 16, 64, None, 0, None), "16-byte"),
    ("lf_expert_linear", (2, 16, 64, 3, None, 16, 4096, 64, 16, 1, 4, 64, 64, 16, 64, None, 0, None), "rows"),
    ("lf_expert_linear_input_grad", (2, 16, 64, 16, 4000, 64, 16, 1, 4, 64, 64, 16, 64, None), "W and dy"),
    ("lf_expert_linear_weight_grad", (2, 16, 64, 16, 64, 4, None, 16, 1, 4, 64, 64, 1, 16, None, 0, None), "FP32"),
    ("lf_mxfp4_quantize", (2, 16, 40, 4, 40, 16, 16, None), "multiple of 32"),
    ("lf_mxfp4_quantize", (2, 16, 32, 4, 64, 16, 16, None), "stride"),
    ("lf_mxfp4_dequantize", (2, 16, 16, 4, 64, 8, None), "16-byte"),
    ("lf_expert_linear_mxfp4", (2, 16, 16, 4, None, 16, 16, 16, 1, 4, 64, 48, 16, 64, None, 0, None), "multiple of 32"),
    ("lf_expert_linear_mxfp4", (2, 16, 16, 4, None, 16, 16, 16, 1, 4, 64, 64, 16, 63, None, 0, None), "overlap"),
    ("lf_expert_linear_mxfp4", (2, 16, 16, 200, None, 16, 16, 16, 1, 200, 64, 64, 16, 64, None, 0, None), "workspace"),
])
def test_sizes_are_checked_on_the_host(entry, args, match):
    with pytest.raises(RuntimeError, match=match):
        call(entry, args)


@pytest.mark.parametrize("tokens", [2**58, 2**59, 2**62, 2**63 - 1])
@pytest.mark.parametrize("entry,args", [
    ("lf_route_experts", lambda t: (0, 16, 32, t, 32, 32, 1, 1.0, 16, 16, 16, 16, 16, 16, 2**62, None)),
    ("lf_route_experts_backward", lambda t: (0, 16, 32, 16, 16, 16, 32, t, 32, 32, 1, 1.0, 16, 32, None)),
    ("lf_combine_experts", lambda t: (0, 16, 8, 4, 16, 16, t, 32, 8, 16, 8, None)),
    ("lf_combine_experts_backward", lambda t: (0, 16, 8, 16, 8, 4, 16, 16, t, 32, 8, 16, 8, 16, None)),
])
def test_slots_that_pass_64_bits(entry, args, tokens):
    with pytest.raises(RuntimeError, match="fit int32"):
        call(entry, args(tokens))


@pytest.mark.parametrize("entry,args", [
    ("lf_combine_experts", lambda n: (2, 16, n, 4, 16, 16, 2, 2, n, 16, n, None)),
    ("lf_combine_experts_backward", lambda n: (2, 16, n, 16, n, 4, 16, 16, 2, 2, n, 16, n, 16, None)),
])
@pytest.mark.parametrize("width", [2**31 - 1, 2**31 - 2048])
def test_widths_whose_columns_int32_does_not_hold(entry, args, width):
    with pytest.raises(RuntimeError, match="fit int32"):
        call(entry, args(width))


def test_workspace_sizes():
    assert _native.route_experts_workspace_ints(64, 64) == 0 and _native.route_experts_workspace_ints(65, 64) == 128
    assert _native.expert_linear_workspace_bytes(8, 64, 512) == 0  # eight rows a group: gathered by the loads
    assert _native.expert_linear_workspace_bytes(8, 65, 512) == 65 * 1024
    assert _native.expert_linear_workspace_bytes(8, 64, 512, weight_grad=True) == 64 * 1024
    assert _native.expert_linear_mxfp4_workspace_bytes(8, 16, 256, 512, True) == 0
    assert _native.expert_linear_mxfp4_workspace_bytes(8, 4000, 256, 512, True) > 2000 * 512
    with pytest.raises(ValueError, match="sizes"):
        _native.route_experts_workspace_ints(4, 1025)


def test_operators_need_a_cuda_tensor():
    torch = pytest.importorskip("torch")
    from loraforge_b200.ops.experts import combine_experts, expert_linear, route_experts
    from loraforge_b200.ops.mxfp4 import mxfp4_quantize

    x = torch.zeros(4, 32)
    for call in (lambda: route_experts(x, 2), lambda: mxfp4_quantize(x),
                 lambda: combine_experts(x, None, torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: expert_linear(x.bfloat16(), torch.zeros(1, 8, 32).bfloat16(), torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
