"""Routing and combination for mixture-of-experts layers against 64-bit forms, on the B200.

Tolerances.  A routing weight carries the rounding of l - peak (|l - peak| * 2^-24 relative,
below 2e-6 for |l| <= 15), expf (2 ulp) and sums of at most 32 + 5 FP32 additions (37 * 2^-24):
5e-6 relative in all; its gradient is a sum of at most k + 2 such products, so 2e-5 of the
row's largest |w g|.  combine: k FP32 FMAs and one rounding to the output type u: (k * 2^-24 + u)
of the sum of |w y|; a dot product over N: (N / 128 + 12) * 2^-24 of the sum of |g y|.
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200.ops.experts import (  # noqa: E402
    ExpertRouting, combine_experts, combine_experts_backward, route_experts, route_experts_backward)

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def reference(logits, k, renormalize, scale):
    """(weights, experts, offsets, rows, positions) in 64 bits, token by token."""
    l = logits.double().cpu().numpy().copy()
    l[np.isnan(l)] = -np.inf
    l = np.minimum(l, np.finfo(np.float32).max)
    T, E = l.shape
    weights, experts = np.zeros((T, k)), np.full((T, k), -1)
    for t in range(T):
        order = np.argsort(-l[t], kind="stable")[:k]
        order = order[l[t, order] > -np.inf]
        if not len(order):
            continue
        p = np.exp(l[t] - l[t].max())
        weights[t, : len(order)] = scale * p[order] / (p[order].sum() if renormalize else p.sum())
        experts[t, : len(order)] = order
    flat = experts.reshape(-1)
    rows, positions, offsets = np.full(T * k, -1), np.full(T * k, -1), np.zeros(E + 1, int)
    at = 0
    for e in range(E):
        offsets[e] = at
        for s in np.nonzero(flat == e)[0]:
            rows[at], positions[s] = s // k, at
            at += 1
    offsets[E] = at
    return weights, experts, offsets, rows, positions.reshape(T, k)


def check_routing(r, logits, k, renormalize, scale):
    weights, experts, offsets, rows, positions = reference(logits, k, renormalize, scale)
    for got, want in ((r.experts, experts), (r.offsets, offsets), (r.rows, rows), (r.positions, positions)):
        assert np.array_equal(got.cpu().numpy(), want)
    np.testing.assert_allclose(r.weights.double().cpu().numpy(), weights, rtol=5e-6, atol=1e-37)


@pytest.mark.parametrize("tokens,num_experts,k", [
    (1, 1, 1), (1, 64, 8), (5, 33, 6), (32, 8, 2), (33, 8, 2), (64, 1024, 32), (257, 40, 3), (1003, 256, 8),
    (300, 32, 32), (9000, 16, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_routing(tokens, num_experts, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    logits = (2 * torch.randn(tokens, num_experts, generator=g, device="cuda")).clamp(-15, 15).to(dtype)
    for renormalize, scale in ((True, 1.0), (False, 2.5)):
        check_routing(route_experts(logits, k, renormalize=renormalize, scale=scale), logits, k, renormalize, scale)


def test_masks_ties_and_special_values():
    inf, low = math.inf, torch.finfo(torch.float32).min
    rows = [
        [0.0] * 6,                                   # ties: the lowest indices
        [-inf] * 6,                                  # a padding token
        [-inf, -inf, 1.0, -inf, -inf, -inf],         # fewer than k left
        [low, low, low, 1.0, 2.0, low],              # masks of the lowest finite value can be taken
        [low] * 6,
        [math.nan, 1.0, math.nan, 3.0, -inf, 2.0],   # NaN is never taken
        [inf, 1.0, inf, 3.0, -inf, 2.0],             # +inf: the largest value
        [math.nan] * 6,
        [-0.0, 0.0, -0.0, 0.0, -1.0, 0.0],           # -0 and +0 tie
    ]
    logits = torch.tensor(rows, device="cuda")
    for k in (1, 3, 6):
        for renormalize in (True, False):
            r = route_experts(logits, k, renormalize=renormalize)
            check_routing(r, logits, k, renormalize, 1.0)
            grad = torch.randn(len(rows), k, device="cuda")
            d = route_experts_backward(logits, r, grad, renormalize=renormalize)
            assert torch.isfinite(d).all() and not d[1].any() and not d[7].any()
    every = route_experts(logits[1:2].expand(40, 6).contiguous(), 3)  # no token has an expert
    assert not every.offsets.any() and (every.rows == -1).all() and not every.weights.any()


def test_rows_of_a_wider_buffer_and_reused_tables():
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn(70, 50, generator=g, device="cuda").bfloat16()
    logits = wide[:, 3:43]
    first = route_experts(logits, 4)
    check_routing(first, logits, 4, True, 1.0)
    other = torch.randn(70, 40, generator=g, device="cuda").bfloat16()
    again = route_experts(other, 4, out=first)
    assert again.rows.data_ptr() == first.rows.data_ptr()
    check_routing(again, other, 4, True, 1.0)
    empty = route_experts(logits[:0], 4)
    assert empty.rows.numel() == 0 and empty.offsets.tolist() == [0] * 41


def forward64(l, experts, renormalize, scale):
    """Weights of fixed experts as a function of 64-bit logits."""
    p = np.exp(l - l.max(1, keepdims=True))
    taken = np.take_along_axis(p, np.maximum(experts, 0), 1) * (experts >= 0)
    return scale * taken / (taken if renormalize else p).sum(1, keepdims=True)


@pytest.mark.parametrize("tokens,num_experts,k", [(1, 8, 2), (65, 64, 6), (40, 300, 8)])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (False, 1.0), (False, 2.5), (True, 0.5)])
def test_routing_gradient(tokens, num_experts, k, renormalize, scale):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    logits = 2 * torch.randn(tokens, num_experts, generator=g, device="cuda")
    grad = torch.randn(tokens, k, generator=g, device="cuda")
    r = route_experts(logits, k, renormalize=renormalize, scale=scale)
    got = route_experts_backward(logits, r, grad, renormalize=renormalize, scale=scale).double().cpu().numpy()
    l, gw, experts = logits.double().cpu().numpy(), grad.double().cpu().numpy(), r.experts.cpu().numpy()
    # The formula's gradient, by 64-bit autograd.
    tl = torch.tensor(l, requires_grad=True)
    p = torch.softmax(tl, 1)
    w = torch.gather(p, 1, torch.tensor(experts).long())
    w = scale * (w / w.sum(1, keepdim=True) if renormalize else w)
    (w * torch.tensor(gw)).sum().backward()
    size = np.abs(forward64(l, experts, renormalize, scale) * gw).max(1, keepdims=True)
    assert (np.abs(got - tl.grad.numpy()) <= 2e-5 * size).all()
    # And differences of the 64-bit forward along a few logits.
    h = 1e-5
    for i in range(0, num_experts, max(1, num_experts // 5)):
        up, down = l.copy(), l.copy()
        up[:, i] += h
        down[:, i] -= h
        slope = ((forward64(up, experts, renormalize, scale) - forward64(down, experts, renormalize, scale)) * gw).sum(1)
        # central differences: h^2 / 6 of third derivatives (a few |w g|) and 2^-53 / h of rounding
        assert (np.abs(got[:, i] - slope / (2 * h)) <= 3e-5 * size[:, 0] + 1e-9).all()


def combine64(y, weights, positions):
    y, w, at = y.double(), weights.double(), positions.long()
    live = (at >= 0)[..., None]
    rows = torch.where(live, y[at.clamp(min=0)], 0.0)
    return (w[..., None] * rows).sum(1), (w.abs()[..., None] * rows.abs()).sum(1), rows


@pytest.mark.parametrize("tokens,k,width", [(1, 1, 1), (1, 8, 2048), (7, 2, 129), (64, 6, 520), (300, 32, 40), (33, 2, 14336)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_combination_and_gradients(tokens, k, width, dtype):
    g = torch.Generator(device="cuda").manual_seed(width)
    logits = torch.randn(tokens, max(k, 12), generator=g, device="cuda")
    if tokens > 2:
        logits[1] = -math.inf  # a token without rows
    r = route_experts(logits, k)
    y = torch.randn(tokens * k, width, generator=g, device="cuda").to(dtype)
    y[r.rows < 0] = math.nan  # rows of no slot are not read
    grad = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    out = combine_experts(y, r.weights, r.positions)
    want, size, rows = combine64(y, r.weights, r.positions)
    assert ((out.double() - want).abs() <= (k * 2.0**-24 + UNIT[dtype]) * size + 1e-30).all()
    if tokens > 2:
        assert not out[1].any()
    grad_y, grad_w = combine_experts_backward(grad, y, r.weights, r.positions)
    dot, dot_size = (grad.double()[:, None] * rows).sum(2), (grad.double()[:, None] * rows).abs().sum(2)
    assert ((grad_w.double() - dot).abs() <= (width / 128 + 12) * 2.0**-24 * dot_size).all()
    live = r.positions >= 0
    scaled = r.weights.double()[..., None] * grad.double()[:, None]
    near = torch.zeros_like(y, dtype=torch.float64)
    near[r.positions[live].long()] = scaled[live]
    assert ((grad_y.double() - near).abs() <= UNIT[dtype] * near.abs() + 6e-8).all()  # 2^-24: fp16's subnormals
    # The sum is linear in y and in the weights: a difference along a direction is exact in 64 bits.
    step = torch.zeros_like(y, dtype=torch.float64)
    step[r.rows >= 0] = torch.randn(int((r.rows >= 0).sum()), width, generator=g, device="cuda").double()
    clean = torch.where(torch.isnan(y), torch.zeros_like(y), y).double()
    moved = combine64(clean + step, r.weights, r.positions)[0] - combine64(clean, r.weights, r.positions)[0]
    left, right = (moved * grad.double()).sum(), (step * grad_y.double()).sum()
    bound = (UNIT[dtype] * (step.abs() * near.abs()).sum() + 6e-8 * step.abs().sum() + 1e-9)
    assert (left - right).abs() <= bound
    # Ones for weights: the gradient of a gather.
    ones = combine_experts(y, None, r.positions)
    want, size, _ = combine64(y, torch.ones_like(r.weights), r.positions)
    assert ((ones.double() - want).abs() <= (k * 2.0**-24 + UNIT[dtype]) * size + 1e-30).all()
    assert combine_experts_backward(grad, y, None, r.positions)[1] is None


def test_unaligned_rows_and_streams():
    g = torch.Generator(device="cuda").manual_seed(8)
    wide = torch.randn(40, 131, generator=g, device="cuda").bfloat16()
    y, side = wide[:, 1:130], torch.cuda.Stream()
    r = route_experts(torch.randn(20, 5, generator=g, device="cuda"), 2)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = combine_experts(y, r.weights, r.positions)
    torch.cuda.current_stream().wait_stream(side)
    want, size, _ = combine64(y, r.weights, r.positions)
    assert ((out.double() - want).abs() <= (2 * 2.0**-24 + 2.0**-8) * size).all()


def test_layer_tables_in_a_captured_graph():
    g = torch.Generator(device="cuda").manual_seed(9)
    logits = torch.randn(50, 16, generator=g, device="cuda")
    y = torch.randn(100, 64, generator=g, device="cuda").bfloat16()
    r = route_experts(logits, 2)
    out = combine_experts(y, r.weights, r.positions)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        route_experts(logits, 2, out=r)
        combine_experts(y, r.weights, r.positions, out=out)
    logits.copy_(torch.randn(50, 16, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    check_routing(r, logits, 2, True, 1.0)
    assert torch.equal(out, combine_experts(y, r.weights, r.positions))


def test_refusals():
    logits = torch.randn(4, 8, device="cuda")
    for bad, error in ((dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"), (dict(top_k=2.0), "top_k"),
                       (dict(top_k=2, scale=0.0), "scale"), (dict(top_k=2, scale=math.inf), "scale"),
                       (dict(top_k=2, renormalize=1), "renormalize")):
        with pytest.raises(ValueError, match=error):
            route_experts(logits, **bad)
    with pytest.raises(TypeError, match="logits"):
        route_experts([1.0], 1)
    with pytest.raises(ValueError, match="dtype"):
        route_experts(logits.double(), 2)
    with pytest.raises(ValueError, match="CUDA"):
        route_experts(logits.cpu(), 2)
    with pytest.raises(ValueError, match="unit column stride"):
        route_experts(torch.randn(8, 4, device="cuda").T, 2)
    with pytest.raises(ValueError, match="experts"):
        route_experts(torch.randn(2, 1025, device="cuda"), 2)
    r = route_experts(logits, 2)
    with pytest.raises(ValueError, match="out.rows"):
        route_experts(logits, 2, out=r._replace(rows=r.rows[:-1]))
    with pytest.raises(TypeError, match="routing"):
        route_experts_backward(logits, tuple(r), r.weights)
    with pytest.raises(ValueError, match="grad_weights"):
        route_experts_backward(logits, r, r.weights[:2])
    y = torch.randn(8, 16, device="cuda")
    with pytest.raises(ValueError, match="weights"):
        combine_experts(y, r.weights.double(), r.positions)
    with pytest.raises(ValueError, match="positions"):
        combine_experts(y, r.weights, r.positions.long())
    with pytest.raises(ValueError, match="share storage"):
        combine_experts(y, r.weights, r.positions, out=y[:4])
    with pytest.raises(ValueError, match="grad"):
        combine_experts_backward(y[:3], y, r.weights, r.positions)
    assert isinstance(r, ExpertRouting)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradient_of_the_weights_adds_up_short_chains(dtype):
    # The first value each lane of the warp reads is 1, all others half a unit in 1's last place,
    # which an addition to it drops: a lane's chain over its N / 32 terms would lose 447 units of
    # 2^-24 of the sum, chains of at most N / 128 terms and their joining stay below N / 128 + 12.
    N, lane = 14336, 16 // torch.empty(0, dtype=dtype).element_size()
    r = route_experts(torch.zeros(2, 3, device="cuda"), 2)
    y = torch.full((4, N), 2.0**-24, device="cuda", dtype=dtype)
    y[:, : 32 * lane : lane] = 1.0
    grad = torch.ones(2, N, device="cuda", dtype=dtype)
    got = combine_experts_backward(grad, y, r.weights, r.positions)[1].double()
    want = y.double().sum(1)[r.positions.long()]
    assert ((got - want).abs() <= (N / 128 + 12) * 2.0**-24 * want).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renormalize,scale", [(True, 1.0), (False, 1.0), (False, 2.5), (True, 0.5)])
def test_routing_gradient_with_fewer_experts_than_choices(renormalize, scale, dtype):
    # Most experts masked: 0, 1, .. k + 1 of them left, by -inf and by NaN, some of the finite logits
    # near the lowest value; the rows of the gradients are strided.
    g = torch.Generator(device="cuda").manual_seed(7)
    E, k = 12, 4
    logits = (2 * torch.randn(36, E, generator=g, device="cuda")).to(dtype)
    for t in range(36):
        gone = torch.randperm(E, generator=g, device="cuda")[: E - t % 6]
        logits[t, gone] = -math.inf if t % 2 else math.nan
    logits[5, torch.isfinite(logits[5])] -= 1e30
    wide = torch.randn(36, 9, generator=g, device="cuda")
    grad = wide[:, 2 : 2 + k]
    r = route_experts(logits, k, renormalize=renormalize, scale=scale)
    check_routing(r, logits, k, renormalize, scale)
    got = route_experts_backward(logits, r, grad, renormalize=renormalize, scale=scale).double()
    # The formula in 64 bits over the experts left.
    l = torch.where(torch.isfinite(logits), logits, -math.inf).double().cpu().requires_grad_()
    experts = r.experts.cpu().long()
    for t in range(36):
        left = torch.isfinite(l[t].detach())
        taken = experts[t][experts[t] >= 0]
        assert len(taken) == min(k, int(left.sum())) == min(k, t % 6)
        if not len(taken):
            assert not got[t].any()
            continue
        p = torch.softmax(l[t][left], 0)
        full = torch.zeros(E, dtype=torch.float64).masked_scatter(left, p)
        w = full[taken] / (full[taken].sum() if renormalize else 1.0) * scale
        gw = grad[t, : len(taken)].double().cpu()
        (want,) = torch.autograd.grad((w * gw).sum(), l)
        far = (got[t].cpu() - want[t].nan_to_num(0.0)).abs() - UNIT[dtype] * want[t].nan_to_num(0.0).abs()
        assert (far <= 2e-5 * (w * gw).abs().max()).all(), t


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_combination_of_strided_gradients(dtype):
    g = torch.Generator(device="cuda").manual_seed(10)
    r = route_experts(torch.randn(30, 7, generator=g, device="cuda"), 3)
    for N, pad in ((64, 16), (61, 3)):  # 16-byte and element-wise rows
        y = torch.randn(90, N + pad, generator=g, device="cuda").to(dtype)[:, pad // 2 : pad // 2 + N]
        grad = torch.randn(30, N + 2 * pad, generator=g, device="cuda").to(dtype)[:, pad : pad + N]
        got = combine_experts_backward(grad, y, r.weights, r.positions)
        want = combine_experts_backward(grad.contiguous(), y.contiguous(), r.weights, r.positions)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        rows = y.double()[r.positions.long()]
        near = (r.weights.double()[..., None] * grad.double()[:, None]).reshape(90, N)
        assert ((got[0].double()[r.positions.long().reshape(-1)] - near).abs() <= UNIT[dtype] * near.abs() + 6e-8).all()
        size = (grad.double()[:, None] * rows).abs().sum(2)
        assert ((got[1].double() - (grad.double()[:, None] * rows).sum(2)).abs() <= (N / 128 + 12) * 2.0**-24 * size).all()


def test_combination_past_32_bits():
    # 2.2e9 values of y and of its gradient, 1.1e9 of the output: the last tokens against 64 bits.
    T, k, N = 67600, 2, 16384
    g = torch.Generator(device="cuda").manual_seed(11)
    r = route_experts(torch.randn(T, 4, generator=g, device="cuda"), k)
    y = torch.empty(T * k, N, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    grad = torch.empty(T, N, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    assert T * k * N > 2**31
    out = combine_experts(y, r.weights, r.positions)
    grad_y, grad_w = combine_experts_backward(grad, y, r.weights, r.positions)
    last = slice(T - 64, T)
    at, w, gl = r.positions[last].long(), r.weights[last].double(), grad[last].double()
    rows = y[at].double()
    assert int(at.max()) * N > 2**31
    far = (out[last].double() - (w[..., None] * rows).sum(1)).abs() - (w[..., None] * rows).abs().sum(1) * (k * 2.0**-24 + 2.0**-8)
    assert (far <= 0).all()
    near = w[..., None] * gl[:, None]
    assert ((grad_y[at].double() - near).abs() <= 2.0**-8 * near.abs() + 1e-30).all()
    terms = gl[:, None] * rows
    assert ((grad_w[last].double() - terms.sum(2)).abs() <= (N / 128 + 12) * 2.0**-24 * terms.abs().sum(2)).all()
