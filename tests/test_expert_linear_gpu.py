"""Products grouped by expert and their gradients against 64-bit sums, on the B200.

Tolerance: FP32 sums of C exact products of 16-bit values in any order and grouping stay within
C * 2^-22 of the sum of magnitudes (tensor cores may cut, not round: 2^-23 a step, twice that
for aligning a group of products), and the output is rounded once to its type (half a unit,
2^-8 for BF16's and 2^-11 for FP16's spacing, 2^-24 for FP16's subnormals).
"""

import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="CUDA device required"),
]

from loraforge_b200 import _native  # noqa: E402
from loraforge_b200.ops.experts import (  # noqa: E402
    combine_experts, expert_linear, expert_linear_backward, route_experts)

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def bound(size, C, dtype):
    return size * (C * 2.0**-22 + UNIT[dtype]) + 2.0**-24


def near(got, want, size, C):
    far = (got.double() - want).abs() - bound(size, C, got.dtype)
    assert torch.isfinite(got).all() and (far <= 0).all(), far.max().item()


def check_forward(x, w, offsets, rows, y):
    bounds = offsets.tolist()
    for e in range(w.shape[0]):
        a, b = bounds[e], bounds[e + 1]
        xe = (x[rows[a:b].long()] if rows is not None else x[a:b]).double()
        we = w[e].double()
        near(y[a:b], xe @ we.T, xe.abs() @ we.abs().T, w.shape[2])
    assert not y[bounds[-1]:].any()


def check_backward(grad, x, w, offsets, rows, dx, dw):
    bounds = offsets.tolist()
    for e in range(w.shape[0]):
        a, b = bounds[e], bounds[e + 1]
        xe = (x[rows[a:b].long()] if rows is not None else x[a:b]).double()
        ge, we = grad[a:b].double(), w[e].double()
        near(dx[a:b], ge @ we, ge.abs() @ we.abs(), w.shape[1])
        near(dw[e], ge.T @ xe, ge.abs().T @ xe.abs(), max(1, b - a))
    assert not dx[bounds[-1]:].any()


def make(counts, N, K, dtype, seed, tail=0, tokens=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    E, R = len(counts), sum(counts) + tail
    tokens = max(1, R // 2) if tokens is None else tokens
    offsets = torch.tensor([0, *counts], device="cuda").cumsum(0).to(torch.int32)
    rows = torch.randint(0, tokens, (R,), generator=g, device="cuda").to(torch.int32)
    x = torch.randn(tokens, K, generator=g, device="cuda").to(dtype)
    w = (torch.randn(E, N, K, generator=g, device="cuda") / math.sqrt(K)).to(dtype)
    grad = torch.randn(R, N, generator=g, device="cuda").to(dtype)
    return x, w, offsets, rows, grad


COUNTS = {
    "one row": [1],
    "one each": [1] * 8,
    "empty groups": [0, 3, 0, 0, 17, 1, 0],
    "few, ragged": [5, 64, 0, 65, 2, 33, 16, 15],
    "even": [128, 128],
    "wide": [300, 0, 17, 600, 256, 1, 129],
    "dense": [777],
    "none": [0, 0, 0],
}


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("N,K,dtype", [(128, 64, torch.bfloat16), (264, 200, torch.float16), (1416, 512, torch.bfloat16), (8, 8, torch.bfloat16)])
def test_products_and_gradients(name, N, K, dtype):
    counts = COUNTS[name]
    x, w, offsets, rows, grad = make(counts, N, K, dtype, seed=N + len(counts), tail=3)
    rows[sum(counts):] = -1
    y = expert_linear(x, w, offsets, rows=rows)
    check_forward(x, w, offsets, rows, y)
    dx, dw = expert_linear_backward(grad, x, w, offsets, rows=rows)
    check_backward(grad, x, w, offsets, rows, dx, dw)
    # Rows that are sorted already, and FP32 weight gradients.
    sorted_x = x[rows.clamp(min=0).long()].contiguous()
    y2 = expert_linear(sorted_x, w, offsets)
    assert torch.equal(y2, y)  # the same products in the same order
    dx2, dw2 = expert_linear_backward(grad, sorted_x, w, offsets, weight_grad_dtype=torch.float32)
    check_backward(grad, sorted_x, w, offsets, None, dx2, dw2)
    assert torch.equal(dx2, dx) and torch.equal(dw2.to(dtype), dw)
    assert _native.device_wait_timeouts(reset=True) == 0


@pytest.mark.parametrize("counts,N,K", [([1], 256, 8192), ([3, 2], 64, 4104), ([16, 1, 0, 7], 136, 2048), ([64], 2048, 1024)])
def test_contractions_split_over_a_cluster(counts, N, K):
    x, w, offsets, rows, _ = make(counts, N, K, torch.bfloat16, seed=K)
    y = expert_linear(x, w, offsets, rows=rows)
    check_forward(x, w, offsets, rows, y)
    assert torch.equal(expert_linear(x, w, offsets, rows=rows), y)  # the parts are added in one order
    assert _native.device_wait_timeouts(reset=True) == 0


# Rows on average where the tiles change (16 and 24 rows a group), with groups of one row and of
# more than a tile's, and contractions where the stores do (768).
@pytest.mark.parametrize("counts", [[16] * 4, [1, 64, 0, 3], [20, 17, 15, 20], [1, 90, 4, 1], [24] * 4, [25, 24, 25, 24]])
@pytest.mark.parametrize("N,K", [(136, 776), (776, 768), (520, 264)])
def test_sizes_where_the_tiles_change(counts, N, K):
    x, w, offsets, rows, grad = make(counts, N, K, torch.bfloat16, seed=sum(counts) + K, tail=0)
    y = expert_linear(x, w, offsets, rows=rows)
    check_forward(x, w, offsets, rows, y)
    assert torch.equal(expert_linear(x[rows.long()].contiguous(), w, offsets), y)
    check_backward(grad, x, w, offsets, rows, *expert_linear_backward(grad, x, w, offsets, rows=rows))
    assert _native.device_wait_timeouts(reset=True) == 0


@pytest.mark.parametrize("counts", [[768], [769], [1500, 36], [2, 1536]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weight_gradients_of_many_rows(counts, dtype):
    x, w, offsets, rows, grad = make(counts, 328, 520, dtype, seed=sum(counts))
    check_backward(grad, x, w, offsets, rows, *expert_linear_backward(grad, x, w, offsets, rows=rows))
    dx, dw = expert_linear_backward(grad, x, w, offsets, rows=rows, weight_grad_dtype=torch.float32)
    check_backward(grad, x, w, offsets, rows, dx, dw)
    assert _native.device_wait_timeouts(reset=True) == 0


def test_large_products():
    x, w, offsets, rows, grad = make([1500, 260, 2000, 3], 2048, 1024, torch.bfloat16, seed=1)
    check_forward(x, w, offsets, rows, expert_linear(x, w, offsets, rows=rows))
    check_backward(grad, x, w, offsets, rows, *expert_linear_backward(grad, x, w, offsets, rows=rows))


@pytest.mark.parametrize("counts", [[3, 2, 4], [300, 70, 200]])
def test_a_group_does_not_see_its_neighbours(counts):
    # Infinities and NaN in one expert's rows and weights stay there.
    x, w, offsets, _, grad = make(counts, 200, 136, torch.bfloat16, seed=7, tokens=sum(counts))
    y = expert_linear(x, w, offsets)
    dx, dw = expert_linear_backward(grad, x, w, offsets)
    lo, hi = offsets[1], offsets[2]
    for t in (x, grad):
        t[lo:hi] = math.inf
        t[lo] = math.nan
    w[1] = math.nan
    y2 = expert_linear(x, w, offsets)
    dx2, dw2 = expert_linear_backward(grad, x, w, offsets)
    for a, b in ((y, y2), (dx, dx2)):
        assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:]) and not torch.isfinite(b[lo:hi]).any()
    assert torch.equal(dw[0], dw2[0]) and torch.equal(dw[2], dw2[2]) and torch.isnan(dw2[1]).all()


def test_gradients_against_differences():
    # <dy, y(x + s) - y(x)> for a step s is linear: the gradients' products with s, up to rounding.
    x, w, offsets, _, grad = make([40, 0, 9], 72, 48, torch.bfloat16, seed=3, tokens=49)
    g = torch.Generator(device="cuda").manual_seed(4)
    dx, dw = expert_linear_backward(grad, x, w, offsets, weight_grad_dtype=torch.float32)

    def loss(x64, w64):
        bounds = offsets.tolist()
        return sum((grad[a:b].double() * (x64[a:b] @ w64[e].T)).sum()
                   for e, (a, b) in enumerate(zip(bounds, bounds[1:])))

    step = torch.randn(x.shape, generator=g, device="cuda").double()
    slope = loss(x.double() + step, w.double()) - loss(x.double(), w.double())
    size = 72 * step.abs().sum() * grad.abs().double().max() * w.abs().double().max()
    assert (slope - (dx.double() * step).sum()).abs() <= 2.0**-8 * (dx.double() * step).abs().sum() + 72 * 2.0**-22 * size
    step = torch.randn(w.shape, generator=g, device="cuda").double()
    slope = loss(x.double(), w.double() + step) - loss(x.double(), w.double())
    size = 40 * step.abs().sum() * grad.abs().double().max() * x.abs().double().max()
    assert (slope - (dw.double() * step).sum()).abs() <= 40 * 2.0**-22 * size


def test_strided_operands_and_output():
    g = torch.Generator(device="cuda").manual_seed(5)
    wide = torch.randn(50, 304, generator=g, device="cuda").bfloat16()
    x = wide[:, 8:136]
    store = torch.randn(3, 2, 96, 136, generator=g, device="cuda").bfloat16() / 12
    w = store[:, 1, :, :128]
    offsets = torch.tensor([0, 20, 20, 50], dtype=torch.int32, device="cuda")
    buffer = torch.full((50, 101), 7.0, device="cuda").bfloat16()
    out = expert_linear(x, w, offsets, out=buffer[:, 2:98])
    check_forward(x, w, offsets, None, out)
    assert (buffer[:, :2] == 7).all() and (buffer[:, 98:] == 7).all()
    grad = torch.randn(50, 200, generator=g, device="cuda").bfloat16()[:, 16:112]
    check_backward(grad, x, w, offsets, None, *expert_linear_backward(grad, x, w, offsets))


def test_rows_outside_x_read_zeros_and_bounds_stay_inside():
    x, w, offsets, rows, _ = make([6, 6], 64, 64, torch.bfloat16, seed=9)
    rows[1], rows[7] = -1, x.shape[0] + 5
    y = expert_linear(x, w, offsets, rows=rows)
    assert not y[1].any() and not y[7].any() and y[0].any()
    wild = torch.tensor([-4, 1000, 5], dtype=torch.int32, device="cuda")  # taken as 0, 12, 12
    tame = torch.tensor([0, 12, 12], dtype=torch.int32, device="cuda")
    assert torch.equal(expert_linear(x, w, wild, rows=rows), expert_linear(x, w, tame, rows=rows))


def test_layer_of_experts():
    # Router, two products and the sum, against the same layer in 64 bits over its own tables.
    g = torch.Generator(device="cuda").manual_seed(11)
    T, E, k, H, I = 70, 6, 2, 128, 256
    h = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    up = (torch.randn(E, I, H, generator=g, device="cuda") / math.sqrt(H)).bfloat16()
    down = (torch.randn(E, H, I, generator=g, device="cuda") / math.sqrt(I)).bfloat16()
    r = route_experts(torch.randn(T, E, generator=g, device="cuda"), k)
    y = expert_linear(torch.relu(expert_linear(h, up, r.offsets, rows=r.rows)), down, r.offsets)
    out = combine_experts(y, r.weights, r.positions).double()
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for j in range(k):
        e = r.experts[:, j].long()
        mid = torch.relu(torch.einsum("th,tih->ti", h.double(), up[e].double()))
        want += r.weights[:, j, None].double() * torch.einsum("ti,thi->th", mid, down[e].double())
    # Three roundings to BF16 on the way, each at most 2^-9 relative: well inside 2^-7 of the norm.
    assert (out - want).norm() <= 2.0**-7 * want.norm()


@pytest.mark.parametrize("tokens", [600, 20000])
def test_a_thousand_experts(tokens):
    g = torch.Generator(device="cuda").manual_seed(12)
    r = route_experts(torch.randn(tokens, 1024, generator=g, device="cuda"), 5)
    x = torch.randn(tokens, 72, generator=g, device="cuda").bfloat16()
    w = (torch.randn(1024, 40, 72, generator=g, device="cuda") / 8).bfloat16()
    grad = torch.randn(tokens * 5, 40, generator=g, device="cuda").bfloat16()
    check_forward(x, w, r.offsets, r.rows, expert_linear(x, w, r.offsets, rows=r.rows))
    check_backward(grad, x, w, r.offsets, r.rows, *expert_linear_backward(grad, x, w, r.offsets, rows=r.rows))


def test_offsets_past_32_bits():
    # 2.4e9 weights, then 2.2e9 outputs: the last expert's rows against 64 bits.
    N, K, E = 32768, 24576, 3
    w = torch.empty(E, N, K, dtype=torch.bfloat16, device="cuda")
    for e in range(E):
        w[e].normal_(std=K**-0.5)
    offsets = torch.tensor([0, 2, 3, 5], dtype=torch.int32, device="cuda")
    x = torch.randn(5, K, device="cuda").bfloat16()
    y = expert_linear(x, w, offsets)
    want, size = x[3:].double() @ w[2, -512:].double().T, x[3:].double().abs() @ w[2, -512:].double().abs().T
    near(y[3:, -512:], want, size, K)
    del w, y
    R, N, K = 70000, 32000, 32
    x = torch.randn(R, K, device="cuda").bfloat16()
    w = torch.randn(2, N, K, device="cuda").bfloat16()
    offsets = torch.tensor([0, 30000, R], dtype=torch.int32, device="cuda")
    y = expert_linear(x, w, offsets)
    near(y[-64:], x[-64:].double() @ w[1].double().T, x[-64:].double().abs() @ w[1].double().abs().T, K)


@pytest.mark.parametrize("counts", [[3, 0, 2], [40, 300, 90]])
def test_other_streams_and_captured_graphs(counts):
    x, w, offsets, rows, grad = make(counts, 136, 200, torch.bfloat16, seed=13)
    want, want_grads = expert_linear(x, w, offsets, rows=rows), expert_linear_backward(grad, x, w, offsets, rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = expert_linear(x, w, offsets, rows=rows)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = expert_linear(x, w, offsets, rows=rows)
        grads = expert_linear_backward(grad, x, w, offsets, rows=rows)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(grads, want_grads))


def test_refusals():
    x, w, offsets, rows, grad = make([4, 4], 64, 64, torch.bfloat16, seed=2)
    with pytest.raises(TypeError, match="weight"):
        expert_linear(x, None, offsets)
    with pytest.raises(ValueError, match="dtype"):
        expert_linear(x.float(), w, offsets)
    with pytest.raises(ValueError, match="dtype"):
        expert_linear(x, w.half(), offsets, rows=rows)
    with pytest.raises(ValueError, match="offsets"):
        expert_linear(x, w, offsets[:2], rows=rows)
    with pytest.raises(ValueError, match="offsets"):
        expert_linear(x, w, offsets.long(), rows=rows)
    with pytest.raises(ValueError, match="width"):
        expert_linear(x[:, :32].contiguous(), w, offsets, rows=rows)
    with pytest.raises(ValueError, match="multiples of 8"):
        expert_linear(torch.zeros(8, 70, device="cuda").bfloat16()[:, 1:65], w, offsets)
    with pytest.raises(ValueError, match="multiples of 8"):
        expert_linear(x, w[:, :60], offsets, rows=rows)
    with pytest.raises(ValueError, match="out must"):
        expert_linear(x, w, offsets, rows=rows, out=torch.empty(7, 64, device="cuda").bfloat16())
    with pytest.raises(ValueError, match="share storage"):
        expert_linear(x, w, offsets, out=x)
    with pytest.raises(ValueError, match="grad"):
        expert_linear_backward(grad[:3], x, w, offsets, rows=rows)
    with pytest.raises(ValueError, match="weight_grad_dtype"):
        expert_linear_backward(grad, x, w, offsets, rows=rows, weight_grad_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="workspace"):
        _native.call("lf_expert_linear", 2, 16, 64, 4, 16, 16, 4096, 64, 16, 1, 100, 64, 64, 16, 64, None, 0, None)
    with pytest.raises(RuntimeError, match="experts"):
        _native.call("lf_expert_linear", 2, 16, 64, 4, None, 16, 4096, 64, 16, 2000, 4, 64, 64, 16, 64, None, 0, None)


# A rank that holds the experts lo .. hi - 1 passes its part of the offsets with all rows: those of
# other experts, before the first bound and from the last one on, are rows of no group.
SLICES = [
    ([3, 0, 5, 2, 1, 4], 2, 5),          # few rows: gathered by the loads
    ([9, 14, 17, 12, 11], 1, 3),         # the narrow tiles with rows put in order
    ([40, 300, 90, 0, 260, 7], 1, 5),    # pairs
    ([30, 70, 0, 0], 2, 4),              # no row of its own
    ([600, 5], 1, 2),                    # all but the last few rows are others'
]


@pytest.mark.parametrize("counts,lo,hi", SLICES)
@pytest.mark.parametrize("by_index", [True, False])
@pytest.mark.parametrize("N,K,dtype", [(136, 200, torch.bfloat16), (264, 1024, torch.float16)])
def test_a_slice_of_the_experts(counts, lo, hi, by_index, N, K, dtype):
    x, w, offsets, rows, grad = make(counts, N, K, dtype, seed=sum(counts) + lo, tail=2)
    rows[sum(counts):] = -1
    if not by_index:
        x, rows = x[rows.clamp(min=0).long()].contiguous(), None
    R, mine, part = grad.shape[0], w[lo:hi], offsets[lo : hi + 1]
    y = torch.full((R, N), math.nan, device="cuda", dtype=dtype)
    expert_linear(x, mine, part, rows=rows, out=y)
    check_forward(x, mine, part, rows, y)
    dx = torch.full((R, K), math.nan, device="cuda", dtype=dtype)
    _native.launch("lf_expert_linear_input_grad", 0, _native.dtype_code(dtype), grad.data_ptr(), N, mine.data_ptr(), N * K, K,
                   part.data_ptr(), hi - lo, R, N, K, dx.data_ptr(), K)
    check_backward(grad, x, mine, part, rows, dx, expert_linear_backward(grad, x, mine, part, rows=rows)[1])
    first = int(part[0])
    assert not y[:first].any() and not dx[:first].any()


def test_rows_before_the_first_bound_of_a_strided_output():
    x, w, offsets, rows, _ = make([70, 40, 33], 96, 128, torch.bfloat16, seed=21)
    for width, left in ((104, 0), (101, 2)):  # 16-byte and element-wise stores
        buffer = torch.full((143, width), 7.0, device="cuda").bfloat16()
        y = expert_linear(x, w[1:], offsets[1:], rows=rows, out=buffer[:, left : left + 96])
        check_forward(x, w[1:], offsets[1:], rows, y)
        assert not y[:70].any() and (buffer[:, :left] == 7).all() and (buffer[:, left + 96 :] == 7).all()
